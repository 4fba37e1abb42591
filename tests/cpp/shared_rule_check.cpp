// The table's entry of 16 keys: one line "block half page_shift last" of stdin each; prints each entry.
#include <cstdio>

#include "shared_rule.hpp"

int main() {
  unsigned block, half, last;
  int shift;
  while (std::scanf("%u %u %d %u", &block, &half, &shift, &last) == 4)
    std::printf("%lld\n", static_cast<long long>(praghip::entry_at(block, half, shift, last)));
}
