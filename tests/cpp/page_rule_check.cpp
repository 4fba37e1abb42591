// Sums the new pages of sequences as a call does: one line "old more width shift" of stdin each; prints the sum, or
// "refused" where one of them may not grow so.
#include <cstdio>

#include "page_rule.hpp"

int main() {
  long long old, more, width;
  int shift;
  bool refused = false;
  decltype(praghip::new_pages(0, 0, 0, 0)) sum = 0;
  while (std::scanf("%lld %lld %lld %d", &old, &more, &width, &shift) == 4) {
    const auto pages = praghip::new_pages(old, more, width, shift);
    refused |= pages < 0;
    sum += pages;
  }
  if (refused)
    std::printf("refused\n");
  else
    std::printf("%lld\n", static_cast<long long>(sum));
}
