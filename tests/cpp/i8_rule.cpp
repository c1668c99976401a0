// Prints the kernel that the rule of helixml_amd/csrc/hx_i8_rule.h gives for each line "M N K whole_rows" of the input.
#include <cstdio>

#include "hx_i8_rule.h"

int main() {
    const char* const names[] = {"rows 16x16", "rows 32x32", "rows 64x32", "tiles 128", "tiles 256"};
    long long m, n, k;
    int whole;
    while (std::scanf("%lld %lld %lld %d", &m, &n, &k, &whole) == 4) std::printf("%s\n", names[(int)hx::i8_kernel(m, n, k, whole != 0)]);
}
