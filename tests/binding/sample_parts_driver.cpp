// Prints part_of for the argument lines "float_bits weight up" on stdin.
#include <bit>
#include <cinttypes>
#include <cstdio>
#include "sample_parts.h"
int main() {
    uint32_t bits;
    uint64_t weight;
    int up;
    while (std::scanf("%" SCNu32 " %" SCNu64 " %d", &bits, &weight, &up) == 3)
        std::printf("%" PRIu64 "\n", sandy_hip::part_of(std::bit_cast<float>(bits), weight, up != 0));
}
