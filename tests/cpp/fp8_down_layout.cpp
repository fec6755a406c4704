// LDS of the launch that multiplies few tokens' hidden rows and sums them: parts that do not overlap, each aligned to what is stored there at once.
#include "launch_dims.h"

#include <cstdio>

int main() {
    for (int slots = 1; slots < 1024; slots++) {
        for (int blocks = 1; blocks <= 64; blocks++) {
            const bf16n::dev::fp8_down_lds l = bf16n::dev::fp8_down_layout(slots, blocks);
            if (l.pitch % 16 || l.pitch < blocks * 128 || l.scales % 16 || l.results % 16 || l.scales < slots * l.pitch || l.results < l.scales + slots * blocks * 4 ||
                l.bytes < l.results + slots * 16 * 4) {
                std::printf("%d slots, %d blocks: %d %d %d %d\n", slots, blocks, l.pitch, l.scales, l.results, l.bytes);
                return 1;
            }
        }
    }
    return 0;
}
