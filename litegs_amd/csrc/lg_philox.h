// Counter-based random words: Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC'11).  Word i of a draw is word i % 4 of the block with counter (i / 4 in the low 64 bits, `offset` in the high 64 bits) under the 64-bit
// key `seed`: a word depends on (seed, offset, i) only -- never on the launch, the device or the rank -- so a mask can be drawn again in a
// backward pass instead of being stored, and replicas that call with the same numbers take the same decisions.
#pragma once
#include <stdint.h>

struct LgWords { uint32_t w[4]; };

__device__ __forceinline__ LgWords lg_philox(unsigned long long block, unsigned long long offset, unsigned long long seed)
{
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return LgWords{ { c0, c1, c2, c3 } };
}
