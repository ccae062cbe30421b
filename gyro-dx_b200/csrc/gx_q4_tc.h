// gx_q4_tc.h — sizes of the 4-bit product for batches (gx_q4.cu) and of the rings its warps meet in, plain C++
// so that tests/ring_emu.cpp walks through the same rings on the CPU.
#pragma once
#include <stdint.h>

#include "../../include/gyro_moe.h"

namespace gx {

constexpr int kMaxSmem = 227 * 1024;  // of a CTA
// Bytes of 16 rows x 128 columns of a 4-bit matrix in the device layout.
constexpr int q4_unit_bytes(uint32_t type) { return type == GX_Q4_0 ? 1152 : 1280; }

// Activations of a unit: two tiles of 64 columns (two groups), [N rows][128 B] in the 128-byte swizzle, row
// t + TP p part p of token t, a group's 8 columns of q as the 16-byte chunk 4 (group & 1) + q in the order
// (0,4) (1,5) (2,6) (3,7), as a word of codes is unpacked; Q4_1: a third tile, chunk j the group sums of group
// j in three parts, as m multiplies them.
template <uint32_t TYPE, bool XB, int TP>
struct Tc {
    static constexpr int N = XB ? TP : 3 * TP;
    static constexpr int BU = N * 128 * (TYPE == GX_Q4_1 ? 3 : 2);         // a unit's activations
    static constexpr int STAGE = BU + 8 * q4_unit_bytes(TYPE);              // and the codes of 8 row tiles
    static constexpr int XS = (kMaxSmem - 4096) / STAGE < 6 ? (kMaxSmem - 4096) / STAGE : 6;
    static constexpr int SLOTS = N <= 96 ? 2 : 1, SLOT = (N + 31) / 32 * 32;  // accumulators, their TMEM columns
    static constexpr int AC = TYPE == GX_Q4_1 ? 144 : 128;                  // TMEM columns of a unit's weights
    static constexpr int AS = (512 - SLOTS * SLOT) / AC;                    // stages of those
    // A wait by parity holds only if the turn before of the same stage is known to be complete. Of the weights'
    // stages a set of decoders knows that by the MMA of its unit before, if there are no more sets than stages.
    // Of the copies' stages it knows it where each of them is one set's own. Elsewhere (copies that another set
    // waits for may land later than its own) it waits for its stage of weights first: that stage is free once
    // the MMA of the unit AS before is complete, and with it every copy up to that unit's. The other order has
    // the codes in registers by then: Q4_1, 64 bf16 tokens by 8192 x 8192 take 34.1 us with it and 36.2 without.
    static constexpr int RING = XS < AS ? XS : AS, SETS = RING < 3 ? RING : 3;
    static constexpr bool FREE_FIRST = XS % SETS != 0;
    static_assert(SETS <= AS && (!FREE_FIRST || AS <= XS), "parities of the rings");
    static constexpr int THREADS = (6 + 4 * SETS) * 32;
    static constexpr int BARS = XS * STAGE;
    static constexpr int BYTES = BARS + 512 + 1024;                         // and the alignment
};

}  // namespace gx
