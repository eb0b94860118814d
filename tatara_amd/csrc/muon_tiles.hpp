// The tiles of the Newton-Schulz products, and what lies where in a workgroup's LDS.
#pragma once

#include <cstdint>

namespace tatara {

// A workgroup's tile BM x BN of p q^T: WR x WC waves, KS values of k a stage, S
// stages in LDS (KS 16 or more).  KG groups of such waves share a stage's values of k, and their
// sums are joined in order.
template <int BM_, int BN_, int WR_, int WC_, int KS_, int S_, int KG_ = 1>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WR = WR_, WC = WC_, KS = KS_, S = S_, KG = KG_;
    static constexpr int THREADS = KG * WR * WC * 64;
    static constexpr int TM = BM / WR / 32, TN = BN / WC / 32;  // 32 x 32 blocks of a wave
    static constexpr int PIECES = (BM + BN) * (KS / 8) * 2;  // of 16 bytes, of a stage's hi and lo
    static constexpr int LOADS = PIECES / THREADS;            // of a thread
    static_assert(PIECES % THREADS == 0, "every thread loads alike");
};

using Wide = Tile<128, 128, 2, 2, 16, 4>;
using Narrow = Tile<64, 64, 2, 2, 64, 2, 2>;
using Deep = Tile<64, 64, 2, 2, 64, 3, 2>;
using Half = Tile<64, 32, 2, 1, 64, 3, 2>;
using Tiny = Tile<32, 32, 1, 1, 64, 4, 4>;

// The strip of 32 rows that each wave of the first group stores its results through.
template <typename L>
struct StripShape {
    static constexpr int DOWN = L::TM < 2 ? L::TM : 2, OVER = L::TN < 2 ? L::TN : 2;  // blocks of a strip
    static constexpr int PITCH = (DOWN > OVER ? DOWN : OVER) * 32 + 4;
    static constexpr int BYTES = (int)sizeof(float) * 32 * PITCH;
};

// LDS holds the stages; when all are multiplied, the sums of the groups but the
// first and, behind them, a strip a wave.  Sums and strips overlap nowhere: one wave
// may fill its strip while another still reads its sums.
template <typename L>
struct ProductLds {
    static constexpr int WAVES = L::WR * L::WC, QUADS = L::TM * L::TN * 4;  // of a group; four values a lane
    static constexpr int STAGES_BYTES = L::S * L::PIECES * 16;
    static constexpr int SUMS_BYTES = (L::KG - 1) * WAVES * QUADS * 64 * 16;
    static constexpr int LATER_BYTES = SUMS_BYTES + WAVES * StripShape<L>::BYTES;
    static constexpr int BYTES = STAGES_BYTES > LATER_BYTES ? STAGES_BYTES : LATER_BYTES;
    // of a group's, from the second on, the wave's and the lane's four sums; by 16 bytes
    static constexpr uint32_t sum(uint32_t group, uint32_t wave, uint32_t quad, uint32_t lane) {
        return (((group - 1) * WAVES + wave) * QUADS + quad) * 64 + lane;
    }
    // where the wave's strip begins
    static constexpr uint32_t strip(uint32_t wave) { return SUMS_BYTES + wave * StripShape<L>::BYTES; }
    static_assert(L::KG == 1 || 16 * sum(L::KG - 1, WAVES - 1, QUADS - 1, 63) + 16 <= strip(0),
                  "the strips lie behind all sums");
    static_assert(strip(WAVES - 1) + StripShape<L>::BYTES <= BYTES, "the strips lie inside");
};

}  // namespace tatara
