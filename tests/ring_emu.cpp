// The warps of the 4-bit batch product and the rings between them, as q4_tc_kernel (csrc/gx_q4.cu) runs them, with
// the stage counts of csrc/gx_q4_tc.h: which copies have landed, which codes a decoder reads, which weights and
// activations an MMA multiplies. One step of one role at a time, in an order that a seed picks; the copies of the
// units in `slow` land only when nothing else can move.
#include <stdint.h>

#include <vector>

#include "../gyro-dx_b200/csrc/gx_q4_tc.h"

namespace {

struct Barrier {
    int need = 1, arrived = 0;
    long phase = 0;  // turns that are complete
    void arrive() {
        if (++arrived == need) {
            arrived = 0;
            ++phase;
        }
    }
    // mbarrier.try_wait.parity: the turn before the present one has this parity
    bool passed(int parity) const { return (int)((phase & 1) ^ 1) == parity; }
};

// 0: every unit was read as it should be; 1: a decoder read another unit's codes; 2: an MMA multiplied other
// weights or activations; 3: a stage was written while it was still read; 4: nobody can move.
template <uint32_t TYPE, bool XB, int TP>
int walk(int total, uint64_t slow, uint64_t seed) {
    using C = gx::Tc<TYPE, XB, TP>;
    constexpr int XS = C::XS, AS = C::AS, SETS = C::SETS, W = 4;  // warps of a set
    std::vector<Barrier> full_x(XS), empty_x(XS), full_a(AS), empty_a(AS);
    for (auto &b : full_x) b.need = 3;  // the announcement and two copies
    for (auto &b : full_a) b.need = W;
    std::vector<int> codes(XS, -1), acts(XS, -1);
    std::vector<std::vector<int>> a(AS, std::vector<int>(W, -1));
    struct Copy {
        int unit, stage;
        bool code;
    };
    std::vector<Copy> flying;
    int cn = 0, cstep = 0, prologue = 0;                       // copying thread
    int issued = 0, done = 0;                                   // MMAs in order
    std::vector<int> dn(SETS * W), dstep(SETS * W, 0);          // decoder warps: the unit, where in it
    for (int i = 0; i < SETS * W; ++i) dn[i] = i / W;
    auto rnd = [&](int n) {
        seed = seed * 6364136223846793005ull + 1442695040888963407ull;
        return (int)((seed >> 33) % (uint64_t)n);
    };
    auto copy_codes = [&](int n) {
        full_x[n % XS].arrive();
        flying.push_back({n, n % XS, true});
    };
    auto late = [&](const Copy &c) { return c.unit < 64 && (slow >> c.unit & 1); };
    int bad = 0;
    auto land = [&](size_t i) {
        const Copy c = flying[i];
        flying.erase(flying.begin() + (long)i);
        (c.code ? codes : acts)[c.stage] = c.unit;
        full_x[c.stage].arrive();
    };
    auto move = [&](int who) -> bool {
        if (who == 0) {  // the copying thread
            if (prologue < XS && prologue < total) return copy_codes(prologue++), true;
            if (cn >= total) return false;
            if (cstep == 0) {
                if (cn >= XS) {
                    if (!empty_x[cn % XS].passed((cn / XS & 1) ^ 1)) return false;
                    if (done < cn - XS + 1) bad = 3;
                    copy_codes(cn);
                }
                return cstep = 1, true;
            }
            flying.push_back({cn, cn % XS, false});
            return cstep = 0, ++cn, true;
        }
        if (who == 1) {  // the issuing thread
            if (issued >= total) return false;
            const int n = issued;
            if (!full_x[n % XS].passed(n / XS & 1) || !full_a[n % AS].passed(n / AS & 1)) return false;
            if (codes[n % XS] != n || acts[n % XS] != n) bad = 2;
            for (int w = 0; w < W; ++w)
                if (a[n % AS][w] != n) bad = 2;
            return ++issued, true;
        }
        if (who == 2) {  // the tensor core ends one
            if (done >= issued) return false;
            empty_a[done % AS].arrive();
            empty_x[done % XS].arrive();
            return ++done, true;
        }
        if (who == 3) {  // a copy lands
            std::vector<size_t> can;
            for (size_t i = 0; i < flying.size(); ++i)
                if (!late(flying[i])) can.push_back(i);
            if (can.empty()) return false;
            return land(can[rnd((int)can.size())]), true;
        }
        const int d = who - 4, w = d % W, n = dn[d];
        if (n >= total) return false;
        // a decoder waits for its codes and for its stage of weights, in the order of the header
        const bool free_turn = (dstep[d] == 0) == C::FREE_FIRST;
        if (free_turn) {
            if (!empty_a[n % AS].passed((n / AS & 1) ^ 1)) return false;
            if (done < n - AS + 1) bad = 3;
        } else {
            if (!full_x[n % XS].passed(n / XS & 1)) return false;
            if (codes[n % XS] != n) bad = 1;
        }
        if (dstep[d] == 0) return dstep[d] = 1, true;
        a[n % AS][w] = n;
        full_a[n % AS].arrive();
        dn[d] += SETS;
        return dstep[d] = 0, true;
    };
    while (done < total) {
        bool moved = false;
        const int roles = 4 + SETS * W, first = rnd(roles);
        for (int k = 0; k < roles && !moved; ++k) moved = move((first + k) % roles);
        if (!moved && !flying.empty()) land((size_t)rnd((int)flying.size())), moved = true;
        if (!moved) return 4;
        if (bad) return bad;
    }
    return 0;
}

template <uint32_t TYPE, bool XB>
int walk_tp(int tp, int total, uint64_t slow, uint64_t seed) {
    return tp == 16 ? walk<TYPE, XB, 16>(total, slow, seed)
                    : tp == 32 ? walk<TYPE, XB, 32>(total, slow, seed) : walk<TYPE, XB, 64>(total, slow, seed);
}

}  // namespace

extern "C" int ring_walk(uint32_t type, int xb, int tp, int total, uint64_t slow, uint64_t seed) {
    if (type == GX_Q4_0) return xb ? walk_tp<GX_Q4_0, true>(tp, total, slow, seed) : walk_tp<GX_Q4_0, false>(tp, total, slow, seed);
    return xb ? walk_tp<GX_Q4_1, true>(tp, total, slow, seed) : walk_tp<GX_Q4_1, false>(tp, total, slow, seed);
}
