// Forward kernels of differential attention on the matrix units.
//
// A wave takes 32 query rows of one head as the COLUMNS of its products: S_m^T = K_m Q_m^T has its keys in registers and one
// query per lane, so the softmax's running maximum and sum are one number per lane and map, and P^T is already laid out as
// the right operand of O^T += V^T P^T.  Rows of different sequences share a tile: every column has its own span of keys, and
// the tile walks the union (which for ascending pointers is one run).
//
// Heads up to 64 wide (16-bit; fp32 up to 32) keep both maps in one wave, and a fragment of the values feeds both.  Wider ones have no registers for
// that: two waves take a map each and join at the end.
//
// One query per sequence over a long history (no q_ptr): the query heads of a group are the columns, a map to a wave, and two
// groups of waves take every other sub-tile of keys.
//
// Probabilities are rounded to the inputs' type for their product with the values (the matrix units take no other): by at most
// h = 2^-8 in bf16 (2^-11 in fp16) of each, once; their sum is taken before.  Sums, maxima and results are fp32.  Over 4096 keys
// each map is off by 0.0017 in bf16 (2-norm; by 0.0002 in fp16), out, a difference of two that have the values' mean in common, by
// 0.0025 where rounding the exact result alone gives 0.0017.  P in two operands would take that away for half as many products again.
//
// Bound by the matrix and vector instructions, which overlap between the two waves of a SIMD only in part (a tile of 32 x 32: 768
// cycles of products, about 720 of vector instructions, 2000 measured).  8 sequences of 2048, 16 heads over 4, 64 wide, causal,
// bf16: 270 us, 0.76 PFLOP/s; 2 of 4096, 8 over 2, 128 wide: 405 us, 1.02 PFLOP/s; with both maps' results kept for a backward call
// 315 and 440 us.  Tiles of 32 keys: 277 us for the first; the exponentials of one map between the products of the other, which
// reads the values twice: 288 us.  Single queries are bound by the keys' bytes: 16 histories of up to 32768 keys, 16 heads over 4, 117 us, 4.7 TB/s (a copy reaches 5.0).
#pragma once

#include "diff_attn.hpp"

namespace sgl {
namespace attn {
namespace {

template <typename T, int DP, bool HEADS>
struct Shape {
    static constexpr int RB = 2 * DP * (int)sizeof(T);          // bytes of a staged row, of keys and of values
    static constexpr int MAPS = !HEADS && RB <= 256 ? 2 : 1;    // of a wave
    static constexpr int WAVES = HEADS || MAPS == 2 ? 4 : 8, GROUPS = WAVES * MAPS / 2, NT = WAVES * 64;
    static constexpr int BN = RB <= 256 ? 64 : 32;    // keys of a tile
    static constexpr int TILE = 2 * BN * RB;
    static constexpr int EP = Mat<T>::EP;
    static constexpr int QS = DP / (2 * EP);                    // steps over a half of a head
    static constexpr int PS = 32 / (2 * EP);                    // steps over 32 keys
    static constexpr int VT = 2 * DP / 32;                      // 32-wide tiles of the values
    static constexpr int ROWS = GROUPS * 32;                    // query rows of a block
};

// A maximum may grow by this much (powers of two) before the sums and results are rescaled to it: probabilities stay below
// 2^8, and most tiles leave the 2 DP / 32 x 16 multiplications of every column tile out.
constexpr float SLACK = 8.f;

template <typename T, int DP, int MAPS>
struct State {
    static constexpr int VT = 2 * DP / 32;
    f32x16 o[MAPS][VT];
    float m[MAPS], l[MAPS];
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int c = 0; c < MAPS; ++c) {
            m[c] = NEG_INF;
            l[c] = 0.f;
#pragma unroll
            for (int t = 0; t < VT; ++t) o[c][t] = zero16();
        }
    }
    // whether something that is not a number got in: a value that is not finite, in a key that the column does not see, enters as
    // 0 * NaN or 0 * inf.  The keys are then gone through again without such values.
    __device__ __forceinline__ bool spoilt() const {
        bool bad = false;
#pragma unroll
        for (int c = 0; c < MAPS; ++c)
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) bad = bad || o[c][t][r] != o[c][t][r];
        return bad;
    }
};

// one sub-tile of 32 keys; map0: the first of the wave's maps
template <typename T, int DP, int MAPS>
__device__ __forceinline__ void step(State<T, DP, MAPS>& st, const typename Mat<T>::Frag (&q)[MAPS][Shape<T, DP, false>::QS], const char* ktile, const char* vtile, int sub,
                                     int map0, int32_t j0, bool all, Span span, const AttnArgs& g, int lane) {
    typedef Shape<T, DP, false> S;
    typedef Mat<T> M;
    constexpr int RB = S::RB;
    const int half = lane >> 5, col = lane & 31;
    constexpr int AHEAD = MAPS == 2 || RB > 512 ? 2 : 4;        // (each feeds MAPS products of the values)
    f32x16 s[MAPS];
#pragma unroll
    for (int c = 0; c < MAPS; ++c) s[c] = zero16();
    // (the maps take turns: products into one sum follow each other at a distance)
    auto load_k = [&](int n) { return map_frag<T, RB>(ktile, sub * 32, col, MAPS == 2 ? n & 1 : map0, n / MAPS, half); };
    auto load_v = [&](int n) { return col_frag<T, RB>(vtile, sub * 32, n / S::VT, n % S::VT, lane); };
    Pipe<T, MAPS * S::QS, AHEAD> keys_ahead;
    keys_ahead.fill(load_k);
    keys_ahead.drain(load_k, [&](int n, const typename M::Frag& k) { s[n % MAPS] = M::mma(k, q[n % MAPS][n / MAPS], s[n % MAPS]); });
    // the first values are on their way while the probabilities are formed
    Pipe<T, S::PS * S::VT, AHEAD> values_ahead;
    values_ahead.fill(load_v);
    if (!all) {
        const uint32_t see = (span_bits(j0, span) & mask_bits(g.a.key_mask, j0, lane, (int32_t)g.a.Tk - 1)) >> (4 * half);
#pragma unroll
        for (int c = 0; c < MAPS; ++c)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[c][r] = row_bit(see, r) ? s[c][r] : NEG_INF;
    }
    float top[MAPS];
    bool grows = false;
#pragma unroll
    for (int c = 0; c < MAPS; ++c) {
        float t = s[c][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) t = fmaxf(t, s[c][r]);
        top[c] = half_max(t) * g.c2;
        grows = grows || top[c] > st.m[c] + SLACK;
    }
    if (__any(grows)) {
#pragma unroll
        for (int c = 0; c < MAPS; ++c) {
            const float mn = fmaxf(st.m[c], top[c]);
            const float f = mn == NEG_INF ? 1.f : exp2_hw(st.m[c] - mn);
            st.m[c] = mn;
            st.l[c] *= f;
#pragma unroll
            for (int t = 0; t < S::VT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) st.o[c][t][r] *= f;
        }
    }
#pragma unroll
    for (int c = 0; c < MAPS; ++c) {
        const float ms = st.m[c] == NEG_INF ? 0.f : st.m[c];
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[c][r] = exp2_hw(__builtin_fmaf(s[c][r], g.c2, -ms));
            sum += s[c][r];
        }
        st.l[c] += sum;
    }
    typename M::Frag p[MAPS];
    values_ahead.drain(load_v, [&](int n, const typename M::Frag& v) {
#pragma unroll
        for (int c = 0; c < MAPS; ++c) {
            if (n % S::VT == 0) p[c] = to_frag<T>(s[c], n / S::VT);
            st.o[c][n % S::VT] = M::mma(v, p[c], st.o[c][n % S::VT]);
        }
    });
}

// the results of a column as they are
template <int VT, bool WHOLE>
__device__ __forceinline__ void store_map(const f32x16 (&x)[VT], float* to, int Dv, int half) {
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = t * 32 + 8 * r4 + 4 * half;
            const f32x4 y = {x[t][4 * r4], x[t][4 * r4 + 1], x[t][4 * r4 + 2], x[t][4 * r4 + 3]};
            if (WHOLE || Dv % 4 == 0) {
                if (d < Dv) *reinterpret_cast<f32x4*>(to + d) = y;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < Dv) to[d + e] = y[e];
            }
        }
}

// HEADS: the columns are the query heads of one key head, all at query `seq`; otherwise 32 query rows of one head.  KEEP: the
// results of both maps are kept as they are too (in kernels of their own: the stores cost a forward pass that keeps nothing
// registers, 248 us instead of 226 for 32 ragged histories of up to 2048, 8 heads of 64, causal, fp16)
template <typename T, int DP, bool HEADS, int MODE, bool KEEP>
__global__ __launch_bounds__((Shape<T, DP, HEADS>::NT), (HEADS && Shape<T, DP, HEADS>::RB > 512 ? 1 : 2)) void fwd_kernel(AttnArgs g, FwdWork w) {
    typedef Shape<T, DP, HEADS> S;
    typedef Mat<T> M;
    constexpr int RB = S::RB, BN = S::BN, MAPS = S::MAPS, VT = S::VT;
    constexpr bool WHOLE = MODE == WHOLE_ROWS;
    __shared__ __align__(16) char s_a[S::TILE];
    __shared__ __align__(16) char s_b[S::TILE];
    __shared__ __align__(8) uint8_t s_marks[BN * (RB / 16)];
    __shared__ int s_lo[S::GROUPS], s_hi[S::GROUPS], s_bad;
    const sgl_diff_attn_args& a = g.a;
    const int G = a.Hq / a.Hk;
    // parts of a history in turn over the 8 XCDs: nothing is shared between them, and histories differ in length (as neighbours on one
    // XCD, 16 of up to 32768 keys took 140 us instead of 117)
    const uint32_t item = HEADS ? (uint32_t)g.first + blockIdx.x : xcd_item(g, (uint32_t)w.items);
    if (item >= w.items) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int map0 = MAPS == 2 ? 0 : wave & 1, group = MAPS == 2 ? wave : wave >> 1;
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int split = (int)(item % (uint32_t)w.splits);
    uint32_t rest = item / (uint32_t)w.splits;

    int hk, h;
    int32_t i, i0 = 0, seq;     // the lane's query row, the wave's first
    bool mine;                  // the column is a row of the result
    if constexpr (HEADS) {
        const int cg = (int)(rest % (uint32_t)w.groups);
        rest /= (uint32_t)w.groups;
        hk = (int)(rest % (uint32_t)a.Hk);
        i = (int32_t)(rest / (uint32_t)a.Hk);
        seq = i < B ? i : -1;
        mine = cg * 32 + col < G;
        h = hk * G + (mine ? cg * 32 + col : 0);
    } else {
        // the heads of a group next to each other (they read the same keys); of a causal call the long rows first
        const int hg = (int)(rest % (uint32_t)G);
        rest /= (uint32_t)G;
        hk = (int)(rest / (uint32_t)w.tiles);
        int32_t tile = (int32_t)(rest % (uint32_t)w.tiles);
        if (a.causal) tile = w.tiles - 1 - tile;
        h = hk * G + hg;
        i0 = tile * S::ROWS + group * 32;
        i = i0 + col;
        mine = i < a.Tq;
        const int32_t at[1] = {col};
        int32_t found[1];
        find_seqs<1>(a.q_ptr, B, i0, at, found);
        seq = found[0];
    }
    Span span = keys_of(a, mine ? seq : -1, i);
    // (in flight until the first tile is there)
    typename M::Frag q[MAPS][S::QS];
#pragma unroll
    for (int c = 0; c < MAPS; ++c)
#pragma unroll
        for (int k = 0; k < S::QS; ++k)
            q[c][k] = global_frag<T, WHOLE>(row<T>(a.q, mine ? i : 0, 2 * h + map0 + c), (2 * k + half) * S::EP, a.D, g.grain);
    mine = mine && (seq >= 0 || (a.flags & SGL_ATTN_ZERO_REST));
    Reach reach = reach_of(span);
    if (a.key_mask) reach.to = 0;
    if (lane == 0 && (MAPS == 2 || map0 == 0)) s_lo[group] = reach.lo, s_hi[group] = reach.hi;
    if (threadIdx.x == 0) s_bad = 0;
    clear_image<MODE, S::TILE, S::NT>(s_a);
    clear_image<MODE, S::TILE, S::NT>(s_b);
    __syncthreads();
    int32_t lo = s_lo[0], hi = s_hi[0];
#pragma unroll
    for (int k = 1; k < S::GROUPS; ++k) lo = min(lo, s_lo[k]), hi = max(hi, s_hi[k]);
    if (w.splits > 1 && lo < hi) {
        const int32_t chunk = (int32_t)ceil_div<int64_t>(ceil_div<int64_t>((int64_t)hi - lo, w.splits), BN) * BN;
        const int64_t from = (int64_t)lo + (int64_t)chunk * split;
        lo = (int32_t)min(from, (int64_t)hi);
        hi = (int32_t)min(from + chunk, (int64_t)hi);
        reach.hi = min(reach.hi, hi), reach.lo = max(reach.lo, lo);
        span.lo = max(span.lo, lo), span.hi = min(span.hi, hi);
    }
    const Source ks = halves<T>(a.k, hk, a.D), vs = run<T>(a.v, hk, a.Dv);
    const int32_t last = (int32_t)a.Tk - 1;
    State<T, DP, MAPS> st;
    st.reset();
    Stager<T, DP, BN, S::NT, MODE, true> stage_k;
    Stager<T, DP, BN, S::NT, MODE, false> stage_v;
    stage_k.plan(ks);
    stage_v.plan(vs);
    bool finite = false;        // the pass without what is not finite
    auto load = [&](char* buf, int32_t j) {
        stage_k.load(buf, ks, j, last, g.grain);
        if (finite) stage_finite<T, DP, BN, S::NT>(buf + BN * RB, s_marks, vs, false, j, last);
        else stage_v.load(buf + BN * RB, vs, j, last, g.grain);
    };
    auto work = [&](const char* buf, int32_t j) {
#pragma unroll
        for (int sub = 0; sub < BN / 32; ++sub) {
            const int32_t j0 = j + sub * 32;
            if (j0 >= reach.hi || j0 + 32 <= reach.lo) continue;
            if (HEADS && (((j0 - lo) >> 5) & (S::GROUPS - 1)) != group) continue;
            step<T, DP, MAPS>(st, q, buf, buf + BN * RB, sub, map0, j0, j0 >= reach.from && j0 + 32 <= reach.to, span, g, lane);
        }
    };
    if (lo < hi) {
        load(s_a, lo);
        if (g.negate) {
#pragma unroll
            for (int c = 0; c < MAPS; ++c)
#pragma unroll
                for (int k = 0; k < S::QS; ++k) q[c][k] = -q[c][k];
        }
#pragma unroll 1
        for (;;) {
            staged();
#pragma unroll 1
            for (int32_t j = lo; j < hi; j += 2 * BN) {
                if (j + BN < hi) load(s_b, j + BN);
                work(s_a, j);
                staged();
                if (j + BN >= hi) break;
                if (j + 2 * BN < hi) load(s_a, j + 2 * BN);
                work(s_b, j + BN);
                staged();
            }
            if (finite) break;
            if (st.spoilt() && span.lo < span.hi) s_bad = 1;
            __syncthreads();
            if (!s_bad) break;
            finite = true;
            st.reset();
            load(s_a, lo);
        }
        if (finite) {
            // the queries that see what is not finite get NaN
#pragma unroll 1
            for (int32_t j = lo; j < hi; j += BN) {
                __syncthreads();
                stage_finite<T, DP, BN, S::NT>(s_a, s_marks, vs, false, j, last);
                __syncthreads();
#pragma unroll 1
                for (int r = 0; r < BN && j + r < hi; ++r) {
                    if (HEADS && (((j + r - lo) >> 5) & (S::GROUPS - 1)) != group) continue;
                    if (!marked_any<RB>(s_marks, r, 0, RB / 16)) continue;
                    if (!sees(j + r, span, a.key_mask)) continue;
#pragma unroll
                    for (int c = 0; c < MAPS; ++c) spoil<T, RB, VT>(st.o[c], s_marks, r, half);
                }
            }
            __syncthreads();
        }
    }

    if (HEADS || g.parts > 1) {
        // unnormalised results, to be joined with the other parts'; a column without keys here (sum -1, no result) has gathered what
        // the others of its wave see, where they see all of a tile
        const int part = HEADS ? split * 2 + group : split;
#pragma unroll
        for (int c = 0; c < MAPS; ++c) {
            const float l = half_sum(st.l[c]);
            const bool none = !(span.lo < span.hi);
            if (!mine) continue;
            const int64_t at = (((int64_t)part * a.Tq + i) * a.Hq + h) * 2 + map0 + c;
            if (half == 0) g.part_ml[2 * at] = st.m[c], g.part_ml[2 * at + 1] = none ? -1.f : l;
            if (none) continue;
            store_map<VT, WHOLE>(st.o[c], g.part_o + at * a.Dv, a.Dv, half);
        }
        return;
    }
    if constexpr (!HEADS) {
        float inv[MAPS];        // 0: no key, or only keys whose score is -inf (what such a column gathered may be anything)
#pragma unroll
        for (int c = 0; c < MAPS; ++c) {
            const float l = half_sum(st.l[c]);
            const bool none = !(span.lo < span.hi) || l == 0.f;
            inv[c] = none ? 0.f : 1.f / l;
            if (a.lse && half == 0 && mine) a.lse[pair_at(a, i, h) + map0 + c] = none ? INFINITY : st.m[c] + __builtin_amdgcn_logf(l);
        }
        const float lam = a.lam[h];
        constexpr int SHARE = S::TILE / (S::WAVES / 2);                     // a wave's part of the two buffers
        char* own = (wave < S::WAVES / 2 ? s_a : s_b) + wave % (S::WAVES / 2) * SHARE;
        const uint32_t keep = (uint32_t)__ballot(mine);
        if constexpr (KEEP || MAPS == 1) {
#pragma unroll
            for (int c = 0; c < MAPS; ++c) {
#pragma unroll
                for (int t = 0; t < VT; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) st.o[c][t][r] = inv[c] == 0.f ? 0.f : st.o[c][t][r] * inv[c];
                // (32 bytes of a row at a time, a cache line in four stores)
                if (KEEP && mine) store_map<VT, WHOLE>(st.o[c], map_row(a, i, h, map0 + c), a.Dv, half);
            }
        }
        if constexpr (MAPS == 2) {
            const auto value = [&](int c, int t, int r) { return KEEP ? st.o[c][t][r] : inv[c] == 0.f ? 0.f : st.o[c][t][r] * inv[c]; };
            store_rows<T, SHARE / 32, VT, WHOLE>([&](int t, int r) { return __builtin_fmaf(-lam, value(1, t, r), value(0, t, r)); }, own, lane, a.Dv, g.grain, row_out<T>(a.out, i0, h),
                                                 a.out.row_stride, keep);
            if (a.o2.data)
                store_rows<T, SHARE / 32, VT, WHOLE>([&](int t, int r) { return value(1, t, r); }, own, lane, a.Dv, g.grain, row_out<T>(a.o2, i0, h), a.o2.row_stride, keep);
        } else {
            // the second map's waves hand their results over, the first's subtract them; a 32 x 32 tile takes 4 KB, half the
            // groups use each buffer
            constexpr int SLOT = 4096, AT_ONCE = S::TILE / (S::GROUPS / 2 * SLOT);
            static_assert(AT_ONCE >= 1, "a result of every group fits");
            char* box = (group < S::GROUPS / 2 ? s_a : s_b) + group % (S::GROUPS / 2) * AT_ONCE * SLOT + lane * 16;
#pragma unroll
            for (int u0 = 0; u0 < VT; u0 += AT_ONCE) {
                __syncthreads();
                if (map0 == 1) {
#pragma unroll
                    for (int u = u0; u < u0 + AT_ONCE && u < VT; ++u)
#pragma unroll
                        for (int r4 = 0; r4 < 4; ++r4) {
                            const f32x16& o = st.o[0][u];
                            *reinterpret_cast<f32x4*>(box + (u - u0) * SLOT + r4 * 1024) = f32x4{o[4 * r4], o[4 * r4 + 1], o[4 * r4 + 2], o[4 * r4 + 3]};
                        }
                }
                __syncthreads();
                if (map0 == 0) {
#pragma unroll
                    for (int u = u0; u < u0 + AT_ONCE && u < VT; ++u)
#pragma unroll
                        for (int r4 = 0; r4 < 4; ++r4) {
                            const f32x4 o2 = *reinterpret_cast<const f32x4*>(box + (u - u0) * SLOT + r4 * 1024);
#pragma unroll
                            for (int e = 0; e < 4; ++e) st.o[0][u][4 * r4 + e] = __builtin_fmaf(-lam, o2[e], st.o[0][u][4 * r4 + e]);
                        }
                }
            }
            __syncthreads();
            const sgl_rows& to = map0 ? a.o2 : a.out;
            if (to.data)
                store_rows<T, SHARE / 32, VT, WHOLE>([&](int t, int r) { return st.o[0][t][r]; }, own, lane, a.Dv, g.grain, row_out<T>(to, i0, h), to.row_stride, keep);
        }
    }
}

// Joins the parts of a (row, head), a block each: the weights of the parts first, then 8 groups of 32 lanes add up every eighth
// part and are themselves added in order.  A part whose weight vanishes beside the others' is added all the same, so that what
// is not finite in it counts.
template <typename T>
__global__ __launch_bounds__(BLOCK) void join_kernel(AttnArgs g) {
    constexpr int MOST = 2 * 64;
    __shared__ float s_f[2][MOST], s_lse[2];
    __shared__ __align__(16) float s_o[2][8][256];
    const sgl_diff_attn_args& a = g.a;
    const int64_t n = a.Tq * a.Hq, at = g.first + blockIdx.x;
    const int64_t i = at / a.Hq;
    const int h = (int)(at - i * a.Hq), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int32_t seq = a.q_ptr ? find_seq(a.q_ptr, B, i) : (i < B ? (int32_t)i : -1);
    if (seq < 0 && !(a.flags & SGL_ATTN_ZERO_REST)) return;
    if (wave < 2) {
        // the parts' maxima and sums of map `wave`: two a lane
        float m[2], l[2], top = NEG_INF, sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int p = lane + 64 * u;
            const float* ml = g.part_ml + 2 * (((int64_t)p * n + at) * 2 + wave);
            m[u] = p < g.parts ? ml[0] : NEG_INF;
            l[u] = p < g.parts ? ml[1] : -1.f;
            if (!(l[u] <= 0.f)) top = fmaxf(top, m[u]);
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float f = l[u] <= 0.f ? 0.f : m[u] == top ? 1.f : exp2_hw(m[u] - top);
            s_f[wave][lane + 64 * u] = f;
            sum += l[u] <= 0.f ? 0.f : l[u] * f;
        }
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int u = 0; u < 2; ++u) s_f[wave][lane + 64 * u] = l[u] < 0.f ? -1.f : s_f[wave][lane + 64 * u] * inv;
        if (lane == 0) {
            s_lse[wave] = sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
            if (a.lse) a.lse[at * 2 + wave] = s_lse[wave];
        }
    }
    __syncthreads();
    const int group = threadIdx.x >> 5, l32 = threadIdx.x & 31;
    const bool vec = a.Dv % 4 == 0;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        for (int p = group; p < g.parts; p += 8) {
            const float f = s_f[m][p];
            if (f < 0.f) continue;                      // (a part without keys wrote no result)
            const float* src = g.part_o + (((int64_t)p * n + at) * 2 + m) * a.Dv;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = 4 * l32 + 128 * u;
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                if (vec) {
                    if (d < a.Dv) x = *reinterpret_cast<const f32x4*>(src + d);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d + e < a.Dv) x[e] = src[d + e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[u][e] = __builtin_fmaf(x[e], f, acc[u][e]);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) *reinterpret_cast<f32x4*>(&s_o[m][group][4 * l32 + 128 * u]) = acc[u];
    }
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= a.Dv) return;
    float o[2] = {0.f, 0.f};
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int k = 0; k < 8; ++k) o[m] += s_o[m][k][d];
    for (int m = 0; m < 2; ++m) o[m] = s_lse[m] == INFINITY ? 0.f : o[m];       // no key, or only scores of -inf
    row_out<T>(a.out, i, h)[d] = (T)__builtin_fmaf(-a.lam[h], o[1], o[0]);
    if (a.o2.data) row_out<T>(a.o2, i, h)[d] = (T)o[1];
    if (a.maps) map_row(a, i, h, 0)[d] = o[0], map_row(a, i, h, 1)[d] = o[1];
}

template <typename T, int DP>
void launch(const AttnArgs& g, hipStream_t st) {
    const FwdWork w = forward_work(g.a);
    const int64_t blocks = ceil_div<int64_t>(w.items, 8) * 8;
    constexpr int ROW_NT = Shape<T, DP, false>::NT, HEAD_NT = Shape<T, DP, true>::NT;
    auto go = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        in_parts(g, blocks, [&](const AttnArgs& part, dim3 grid) {
            if (!g.a.q_ptr) hipLaunchKernelGGL((fwd_kernel<T, DP, true, MODE, false>), grid, dim3(HEAD_NT), 0, st, part, w);
            else if (g.a.maps && g.parts == 1) hipLaunchKernelGGL((fwd_kernel<T, DP, false, MODE, true>), grid, dim3(ROW_NT), 0, st, part, w);
            else hipLaunchKernelGGL((fwd_kernel<T, DP, false, MODE, false>), grid, dim3(ROW_NT), 0, st, part, w);
        });
    };
    const int mode = stage_mode(g, DP, {&g.a.k, &g.a.v});
    if (mode == WHOLE_ROWS) go(Int<WHOLE_ROWS>{});
    else if (mode == PADDED) go(Int<PADDED>{});
    else go(Int<BY_REGISTERS>{});
    if (g.parts > 1)
        in_parts(g, g.a.Tq * g.a.Hq, [&](const AttnArgs& part, dim3 grid) { hipLaunchKernelGGL(join_kernel<T>, grid, dim3(BLOCK), 0, st, part); });
}

}  // namespace

template <typename T>
void forward_type(const AttnArgs& g, hipStream_t st) {
    const int need = heads_width(g.a);
    if (need <= 32) launch<T, 32>(g, st);
    else if (need <= 64) launch<T, 64>(g, st);
    else launch<T, 128>(g, st);
}

}  // namespace attn
}  // namespace sgl
