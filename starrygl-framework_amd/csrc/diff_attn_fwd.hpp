// Forward kernels of differential attention on the matrix units.
//
// A wave takes query rows of one head and ONE of the two maps, the queries as the COLUMNS of its products: S^T = K_m Q_m^T has
// its keys in registers and one query per lane, so the softmax's running maximum and sum are one number per lane, and P^T is
// already laid out as the right operand of O^T += V^T P^T.  The two waves of a row group share the staged keys and values
// and join their maps at the end.  Rows of different sequences share a tile: every column has its own span of keys, and
// the tile walks the union (which for ascending pointers is one run).
//
// One query per sequence over a long history (no q_ptr): the query heads of a group are the columns, and the two row groups take
// every other sub-tile of keys.
#pragma once

#include "diff_attn.hpp"

namespace sgl {
namespace attn {
namespace {

template <typename T, int DP>
struct Shape {
    static constexpr int RB = 2 * DP * (int)sizeof(T);          // bytes of a staged row, of keys and of values
    static constexpr int BN = 32768 / (2 * RB) >= 64 ? 64 : 32; // keys of a tile
    static constexpr int TILE = 2 * BN * RB;
    static constexpr int EP = Mat<T>::EP;
    static constexpr int QS = DP / (2 * EP);                    // steps over a half of a head
    static constexpr int PS = 32 / (2 * EP);                    // steps over 32 keys
    static constexpr int VT = 2 * DP / 32;                      // 32-wide tiles of the values
    // column tiles of a wave: with two, every fragment read from LDS feeds two products (16-bit types are bound by LDS reads
    // with one); the 128-wide heads have no registers for them, and fp32's products are slow enough without
    static constexpr int RT = sizeof(T) == 2 && DP <= 64 ? 2 : 1;
    static constexpr int ROWS = 2 * 32 * RT;                    // rows of a block
};

// A maximum may grow by this much (powers of two) before the sums and results are rescaled to it: probabilities stay below
// 2^8, and most tiles leave the 2 DP / 32 x 16 multiplications of every column tile out.
constexpr float SLACK = 8.f;

template <typename T, int DP, int RT>
struct State {
    f32x16 o[RT][Shape<T, DP>::VT];
    float m[RT], l[RT];
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            m[c] = NEG_INF;
            l[c] = 0.f;
#pragma unroll
            for (int t = 0; t < Shape<T, DP>::VT; ++t) o[c][t] = zero16();
        }
    }
    // whether something that is not a number got into a column that sees any key.  A value that is not finite, in a key that
    // the column does not see, enters as 0 * NaN or 0 * inf; the pass is then done again key by key.
    __device__ __forceinline__ bool spoilt(const Span (&span)[RT]) const {
        bool bad = false;
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            bool b = false;
#pragma unroll
            for (int t = 0; t < Shape<T, DP>::VT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) b = b || o[c][t][r] != o[c][t][r];
            bad = bad || (b && span[c].lo < span[c].hi);
        }
        return bad;
    }
};

// one sub-tile of 32 keys
template <typename T, int DP, int RT, bool CAREFUL>
__device__ __forceinline__ void step(State<T, DP, RT>& st, const typename Mat<T>::Frag (&q)[RT][Shape<T, DP>::QS], const char* ktile, const char* vtile, int sub,
                                     int map, int32_t j0, bool all, const Span (&span)[RT], const AttnArgs& g, int lane) {
    typedef Shape<T, DP> S;
    typedef Mat<T> M;
    constexpr int RB = S::RB;
    const int half = lane >> 5, col = lane & 31;
    f32x16 s[RT];
#pragma unroll
    for (int c = 0; c < RT; ++c) s[c] = zero16();
    // a half of a head is RB / 2 bytes: RB / 32 chunks, whole pieces of 8 or (64-byte halves) half a piece
    const char* kmap = RB >= 256 ? ktile + map * (RB / 256) * 1024 : ktile;
#pragma unroll
    for (int i = 0; i < S::QS; ++i) {
        typename M::Frag k;
        if constexpr (RB >= 256) k = row_frag<T, RB>(kmap, sub * 32, col, i, half);
        else k = map ? row_frag<T, RB>(kmap, sub * 32, col, i + 2, half) : row_frag<T, RB>(kmap, sub * 32, col, i, half);
#pragma unroll
        for (int c = 0; c < RT; ++c) s[c] = M::mma(k, q[c][i], s[c]);
    }
    if (!all) {
#pragma unroll
        for (int c = 0; c < RT; ++c) hide(s[c], j0, half, span[c], g.a.key_mask, (int32_t)g.a.Tk - 1);
    }
    float top[RT];
    bool grows = false;
#pragma unroll
    for (int c = 0; c < RT; ++c) {
        float t = s[c][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) t = fmaxf(t, s[c][r]);
        top[c] = half_max(t) * g.c2;
        grows = grows || top[c] > st.m[c] + SLACK;
    }
    if (__any(grows)) {
#pragma unroll
        for (int c = 0; c < RT; ++c) {
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
    for (int c = 0; c < RT; ++c) {
        const float ms = st.m[c] == NEG_INF ? 0.f : st.m[c];
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[c][r] = exp2_hw(__builtin_fmaf(s[c][r], g.c2, -ms));
            sum += s[c][r];
        }
        st.l[c] += sum;
    }
    if constexpr (!CAREFUL) {
#pragma unroll
        for (int i = 0; i < S::PS; ++i) {
            typename M::Frag p[RT];
#pragma unroll
            for (int c = 0; c < RT; ++c) p[c] = to_frag<T>(s[c], i);
#pragma unroll
            for (int t = 0; t < S::VT; ++t) {
                const typename M::Frag v = col_frag<T, RB>(vtile, sub * 32, i, t, lane);
#pragma unroll
                for (int c = 0; c < RT; ++c) st.o[c][t] = M::mma(v, p[c], st.o[c][t]);
            }
        }
    } else {
        // one key at a time, taken over by the columns that see it
        for (int i = 0; i < S::PS; ++i)
            for (int jj = 0; jj < 2 * S::EP; ++jj) {
                const int hh = jj / S::EP, j = jj % S::EP;
                const int32_t key = j0 + row_of<T>(i, j, hh);
#pragma unroll
                for (int c = 0; c < RT; ++c) {
                    const bool on = sees(key, span[c], g.a.key_mask);
                    typename M::Frag p;
                    float x = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (r == i * S::EP + j) x = s[c][r];
#pragma unroll
                    for (int e = 0; e < S::EP; ++e) p[e] = e == j && half == hh ? (T)x : (T)0.f;
#pragma unroll
                    for (int t = 0; t < S::VT; ++t) {
                        typename M::Frag v = col_frag<T, RB>(vtile, sub * 32, i, t, lane);
#pragma unroll
                        for (int e = 0; e < S::EP; ++e) v[e] = e == j && half == hh ? v[e] : (T)0.f;
                        const f32x16 n = M::mma(v, p, st.o[c][t]);
#pragma unroll
                        for (int r = 0; r < 16; ++r) st.o[c][t][r] = on ? n[r] : st.o[c][t][r];
                    }
                }
            }
    }
}

// HEADS: the columns are the query heads of one key head, all at query `seq`; otherwise 32 RT query rows of one head
template <typename T, int DP, bool HEADS, bool DMA>
__global__ __launch_bounds__(BLOCK, 2) void fwd_kernel(AttnArgs g, FwdWork w) {
    typedef Shape<T, DP> S;
    typedef Mat<T> M;
    constexpr int RB = S::RB, BN = S::BN, RT = HEADS ? 1 : S::RT;
    __shared__ __align__(16) char s_a[S::TILE];
    __shared__ __align__(16) char s_b[S::TILE];
    __shared__ int s_lo[2], s_hi[2], s_bad;
    const sgl_diff_attn_args& a = g.a;
    const int G = a.Hq / a.Hk;
    const int64_t item = xcd_item(w.items);
    if (item >= w.items) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int map = wave & 1, group = wave >> 1;
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int split = (int)(item % w.splits);
    int64_t rest = item / w.splits;

    int hk, h[RT];
    int64_t i[RT];
    Span span[RT];
    bool mine[RT];              // the column is a row of the result
#pragma unroll
    for (int c = 0; c < RT; ++c) span[c] = Span{0, 0};
    if constexpr (HEADS) {
        const int cg = (int)(rest % w.groups);
        rest /= w.groups;
        hk = (int)(rest % a.Hk);
        i[0] = rest / a.Hk;
        const int32_t seq = i[0] < B ? (int32_t)i[0] : -1;
        mine[0] = cg * 32 + col < G && (seq >= 0 || (a.flags & SGL_ATTN_ZERO_REST));
        h[0] = hk * G + (cg * 32 + col < G ? cg * 32 + col : 0);
        if (cg * 32 + col < G) span[0] = keys_of(a, seq, i[0]);
    } else {
        // the heads of a group next to each other (they read the same keys); of a causal call the long rows first
        const int hg = (int)(rest % G);
        rest /= G;
        hk = (int)(rest / w.tiles);
        int32_t tile = (int32_t)(rest % w.tiles);
        if (a.causal) tile = w.tiles - 1 - tile;
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            h[c] = hk * G + hg;
            i[c] = (int64_t)tile * S::ROWS + group * 32 * RT + c * 32 + col;
            const int32_t seq = i[c] >= a.Tq ? -1 : a.q_ptr ? find_seq(a.q_ptr, B, i[c]) : (i[c] < B ? (int32_t)i[c] : -1);
            span[c] = keys_of(a, seq, i[c]);
            mine[c] = i[c] < a.Tq && (seq >= 0 || (a.flags & SGL_ATTN_ZERO_REST));
        }
    }
    // the wave's union of spans, and the run that all its columns see
    int32_t ulo = 0x7FFFFFFF, uhi = 0, alo = 0, ahi = 0x7FFFFFFF;
#pragma unroll
    for (int c = 0; c < RT; ++c)
        if (span[c].lo < span[c].hi) ulo = min(ulo, span[c].lo), uhi = max(uhi, span[c].hi), alo = max(alo, span[c].lo), ahi = min(ahi, span[c].hi);
    ulo = wave_min(ulo), uhi = wave_max(uhi), alo = wave_max(alo), ahi = a.key_mask ? 0 : wave_min(ahi);
    if (lane == 0 && map == 0) s_lo[group] = ulo, s_hi[group] = uhi;
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();
    int32_t lo = min(s_lo[0], s_lo[1]), hi = max(s_hi[0], s_hi[1]);
    if (w.splits > 1 && lo < hi) {
        const int32_t chunk = (int32_t)ceil_div<int64_t>(ceil_div<int64_t>((int64_t)hi - lo, w.splits), BN) * BN;
        const int64_t from = (int64_t)lo + (int64_t)chunk * split;
        lo = (int32_t)min(from, (int64_t)hi);
        hi = (int32_t)min(from + chunk, (int64_t)hi);
        uhi = min(uhi, hi), ulo = max(ulo, lo);
#pragma unroll
        for (int c = 0; c < RT; ++c) span[c].lo = max(span[c].lo, lo), span[c].hi = min(span[c].hi, hi);
    }

    typename M::Frag q[RT][S::QS];
#pragma unroll
    for (int c = 0; c < RT; ++c) {
        const bool live = span[c].lo < span[c].hi;
#pragma unroll
        for (int k = 0; k < S::QS; ++k)
            q[c][k] = global_frag<T>(row<T>(a.q, live ? i[c] : 0, 2 * h[c] + map), (2 * k + half) * S::EP, a.D, live, g.aligned, g.negate);
    }
    const Source ks = halves<T>(a.k, hk, a.D), vs = run<T>(a.v, hk, a.Dv);
    const int32_t last = (int32_t)a.Tk - 1;
    State<T, DP, RT> st;
    st.reset();
    auto load = [&](char* buf, int32_t j) {
        stage<T, DP, BN, BLOCK, DMA>(buf, ks, true, j, last, g.aligned);
        stage<T, DP, BN, BLOCK, DMA>(buf + BN * RB, vs, false, j, last, g.aligned);
    };
    auto work = [&](const char* buf, int32_t j) {
#pragma unroll
        for (int sub = 0; sub < BN / 32; ++sub) {
            const int32_t j0 = j + sub * 32;
            if (j0 >= uhi || j0 + 32 <= ulo) continue;
            if (HEADS && (((j0 - lo) >> 5) & 1) != group) continue;
            step<T, DP, RT, false>(st, q, buf, buf + BN * RB, sub, map, j0, j0 >= alo && j0 + 32 <= ahi, span, g, lane);
        }
    };
    if (lo < hi) {
        load(s_a, lo);
        staged();
        for (int32_t j = lo; j < hi; j += 2 * BN) {
            if (j + BN < hi) load(s_b, j + BN);
            work(s_a, j);
            staged();
            if (j + BN >= hi) break;
            if (j + 2 * BN < hi) load(s_a, j + 2 * BN);
            work(s_b, j + BN);
            staged();
        }
        if (st.spoilt(span)) s_bad = 1;
        __syncthreads();
        if (s_bad) {
            st.reset();
            for (int32_t j = lo; j < hi; j += BN) {
                load(s_a, j);
                staged();
                for (int sub = 0; sub < BN / 32; ++sub) {
                    const int32_t j0 = j + sub * 32;
                    if (j0 >= uhi || j0 + 32 <= ulo) continue;
                    if (HEADS && (((j0 - lo) >> 5) & 1) != group) continue;
                    step<T, DP, RT, true>(st, q, s_a, s_a + BN * RB, sub, map, j0, false, span, g, lane);
                }
                __syncthreads();
            }
        }
    }

    if (g.parts > 1) {
        // unnormalised results, to be joined with the other parts'
        const int part = HEADS ? split * 2 + group : split;
#pragma unroll
        for (int c = 0; c < RT; ++c) {
            const float l = half_sum(st.l[c]);
            if (!mine[c]) continue;
            const int64_t at = (((int64_t)part * a.Tq + i[c]) * a.Hq + h[c]) * 2 + map;
            if (half == 0) g.part_ml[2 * at] = st.m[c], g.part_ml[2 * at + 1] = l;
            if (l == 0.f) continue;
            float* o = g.part_o + at * a.Dv;
#pragma unroll
            for (int t = 0; t < S::VT; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int d = t * 32 + 8 * (r / 4) + 4 * half + r % 4;
                    if (d < a.Dv) o[d] = st.o[c][t][r];
                }
        }
        return;
    }
    // normalise; the second map's waves hand their results over, the first's subtract them
#pragma unroll
    for (int c = 0; c < RT; ++c) {
        const float l = half_sum(st.l[c]);
        const bool none = !(span[c].lo < span[c].hi) || l == 0.f;      // no key, or only keys whose score is -inf
        const float inv = none ? 0.f : 1.f / l;
        if (a.lse && half == 0 && mine[c]) a.lse[(i[c] * a.Hq + h[c]) * 2 + map] = none ? INFINITY : st.m[c] + __builtin_amdgcn_logf(l);
#pragma unroll
        for (int t = 0; t < S::VT; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) st.o[c][t][r] = none ? 0.f : st.o[c][t][r] * inv;
    }
    struct alignas(4 * sizeof(T)) Four {
        T e[4];
    };
    constexpr int SLOT = 64 * 16 * 4;                                   // a column tile's 32 x 32 results
    constexpr int AT_ONCE = S::TILE / (2 * SLOT);                       // of them per row group in the first buffer
#pragma unroll
    for (int u0 = 0; u0 < RT * S::VT; u0 += AT_ONCE) {
        __syncthreads();
        char* box = s_a + group * AT_ONCE * SLOT + lane * 16;
        if (map == 1) {
#pragma unroll
            for (int u = u0; u < u0 + AT_ONCE && u < RT * S::VT; ++u)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const f32x16& o = st.o[u / S::VT][u % S::VT];
                    *reinterpret_cast<f32x4*>(box + (u - u0) * SLOT + r4 * 1024) = f32x4{o[4 * r4], o[4 * r4 + 1], o[4 * r4 + 2], o[4 * r4 + 3]};
                }
        }
        __syncthreads();
#pragma unroll
        for (int u = u0; u < u0 + AT_ONCE && u < RT * S::VT; ++u) {
            const int c = u / S::VT, t = u % S::VT;
            if (!mine[c]) continue;
            const sgl_rows& to = map ? a.o2 : a.out;
            if (!to.data) continue;
            T* dst = row_out<T>(to, i[c], h[c]);
            const float lam = a.lam[h[c]];
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                f32x4 o2 = f32x4{0.f, 0.f, 0.f, 0.f};
                if (map == 0) o2 = *reinterpret_cast<const f32x4*>(box + (u - u0) * SLOT + r4 * 1024);
                const int d = t * 32 + 8 * r4 + 4 * half;
                Four y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y.e[e] = (T)(map == 0 ? __builtin_fmaf(-lam, o2[e], st.o[c][t][4 * r4 + e]) : st.o[c][t][4 * r4 + e]);
                if (g.aligned && d + 4 <= a.Dv) {
                    *reinterpret_cast<Four*>(dst + d) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (d + e < a.Dv) dst[d + e] = y.e[e];
                }
            }
        }
    }
}

// joins the parts of a (row, head): one wave each, values dealt to its lanes
template <typename T>
__global__ __launch_bounds__(BLOCK) void join_kernel(AttnArgs g) {
    const sgl_diff_attn_args& a = g.a;
    const int lane = threadIdx.x & 63;
    const int64_t n = a.Tq * a.Hq, at = (int64_t)blockIdx.x * (BLOCK / 64) + (threadIdx.x >> 6);
    if (at >= n) return;
    const int64_t i = at / a.Hq;
    const int h = (int)(at % a.Hq);
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int32_t seq = a.q_ptr ? find_seq(a.q_ptr, B, i) : (i < B ? (int32_t)i : -1);
    if (seq < 0 && !(a.flags & SGL_ATTN_ZERO_REST)) return;
    float o[2][4] = {}, lse[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float top = NEG_INF, sum = 0.f;
        bool nan = false;
        for (int p = lane; p < g.parts; p += 64) {
            const float* ml = g.part_ml + 2 * (((int64_t)p * n + at) * 2 + m);
            if (ml[1] != 0.f) top = fmaxf(top, ml[0]);
            nan = nan || ml[1] != ml[1];
        }
        for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
        for (int p = 0; p < g.parts; ++p) {
            const int64_t k = ((int64_t)p * n + at) * 2 + m;
            const float pm = g.part_ml[2 * k], pl = g.part_ml[2 * k + 1];
            if (pl == 0.f) continue;                // (a part without keys wrote no result)
            const float f = pm == top ? 1.f : exp2_hw(pm - top);
            sum = __builtin_fmaf(pl, f, sum);
            const float* src = g.part_o + k * a.Dv;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (lane + 64 * u < a.Dv) o[m][u] = __builtin_fmaf(src[lane + 64 * u], f, o[m][u]);
        }
        const bool none = sum == 0.f;
        lse[m] = none ? INFINITY : top + __builtin_amdgcn_logf(sum);
#pragma unroll
        for (int u = 0; u < 4; ++u) o[m][u] = none ? 0.f : o[m][u] / sum;
    }
    if (a.lse && lane < 2) a.lse[at * 2 + lane] = lse[lane];
    const float lam = a.lam[h];
    T* out = row_out<T>(a.out, i, h);
    T* out2 = a.o2.data ? row_out<T>(a.o2, i, h) : nullptr;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (lane + 64 * u < a.Dv) {
            out[lane + 64 * u] = (T)__builtin_fmaf(-lam, o[1][u], o[0][u]);
            if (out2) out2[lane + 64 * u] = (T)o[1][u];
        }
}

template <typename T, int DP>
void launch(const AttnArgs& g, hipStream_t st) {
    const FwdWork w = forward_work(g.a);
    const dim3 grid((unsigned)(ceil_div<int64_t>(w.items, 8) * 8)), block(BLOCK);
    const bool dma = g.aligned && g.a.D == DP && g.a.Dv == 2 * DP;
    if (g.a.q_ptr) {
        if (dma) hipLaunchKernelGGL((fwd_kernel<T, DP, false, true>), grid, block, 0, st, g, w);
        else hipLaunchKernelGGL((fwd_kernel<T, DP, false, false>), grid, block, 0, st, g, w);
    } else {
        if (dma) hipLaunchKernelGGL((fwd_kernel<T, DP, true, true>), grid, block, 0, st, g, w);
        else hipLaunchKernelGGL((fwd_kernel<T, DP, true, false>), grid, block, 0, st, g, w);
    }
    if (g.parts > 1)
        hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)ceil_div<int64_t>(g.a.Tq * g.a.Hq, BLOCK / 64)), block, 0, st, g);
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
