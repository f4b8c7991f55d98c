// Backward kernels of differential attention on the matrix units: one that owns query rows (dQ, and the row sums t_m on the
// way), one that owns keys (dK, dV).  Each computes the probabilities anew from the saved log-sum-exp; nothing is added up
// across blocks but the per-tile sums of d_lam, in tile order, so results do not depend on timing.
//
// Both keep the matrix product that ends in registers as the right operand of the next one: with the owned rows as columns,
// S^T (rows: the walked side) goes through the exponential and is the operand that contracts over the walked side.  The left
// operands come from LDS, by rows for S and dP, transposed for the gradients.
#pragma once

#include "diff_attn.hpp"

namespace sgl {
namespace attn {
namespace {

template <typename T, int DP>
struct Shape {
    static constexpr int RB = 2 * DP * (int)sizeof(T);          // bytes of a staged row
    static constexpr int EP = Mat<T>::EP;
    static constexpr int QS = DP / (2 * EP);                    // steps over a half of a head
    static constexpr int VS = 2 * QS;                           // steps over the values
    static constexpr int PS = 32 / (2 * EP);                    // steps over 32 walked rows
    static constexpr int DT = DP / 32, VT = 2 * DP / 32;        // 32-wide tiles of a half, of the values
    // operands of the owned side: in registers while the kernel fits them there beside its sums, else as fragments read
    // from a tile of their own in LDS
    static constexpr bool OWN_REGS = RB <= 256;
    static constexpr bool VAL_REGS = RB <= 512;
    // waves of a block: as many as the owned side's tiles leave room for in 160 KB
    static constexpr int NW = RB <= 512 ? 4 : 1;
    static constexpr int OWN = (OWN_REGS ? 0 : RB) + (VAL_REGS ? 0 : RB);       // bytes of an owned row in LDS
    static constexpr bool TWO = RB <= 512;                      // two buffers of the walked side
};

struct No {
    static constexpr bool value = false;
};
struct Yes {
    static constexpr bool value = true;
};

__device__ __forceinline__ float signed_c2(const AttnArgs& g) { return g.scale < 0.f ? -g.c2 : g.c2; }

// left operand with one live element in each row: element j of the lanes of `half`
template <typename T>
__device__ __forceinline__ typename Mat<T>::Frag only(typename Mat<T>::Frag f, int j, bool on) {
#pragma unroll
    for (int e = 0; e < Mat<T>::EP; ++e) f[e] = e == j && on ? f[e] : (T)0.f;
    return f;
}

template <int N>
__device__ __forceinline__ bool any_nan(const f32x16 (&x)[N]) {
    bool b = false;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) b = b || x[t][r] != x[t][r];
    return b;
}

template <typename T, int N>
__device__ __forceinline__ void store_cols(const f32x16 (&x)[N], T* dst, int len, float scale, int half, int aligned) {
    struct alignas(4 * sizeof(T)) Four {
        T e[4];
    };
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int d = t * 32 + 8 * r4 + 4 * half;
            Four y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y.e[e] = (T)(x[t][4 * r4 + e] * scale);
            if (aligned && d + 4 <= len) {
                *reinterpret_cast<Four*>(dst + d) = y;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d + e < len) dst[d + e] = y.e[e];
            }
        }
}

// acc[t] += (transposed rows row0.. of the tile, elements from 32 (t0 + t)) * x, x the results of 32 walked rows; careful: one
// walked row at a time, taken over by the columns for which `on(row)` holds
template <typename T, int RB, int N, bool CAREFUL, typename On>
__device__ __forceinline__ void add_product(f32x16 (&acc)[N], const char* tile, int row0, int t0, const f32x16& x, int lane, On on) {
    typedef Mat<T> M;
    constexpr int PS = 32 / (2 * M::EP);
    if constexpr (!CAREFUL) {
#pragma unroll
        for (int i = 0; i < PS; ++i) {
            const typename M::Frag p = to_frag<T>(x, i);
#pragma unroll
            for (int t = 0; t < N; ++t) acc[t] = M::mma(col_frag<T, RB>(tile, row0, i, t0 + t, lane), p, acc[t]);
        }
    } else {
        const int half = lane >> 5;
        for (int i = 0; i < PS; ++i)
            for (int jj = 0; jj < 2 * M::EP; ++jj) {
                const int hh = jj / M::EP, j = jj % M::EP;
                const bool take = on(row_of<T>(i, j, hh));
                float v = 0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (r == i * M::EP + j) v = x[r];
                typename M::Frag p;
#pragma unroll
                for (int e = 0; e < M::EP; ++e) p[e] = e == j && half == hh ? (T)v : (T)0.f;
#pragma unroll
                for (int t = 0; t < N; ++t) {
                    const f32x16 n = M::mma(only<T>(col_frag<T, RB>(tile, row0, i, t0 + t, lane), j, half == hh), p, acc[t]);
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[t][r] = take ? n[r] : acc[t][r];
                }
            }
    }
}

// scores of 32 walked rows against the owned columns, both halves of the head
template <typename T, int DP>
__device__ __forceinline__ void scores(f32x16 (&s)[2], const char* walked, int row0, const typename Mat<T>::Frag (&own)[2][Shape<T, DP>::QS], const char* own_tile,
                                       int own_row, int lane) {
    typedef Shape<T, DP> S;
    constexpr int RB = S::RB;
    const int half = lane >> 5, col = lane & 31;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        s[m] = zero16();
#pragma unroll
        for (int i = 0; i < S::QS; ++i) {
            const typename Mat<T>::Frag w = row_frag<T, RB>(walked, row0, col, m * S::QS + i, half);
            if constexpr (S::OWN_REGS) s[m] = Mat<T>::mma(w, own[m][i], s[m]);
            else s[m] = Mat<T>::mma(w, row_frag<T, RB>(own_tile, own_row, col, m * S::QS + i, half), s[m]);
        }
    }
}

// dP of 32 walked rows against the owned columns
template <typename T, int DP>
__device__ __forceinline__ f32x16 value_product(const char* walked, int row0, const typename Mat<T>::Frag (&own)[Shape<T, DP>::VS], const char* own_tile, int own_row,
                                                int lane) {
    typedef Shape<T, DP> S;
    constexpr int RB = S::RB;
    const int half = lane >> 5, col = lane & 31;
    f32x16 s = zero16();
#pragma unroll
    for (int i = 0; i < S::VS; ++i) {
        const typename Mat<T>::Frag w = row_frag<T, RB>(walked, row0, col, i, half);
        if constexpr (S::VAL_REGS) s = Mat<T>::mma(w, own[i], s);
        else s = Mat<T>::mma(w, row_frag<T, RB>(own_tile, own_row, col, i, half), s);
    }
    return s;
}

// ---------------------------------------------------------------------------------------------- owned: query rows
template <typename T, int DP, bool DMA>
__global__ __launch_bounds__((Shape<T, DP>::NW * 64), (Shape<T, DP>::RB <= 256 ? 2 : 1)) void bwd_q_kernel(AttnArgs g, int32_t tiles) {
    typedef Shape<T, DP> S;
    typedef Mat<T> M;
    constexpr int RB = S::RB, NT = S::NW * 64, ROWS = S::NW * 32;
    constexpr int BN = 32768 / (2 * RB) >= 64 ? 64 : 32, TILE = 2 * BN * RB;
    __shared__ __align__(16) char s_a[TILE];
    __shared__ __align__(16) char s_b[S::TWO ? TILE : 16];
    __shared__ __align__(16) char s_own[S::OWN ? ROWS * S::OWN : 16];
    __shared__ int s_lo[S::NW], s_hi[S::NW], s_bad;
    __shared__ float s_lam[S::NW];
    const sgl_diff_attn_args& a = g.a;
    const int G = a.Hq / a.Hk;
    const int64_t n = (int64_t)tiles * a.Hq, item = xcd_item(n);
    if (item >= n) return;
    const int hg = (int)(item % G);
    const int64_t rest = item / G;
    const int hk = (int)(rest / tiles), h = hk * G + hg;
    int32_t tile = (int32_t)(rest % tiles);
    if (a.causal) tile = tiles - 1 - tile;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int64_t i = (int64_t)tile * ROWS + wave * 32 + col;
    const int32_t seq = i >= a.Tq ? -1 : a.q_ptr ? find_seq(a.q_ptr, B, i) : (i < B ? (int32_t)i : -1);
    const Span span = keys_of(a, seq, i);
    const bool live = span.lo < span.hi;
    if (h == 0 && half == 0 && i < a.Tq) g.spans[2 * i] = span.lo, g.spans[2 * i + 1] = span.hi;
    const int32_t ulo = wave_min(live ? span.lo : 0x7FFFFFFF), uhi = wave_max(live ? span.hi : 0);
    const int32_t alo = wave_max(live ? span.lo : 0), ahi = a.key_mask ? 0 : wave_min(live ? span.hi : 0x7FFFFFFF);
    if (lane == 0) s_lo[wave] = ulo, s_hi[wave] = uhi;
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();
    int32_t lo = s_lo[0], hi = s_hi[0];
#pragma unroll
    for (int w = 1; w < S::NW; ++w) lo = min(lo, s_lo[w]), hi = max(hi, s_hi[w]);

    // t_m = sum over the values of d_out * o_m, with o_1 = out + lam o_2
    const float lam = a.lam[h];
    typename M::Frag q[2][S::QS], go[S::VS];
    float t[2] = {0.f, 0.f}, lse[2] = {INFINITY, INFINITY};
    {
        const int64_t ii = live ? i : 0;
        if constexpr (S::OWN_REGS) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int k = 0; k < S::QS; ++k) q[m][k] = global_frag<T>(row<T>(a.q, ii, 2 * h + m), (2 * k + half) * S::EP, a.D, live, g.aligned, false);
        }
#pragma unroll
        for (int k = 0; k < S::VS; ++k) {
            const int e = (2 * k + half) * S::EP;
            const typename M::Frag d = global_frag<T>(row<T>(a.d_out, ii, h), e, a.Dv, live, g.aligned, false);
            const typename M::Frag y = global_frag<T>(row<T>(a.out, ii, h), e, a.Dv, live, g.aligned, false);
            const typename M::Frag y2 = global_frag<T>(row<T>(a.o2, ii, h), e, a.Dv, live, g.aligned, false);
#pragma unroll
            for (int j = 0; j < S::EP; ++j) {
                const float dj = (float)d[j], o2 = (float)y2[j];
                t[1] = __builtin_fmaf(dj, o2, t[1]);
                t[0] = __builtin_fmaf(dj, __builtin_fmaf(lam, o2, (float)y[j]), t[0]);
            }
            if constexpr (S::VAL_REGS) go[k] = d;
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            t[m] = half_sum(t[m]);
            if (live) lse[m] = a.lse[(i * a.Hq + h) * 2 + m];
            if (i < a.Tq && half == 0) g.delta[(i * a.Hq + h) * 2 + m] = t[m];
        }
    }
    const Source ks = halves<T>(a.k, hk, a.D), vs = run<T>(a.v, hk, a.Dv);
    const int32_t last = (int32_t)a.Tk - 1;
    if constexpr (!S::OWN_REGS) {
        stage<T, DP, ROWS, NT, false>(s_own, halves<T>(a.q, h, a.D), true, tile * ROWS, (int32_t)a.Tq - 1, g.aligned);
        if constexpr (!S::VAL_REGS) stage<T, DP, ROWS, NT, false>(s_own + ROWS * RB, run<T>(a.d_out, h, a.Dv), false, tile * ROWS, (int32_t)a.Tq - 1, g.aligned);
    }
    f32x16 dq[2][S::DT];
    float sum2 = 0.f;           // sum of P_2 dP: -d_lam's share
    auto clear = [&]() {
        sum2 = 0.f;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < S::DT; ++d) dq[m][d] = zero16();
    };
    clear();
    const float c2 = signed_c2(g);
    auto load = [&](char* buf, int32_t j) {
        stage<T, DP, BN, NT, DMA>(buf, ks, true, j, last, g.aligned);
        stage<T, DP, BN, NT, DMA>(buf + BN * RB, vs, false, j, last, g.aligned);
    };
    auto step = [&](const char* buf, int32_t j0, int sub, auto careful) {
        constexpr bool CAREFUL = decltype(careful)::value;
        f32x16 s[2];
        scores<T, DP>(s, buf, sub * 32, q, s_own, wave * 32, lane);
        const f32x16 dp = value_product<T, DP>(buf + BN * RB, sub * 32, go, s_own + ROWS * RB, wave * 32, lane);
        const bool all = !CAREFUL && j0 >= alo && j0 + 32 <= ahi;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float p0 = exp2_hw(__builtin_fmaf(s[0][r], c2, -lse[0])), p1 = exp2_hw(__builtin_fmaf(s[1][r], c2, -lse[1]));
            float x = dp[r];
            if (!all) {
                const int32_t j = j0 + 8 * (r / 4) + 4 * half + r % 4;
                const bool see = j >= span.lo && j < span.hi && (a.key_mask == nullptr || a.key_mask[j < last ? j : last]);
                p0 = see ? p0 : 0.f, p1 = see ? p1 : 0.f, x = see ? x : 0.f;
            }
            s[0][r] = p0 * (x - t[0]);
            const float y = p1 * x;
            sum2 += y;
            s[1][r] = -lam * __builtin_fmaf(-p1, t[1], y);
        }
        auto on = [&](int r) { return sees(j0 + r, span, a.key_mask); };
        add_product<T, RB, S::DT, CAREFUL>(dq[0], buf, sub * 32, 0, s[0], lane, on);
        add_product<T, RB, S::DT, CAREFUL>(dq[1], buf, sub * 32, S::DT, s[1], lane, on);
    };
    auto work = [&](const char* buf, int32_t j) {
#pragma unroll
        for (int sub = 0; sub < BN / 32; ++sub) {
            const int32_t j0 = j + sub * 32;
            if (j0 >= uhi || j0 + 32 <= ulo) continue;
            step(buf, j0, sub, No{});
        }
    };
    if (lo < hi) {
        load(s_a, lo);
        staged();
        if constexpr (S::TWO) {
            for (int32_t j = lo; j < hi; j += 2 * BN) {
                if (j + BN < hi) load(s_b, j + BN);
                work(s_a, j);
                staged();
                if (j + BN >= hi) break;
                if (j + 2 * BN < hi) load(s_a, j + 2 * BN);
                work(s_b, j + BN);
                staged();
            }
        } else {
            for (int32_t j = lo; j < hi; j += BN) {
                if (j > lo) {
                    load(s_a, j);
                    staged();
                }
                work(s_a, j);
                __syncthreads();
            }
        }
        if ((any_nan(dq[0]) || any_nan(dq[1]) || sum2 != sum2) && live) s_bad = 1;
        __syncthreads();
        if (s_bad) {
            clear();
            for (int32_t j = lo; j < hi; j += BN) {
                load(s_a, j);
                staged();
                for (int sub = 0; sub < BN / 32; ++sub) {
                    const int32_t j0 = j + sub * 32;
                    if (j0 >= uhi || j0 + 32 <= ulo) continue;
                    step(s_a, j0, sub, Yes{});
                }
                __syncthreads();
            }
        }
    }
    float share = live ? sum2 : 0.f;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) share += __shfl_xor(share, m);
    if (lane == 0) s_lam[wave] = share;
    __syncthreads();
    if (threadIdx.x == 0) {
        float x = 0.f;
        for (int w = 0; w < S::NW; ++w) x += s_lam[w];
        g.lam_part[(int64_t)tile * a.Hq + h] = x;
    }
    if (i >= a.Tq || (seq < 0 && !(a.flags & SGL_ATTN_ZERO_REST))) return;
    const float scale = live ? g.scale : 0.f;
    if (!live) clear();
#pragma unroll
    for (int m = 0; m < 2; ++m) store_cols<T>(dq[m], row_out<T>(a.d_q, i, 2 * h + m), a.D, scale, half, g.aligned);
}

// ----------------------------------------------------------------------------------------------------- owned: keys
template <typename T, int DP, bool DMA>
__global__ __launch_bounds__((Shape<T, DP>::NW * 64), 1) void bwd_kv_kernel(AttnArgs g, int32_t tiles, int32_t row_tiles) {
    typedef Shape<T, DP> S;
    typedef Mat<T> M;
    constexpr int RB = S::RB, NT = S::NW * 64, ROWS = S::NW * 32;
    constexpr int BQ = 32, TILE = 2 * BQ * RB;
    constexpr int STAT = BQ * 6 * 4;                            // lse, t (two each) and span of a row
    __shared__ __align__(16) char s_a[TILE + STAT];
    __shared__ __align__(16) char s_b[S::TWO ? TILE + STAT : 16];
    __shared__ __align__(16) char s_own[S::OWN ? ROWS * S::OWN : 16];
    __shared__ int s_lo[S::NW], s_hi[S::NW], s_bad;
    __shared__ float s_sum[NT];
    const sgl_diff_attn_args& a = g.a;
    const int G = a.Hq / a.Hk;
    const int64_t n = (int64_t)tiles * a.Hk;
    if ((int64_t)blockIdx.x >= ceil_div<int64_t>(n, 8) * 8) {
        // the last Hq blocks: d_lam of a head
        const int h = (int)(blockIdx.x - ceil_div<int64_t>(n, 8) * 8);
        float x = 0.f;
        for (int k = threadIdx.x; k < row_tiles; k += NT) x += g.lam_part[(int64_t)k * a.Hq + h];
        s_sum[threadIdx.x] = x;
        __syncthreads();
        if (threadIdx.x == 0) {
            float y = 0.f;
            for (int k = 0; k < NT; ++k) y += s_sum[k];
            a.d_lam[h] = -y;
        }
        return;
    }
    const int64_t per = ceil_div<int64_t>(n, 8), item = ((int64_t)blockIdx.x % 8) * per + blockIdx.x / 8;
    if (item >= n) return;
    const int hk = (int)(item / tiles);
    const int32_t tile = (int32_t)(item % tiles);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int64_t j = (int64_t)tile * ROWS + wave * 32 + col;
    const int32_t seq = j >= a.Tk ? -1 : find_seq(a.k_ptr, B, j);
    // the query rows that may see the key
    int32_t qlo = 0, qhi = 0;
    bool shown = seq >= 0 && (a.key_mask == nullptr || a.key_mask[j]);
    if (shown) {
        const int64_t q0 = a.q_ptr ? clamp_to(a.q_ptr[seq], a.Tq) : seq, q1 = a.q_ptr ? clamp_to(a.q_ptr[seq + 1], a.Tq) : seq + 1;
        int64_t from = q0, to = q1;
        if (a.causal) {
            const int64_t with = q1 - (clamp_to(a.k_ptr[seq + 1], a.Tk) - j);      // the query that stands where the key does
            if (with > from) from = with;
            if (a.window > 0 && with + a.window < to) to = with + a.window;
        }
        if (from < to) qlo = (int32_t)from, qhi = (int32_t)to;
    }
    shown = qlo < qhi;
    const int32_t wlo = wave_min(shown ? qlo : 0x7FFFFFFF), whi = wave_max(shown ? qhi : 0);
    if (lane == 0) s_lo[wave] = wlo, s_hi[wave] = whi;
    if (threadIdx.x == 0) s_bad = 0;
    __syncthreads();
    int32_t lo = s_lo[0], hi = s_hi[0];
#pragma unroll
    for (int w = 1; w < S::NW; ++w) lo = min(lo, s_lo[w]), hi = max(hi, s_hi[w]);
    // a wave whose 32 keys are all live may take the short way where every row of a tile sees all of them
    const int32_t key0 = (int32_t)(tile * ROWS + wave * 32);
    const bool whole = __all(shown);

    typename M::Frag k[2][S::QS], v[S::VS];
    {
        const int64_t jj = j < a.Tk ? j : 0;
        if constexpr (S::OWN_REGS) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < S::QS; ++e) k[m][e] = global_frag<T>(row<T>(a.k, jj, 2 * hk + m), (2 * e + half) * S::EP, a.D, shown, g.aligned, false);
        }
        if constexpr (S::VAL_REGS) {
#pragma unroll
            for (int e = 0; e < S::VS; ++e) v[e] = global_frag<T>(row<T>(a.v, jj, hk), (2 * e + half) * S::EP, a.Dv, shown, g.aligned, false);
        }
    }
    if constexpr (!S::OWN_REGS) {
        stage<T, DP, ROWS, NT, false>(s_own, halves<T>(a.k, hk, a.D), true, tile * ROWS, (int32_t)a.Tk - 1, g.aligned);
        if constexpr (!S::VAL_REGS) stage<T, DP, ROWS, NT, false>(s_own + ROWS * RB, run<T>(a.v, hk, a.Dv), false, tile * ROWS, (int32_t)a.Tk - 1, g.aligned);
    }
    f32x16 dk[2][S::DT], dv[S::VT];
    auto clear = [&]() {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < S::DT; ++d) dk[m][d] = zero16();
#pragma unroll
        for (int d = 0; d < S::VT; ++d) dv[d] = zero16();
    };
    clear();
    const int32_t last = (int32_t)a.Tq - 1;
    const float c2 = signed_c2(g);
    const int32_t steps = lo < hi ? (hi - lo + BQ - 1) / BQ * G : 0;       // head by head, row tile by row tile
    const int32_t per_head = G > 0 ? steps / G : 0;
    auto load = [&](char* buf, int32_t s) {
        const int h = hk * G + s / per_head;
        const int32_t i0 = lo + s % per_head * BQ;
        stage<T, DP, BQ, NT, DMA>(buf, halves<T>(a.q, h, a.D), true, i0, last, g.aligned);
        stage<T, DP, BQ, NT, DMA>(buf + BQ * RB, run<T>(a.d_out, h, a.Dv), false, i0, last, g.aligned);
        // 64 numbers each: (lse_1, lse_2), (t_1, t_2) and (lo, hi) of the rows
        for (int w = wave; w < 3; w += S::NW) {
            const int32_t i = min(i0 + (lane >> 1), last);
            const char* src = w == 0 ? reinterpret_cast<const char*>(a.lse + ((int64_t)i * a.Hq + h) * 2 + (lane & 1))
                            : w == 1 ? reinterpret_cast<const char*>(g.delta + ((int64_t)i * a.Hq + h) * 2 + (lane & 1))
                                     : reinterpret_cast<const char*>(g.spans + 2 * (int64_t)i + (lane & 1));
            const int ww = __builtin_amdgcn_readfirstlane(w);
            __builtin_amdgcn_global_load_lds((SGL_GLOBAL void*)src, (SGL_LDS void*)(buf + TILE + ww * 256), 4, 0, 0);
        }
    };
    auto step = [&](const char* buf, int32_t s0, auto careful) {
        constexpr bool CAREFUL = decltype(careful)::value;
        const int h = hk * G + s0 / per_head;
        const int32_t i0 = lo + s0 % per_head * BQ;
        if (i0 >= whi || i0 + BQ <= wlo) return;
        const float lam = a.lam[h];
        const float* stat = reinterpret_cast<const float*>(buf + TILE);
        const int2* spans = reinterpret_cast<const int2*>(buf + TILE + 512);
        const int2 mine = spans[col];
        const bool all = !CAREFUL && whole && i0 + BQ <= hi && __all(mine.x <= key0 && mine.y >= key0 + 32);
        f32x16 s[2];
        scores<T, DP>(s, buf, 0, k, s_own, wave * 32, lane);
        f32x16 dp = value_product<T, DP>(buf + BQ * RB, 0, v, s_own + ROWS * RB, wave * 32, lane);
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const int r0 = 8 * r4 + 4 * half;
            f32x4 l[2], t[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                l[u] = *reinterpret_cast<const f32x4*>(stat + 2 * (r0 + 2 * u));
                t[u] = *reinterpret_cast<const f32x4*>(stat + 64 + 2 * (r0 + 2 * u));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * r4 + e;
                float p0 = exp2_hw(__builtin_fmaf(s[0][r], c2, -l[e / 2][2 * (e % 2)])), p1 = exp2_hw(__builtin_fmaf(s[1][r], c2, -l[e / 2][2 * (e % 2) + 1]));
                float x = dp[r], t0 = t[e / 2][2 * (e % 2)], t1 = t[e / 2][2 * (e % 2) + 1];
                if (!all) {
                    const int2 sp = spans[r0 + e];
                    const bool see = shown && i0 + r0 + e < hi && j >= sp.x && j < sp.y;
                    p0 = see ? p0 : 0.f, p1 = see ? p1 : 0.f, x = see ? x : 0.f, t0 = see ? t0 : 0.f, t1 = see ? t1 : 0.f;
                }
                p1 *= -lam;
                s[0][r] = p0 * (x - t0);
                s[1][r] = p1 * (x - t1);
                dp[r] = p0 + p1;
            }
        }
        auto on = [&](int r) { return shown && i0 + r < hi && j >= spans[r].x && j < spans[r].y; };
        add_product<T, RB, S::VT, CAREFUL>(dv, buf + BQ * RB, 0, 0, dp, lane, on);
        add_product<T, RB, S::DT, CAREFUL>(dk[0], buf, 0, 0, s[0], lane, on);
        add_product<T, RB, S::DT, CAREFUL>(dk[1], buf, 0, S::DT, s[1], lane, on);
    };
    if (steps > 0) {
        if constexpr (S::TWO) {
            load(s_a, 0);
            staged();
            for (int32_t s = 0; s < steps; s += 2) {
                if (s + 1 < steps) load(s_b, s + 1);
                step(s_a, s, No{});
                staged();
                if (s + 1 >= steps) break;
                if (s + 2 < steps) load(s_a, s + 2);
                step(s_b, s + 1, No{});
                staged();
            }
        } else {
            for (int32_t s = 0; s < steps; ++s) {
                load(s_a, s);
                staged();
                step(s_a, s, No{});
                __syncthreads();
            }
        }
        if ((any_nan(dk[0]) || any_nan(dk[1]) || any_nan(dv)) && shown) s_bad = 1;
        __syncthreads();
        if (s_bad) {
            clear();
            for (int32_t s = 0; s < steps; ++s) {
                load(s_a, s);
                staged();
                step(s_a, s, Yes{});
                __syncthreads();
            }
        }
    }
    if (j >= a.Tk || (seq < 0 && !(a.flags & SGL_ATTN_ZERO_REST))) return;
    if (!shown) clear();
#pragma unroll
    for (int m = 0; m < 2; ++m) store_cols<T>(dk[m], row_out<T>(a.d_k, j, 2 * hk + m), a.D, shown ? g.scale : 0.f, half, g.aligned);
    store_cols<T>(dv, row_out<T>(a.d_v, j, hk), a.Dv, 1.f, half, g.aligned);
}

template <typename T, int DP>
void launch(const AttnArgs& g, hipStream_t st) {
    const sgl_diff_attn_args& a = g.a;
    constexpr int NT = Shape<T, DP>::NW * 64, ROWS = Shape<T, DP>::NW * 32;
    const int32_t qt = (int32_t)ceil_div<int64_t>(a.Tq, ROWS), kt = (int32_t)ceil_div<int64_t>(a.Tk, ROWS);
    const bool dma = g.aligned && a.D == DP && a.Dv == 2 * DP;
    if (qt > 0) {
        const dim3 grid((unsigned)(ceil_div<int64_t>((int64_t)qt * a.Hq, 8) * 8)), block(NT);
        if (dma) hipLaunchKernelGGL((bwd_q_kernel<T, DP, true>), grid, block, 0, st, g, qt);
        else hipLaunchKernelGGL((bwd_q_kernel<T, DP, false>), grid, block, 0, st, g, qt);
    }
    const dim3 grid((unsigned)(ceil_div<int64_t>((int64_t)kt * a.Hk, 8) * 8 + a.Hq)), block(NT);
    if (dma) hipLaunchKernelGGL((bwd_kv_kernel<T, DP, true>), grid, block, 0, st, g, kt, qt);
    else hipLaunchKernelGGL((bwd_kv_kernel<T, DP, false>), grid, block, 0, st, g, kt, qt);
}

}  // namespace

template <typename T>
void backward_type(const AttnArgs& g, hipStream_t st) {
    const int need = heads_width(g.a);
    if (need <= 32) launch<T, 32>(g, st);
    else if (need <= 64) launch<T, 64>(g, st);
    else launch<T, 128>(g, st);
}

}  // namespace attn
}  // namespace sgl
