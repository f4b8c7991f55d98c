// Backward kernels of differential attention on the matrix units: one that owns query rows (dQ, and the row sums t_m on the
// way), one that owns keys (dK, dV).  Each computes the probabilities anew from the saved log-sum-exp; nothing is added up
// across blocks but the per-tile sums of d_lam, in tile order, so results do not depend on timing.
//
// Both keep the matrix product that ends in registers as the right operand of the next one: with the owned rows as columns,
// S^T (rows: the walked side) goes through the exponential and is the operand that contracts over the walked side.  The left
// operands come from LDS, by rows for S and dP, transposed for the gradients.  P_1 - lam P_2 and dS_m are rounded to the inputs'
// type for those products, once each; everything else is fp32.
//
// Bound by the matrix and vector instructions of a wave, which alternate in the order written here.  8 sequences of 2048, 16
// heads over 4, 64 wide, causal, bf16: rows 315 us (0.66 PFLOP/s), keys 455 us (0.60 PFLOP/s); 2 of 4096, 8 over 2, 128 wide:
// 480 us (0.86) and 757 us (0.73).  A map to a wave, dP formed twice: rows 367 and 507 us.  Keys with dK and dV in waves of their
// own, scores formed twice: 525 and 1098 us; a map to a wave, dP twice: 517 and 981 us.
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
    static constexpr int DT = DP / 32, VT = 2 * DP / 32;        // 32-wide tiles of a half, of the values
};

__device__ __forceinline__ float signed_c2(const AttnArgs& g) { return g.scale < 0.f ? -g.c2 : g.c2; }

template <int N>
__device__ __forceinline__ bool any_nan(const f32x16 (&x)[N]) {
    bool b = false;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) b = b || x[t][r] != x[t][r];
    return b;
}

// results of 32 walked rows as right operands
template <typename T>
struct Operand {
    static constexpr int EP = Mat<T>::EP, PS = 32 / (2 * EP);
    typename Mat<T>::Frag f[PS];
    // registers r, r + 1 (r even): rounded as a pair, one instruction
    __device__ __forceinline__ void set2(int r, float x, float y) {
        if constexpr (sizeof(T) == 2) {
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            typedef T pair __attribute__((ext_vector_type(2)));
            typedef uint32_t words __attribute__((ext_vector_type(4)));
            words w = __builtin_bit_cast(words, f[r / EP]);
            w[r % EP / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x, y}), pair));
            f[r / EP] = __builtin_bit_cast(typename Mat<T>::Frag, w);
        } else {
            f[r / EP][r % EP] = x;
            f[r / EP][r % EP + 1] = y;
        }
    }
    __device__ __forceinline__ void mask(uint32_t see) {
        asm volatile("" : "+v"(see));       // (or the 16 bits are kept from one mask to the next, whether there is one or not)
#pragma unroll
        for (int r = 0; r < 16; ++r) f[r / EP][r % EP] = row_bit(see, r) ? f[r / EP][r % EP] : (T)0.f;
    }
};
template <typename T>
__device__ __forceinline__ Operand<T> operand(const f32x16& x) {
    Operand<T> o;
#pragma unroll
    for (int k = 0; k < Operand<T>::PS; ++k) o.f[k] = to_frag<T>(x, k);
    return o;
}

// acc[t] += (transposed rows row0.. of the tile, elements from 32 (t0 + t)) * x
template <typename T, int RB, int N, int AHEAD>
__device__ __forceinline__ void add_product(f32x16 (&acc)[N], const char* tile, int row0, int t0, const Operand<T>& x, int lane) {
    typedef Mat<T> M;
    constexpr int PS = Operand<T>::PS;
    auto load = [&](int n) { return col_frag<T, RB>(tile, row0, n / N, t0 + n % N, lane); };
    Pipe<T, PS * N, AHEAD> ahead;
    ahead.fill(load);
    ahead.drain(load, [&](int n, const typename M::Frag& f) { acc[n % N] = M::mma(f, x.f[n / N], acc[n % N]); });
}

// ---------------------------------------------------------------------------------------------- owned: query rows
// A wave owns 32 rows of a head: both maps' scores, dP and dQ of a tile of 32 keys, the products between the vector
// instructions of the phase before, as above.
template <typename T, int DP>
struct Rows {
    static constexpr int RB = Shape<T, DP>::RB, WAVES = 4, ROWS = QUERY_ROWS, OCC = RB <= 256 ? 2 : 1, AHEAD = RB <= 256 ? 2 : 4;
    static constexpr int BN = RB <= 512 ? 64 : 32, TILE = 2 * BN * RB;
    static_assert(ROWS == WAVES * 32, "the row tiles of the workspace");
};

template <typename T, int DP, int MODE>
__global__ __launch_bounds__((Rows<T, DP>::WAVES * 64), (Rows<T, DP>::OCC)) void bwd_rows_kernel(AttnArgs g, int32_t tiles) {
    typedef Shape<T, DP> S;
    typedef Rows<T, DP> P;
    typedef Mat<T> M;
    constexpr int RB = S::RB, NT = P::WAVES * 64, BN = P::BN, AHEAD = P::AHEAD;
    __shared__ __align__(16) char s_a[P::TILE];
    __shared__ __align__(16) char s_b[P::TILE];
    __shared__ __align__(8) uint8_t s_marks[2 * BN * (RB / 16)];
    __shared__ int s_lo[P::WAVES], s_hi[P::WAVES], s_bad;
    __shared__ float s_lam[P::WAVES];
    const sgl_diff_attn_args& a = g.a;
    const int G = a.Hq / a.Hk;
    const uint32_t n = (uint32_t)tiles * (uint32_t)a.Hq, item = xcd_item(g, n);
    if (item >= n) return;
    const int hg = (int)(item % (uint32_t)G);
    const uint32_t rest = item / (uint32_t)G;
    const int hk = (int)(rest / (uint32_t)tiles), h = hk * G + hg;
    int32_t tile = (int32_t)(rest % (uint32_t)tiles);
    if (a.causal) tile = tiles - 1 - tile;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int32_t i0 = tile * P::ROWS + wave * 32, i = i0 + col;
    const int32_t at[1] = {col};
    int32_t found[1];
    find_seqs<1>(a.q_ptr, B, i0, at, found);
    const int32_t seq = i >= a.Tq ? -1 : found[0];
    const Span span = keys_of(a, seq, i);
    const bool live = span.lo < span.hi;
    Reach reach = reach_of(span);
    if (a.key_mask) reach.to = 0;
    if (lane == 0) s_lo[wave] = reach.lo, s_hi[wave] = reach.hi;
    if (threadIdx.x == 0) s_bad = 0;
    clear_image<MODE, P::TILE, NT>(s_a);
    clear_image<MODE, P::TILE, NT>(s_b);
    __syncthreads();
    int32_t lo = s_lo[0], hi = s_hi[0];
#pragma unroll
    for (int w = 1; w < P::WAVES; ++w) lo = min(lo, s_lo[w]), hi = max(hi, s_hi[w]);

    // t_m = sum over the values of d_out * o_m: of the unrounded results if they were kept, or with o_1 = out + lam o_2
    const float lam = a.lam[h];
    typename M::Frag q[2][S::QS], go[S::VS];
    float t[2] = {0.f, 0.f};
    const int64_t ii = i < a.Tq ? i : 0;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int k = 0; k < S::QS; ++k) q[m][k] = global_frag<T, MODE == WHOLE_ROWS>(row<T>(a.q, ii, 2 * h + m), (2 * k + half) * S::EP, a.D, g.grain);
#pragma unroll
    for (int k = 0; k < S::VS; ++k) go[k] = global_frag<T, MODE == WHOLE_ROWS>(row<T>(a.d_out, ii, h), (2 * k + half) * S::EP, a.Dv, g.grain);
    if (a.maps) {
#pragma unroll
        for (int k = 0; k < S::VS; ++k)
#pragma unroll
            for (int m = 0; m < 2; ++m) t[m] = dot_map<T, MODE == WHOLE_ROWS>(go[k], map_row(a, ii, h, m), (2 * k + half) * S::EP, a.Dv, g.map_grain, t[m]);
    } else {
#pragma unroll
        for (int k = 0; k < S::VS; ++k) {
            const int e = (2 * k + half) * S::EP;
            const typename M::Frag y2 = global_frag<T, MODE == WHOLE_ROWS>(row<T>(a.o2, ii, h), e, a.Dv, g.grain);
            const typename M::Frag y = global_frag<T, MODE == WHOLE_ROWS>(row<T>(a.out, ii, h), e, a.Dv, g.grain);
#pragma unroll
            for (int j = 0; j < S::EP; ++j) {
                t[0] = __builtin_fmaf((float)go[k][j], __builtin_fmaf(lam, (float)y2[j], (float)y[j]), t[0]);
                t[1] = __builtin_fmaf((float)go[k][j], (float)y2[j], t[1]);
            }
        }
    }
    float lse[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        t[m] = half_sum(t[m]);
        lse[m] = live ? a.lse[pair_at(a, i, h) + m] : INFINITY;
    }
    if (i < a.Tq && half == 0) g.delta[pair_at(a, i, h)] = t[0], g.delta[pair_at(a, i, h) + 1] = t[1];

    const Source ks = halves<T>(a.k, hk, a.D), vs = run<T>(a.v, hk, a.Dv);
    const int32_t last = (int32_t)a.Tk - 1;
    f32x16 dq[2][S::DT];
    float sum = 0.f;            // sum of P_2 dP: -d_lam's share
    auto clear = [&]() {
        sum = 0.f;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < S::DT; ++d) dq[m][d] = zero16();
    };
    clear();
    const float c2 = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(signed_c2(g))));
    Stager<T, DP, BN, NT, MODE, true> stage_k;
    Stager<T, DP, BN, NT, MODE, false> stage_v;
    stage_k.plan(ks);
    stage_v.plan(vs);
    bool finite = false;        // the pass without what is not finite
    auto load = [&](char* buf, int32_t j) {
        if (finite) {
            stage_finite<T, DP, BN, NT>(buf, s_marks, ks, true, j, last);
            stage_finite<T, DP, BN, NT>(buf + BN * RB, s_marks + BN * (RB / 16), vs, false, j, last);
        } else {
            stage_k.load(buf, ks, j, last, g.grain);
            stage_v.load(buf + BN * RB, vs, j, last, g.grain);
        }
    };
    // (the lane's parts of the addresses, as of the keys' kernel)
    int32_t by_row[4], by_col[2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        by_row[e] = lane_row<RB>(col, e, half);
        asm volatile("" : "+v"(by_row[e]));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        by_col[e] = lane_col<T, RB>(e, lane);
        asm volatile("" : "+v"(by_col[e]));
    }
    auto of_row = [](const char* base, const int32_t (&by)[4], int k) { return *reinterpret_cast<const typename M::Frag*>(base + (k >> 2) * 1024 + by[k & 3]); };
    auto work = [&](const char* buf, int32_t j) {
#pragma unroll
        for (int sub = 0; sub < BN / 32; ++sub) {
            const int32_t j0 = j + sub * 32;
            if (j0 >= reach.hi || j0 + 32 <= reach.lo) continue;
            constexpr int PS = Operand<T>::PS, QS = S::QS, NK = S::DT * PS, N1 = QS, N2 = 2 * QS, N3 = N2 + S::VS, N4 = N3 + NK, N5 = N4 + NK;
            const char* kt = buf + sub * 32 * RB;
            const char* vt = buf + (BN + sub * 32) * RB;
            const bool some = !(j0 >= reach.from && j0 + 32 <= reach.to);
            uint32_t see = 0;
            if (some) see = (span_bits(j0, span) & mask_bits(a.key_mask, j0, lane, last)) >> (4 * half);
            auto hide = [&](f32x16& x) {
                uint32_t bits = see;
                asm volatile("" : "+v"(bits));
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = row_bit(bits, r) ? x[r] : 0.f;
            };
            f32x16 s[2], dp;
            s[0] = s[1] = dp = zero16();
            Operand<T> ds[2];
            auto load_n = [&](int n) {
                if (n < N2) return of_row(kt, by_row, n);
                if (n < N3) return of_row(vt, by_row, n - N2);
                const int m = n < N4 ? 0 : 1, u = n - (m ? N4 : N3);
                return col_at<T, RB>(kt, by_col, 0, u / S::DT, m * S::DT + u % S::DT);
            };
            auto exps = [&](int m, int r) {
#pragma unroll
                for (int e = r; e < r + 2; ++e) s[m][e] = exp2_hw(__builtin_fmaf(s[m][e], c2, -lse[m]));
            };
            auto scores = [&](int m, int r) { ds[m].set2(r, s[m][r] * (dp[r] - t[m]), s[m][r + 1] * (dp[r + 1] - t[m])); };
            Pipe<T, N5, AHEAD> ahead;
            ahead.fill(load_n);
            ahead.template part<0, N1>(load_n, [&](int n, const typename M::Frag& x) { s[0] = M::mma(x, q[0][n], s[0]); });
            ahead.template part<N1, N2>(load_n, [&](int n, const typename M::Frag& x) {
                s[1] = M::mma(x, q[1][n - N1], s[1]);
#pragma unroll
                for (int r = 8 * (n - N1) / QS * 2; r < 8 * (n - N1 + 1) / QS * 2; r += 2) exps(0, r);
            });
            ahead.template part<N2, N3>(load_n, [&](int n, const typename M::Frag& x) {
                dp = M::mma(x, go[n - N2], dp);
#pragma unroll
                for (int r = 8 * (n - N2) / S::VS * 2; r < 8 * (n - N2 + 1) / S::VS * 2; r += 2) exps(1, r);
            });
            if (some) hide(s[0]), hide(s[1]);
#pragma unroll
            for (int r = 0; r < 16; r += 2) scores(0, r);
            float part = 0.f;       // (of the 32 keys: a sum of sums is off by less)
            ahead.template part<N3, N4>(load_n, [&](int n, const typename M::Frag& x) {
                const int u = n - N3;
                dq[0][u % S::DT] = M::mma(x, ds[0].f[u / S::DT], dq[0][u % S::DT]);
#pragma unroll
                for (int r = 8 * u / NK * 2; r < 8 * (u + 1) / NK * 2; r += 2) {
                    part = __builtin_fmaf(s[1][r], dp[r], part);
                    part = __builtin_fmaf(s[1][r + 1], dp[r + 1], part);
                    scores(1, r);           // (times -lam at the end)
                }
            });
            sum += part;
            ahead.template part<N4, N5>(load_n, [&](int n, const typename M::Frag& x) {
                const int u = n - N4;
                dq[1][u % S::DT] = M::mma(x, ds[1].f[u / S::DT], dq[1][u % S::DT]);
            });
        }
    };
    bool spoilt[2] = {false, false};        // the query sees something not finite: NaN
    if (lo < hi) {
#pragma unroll 1
        for (;;) {
            load(s_a, lo);
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
            if ((any_nan(dq[0]) || any_nan(dq[1]) || sum != sum) && live) s_bad = 1;
            __syncthreads();
            if (!s_bad) break;
            finite = true;
            clear();
        }
        if (finite) {
            // the queries that see what is not finite get NaN
#pragma unroll 1
            for (int32_t j = lo; j < hi; j += BN) {
                __syncthreads();
                stage_finite<T, DP, BN, NT>(s_a, s_marks, ks, true, j, last);
                stage_finite<T, DP, BN, NT>(s_b, s_marks + BN * (RB / 16), vs, false, j, last);
                __syncthreads();
#pragma unroll 1
                for (int r = 0; r < BN && j + r < hi; ++r) {
                    if (!sees(j + r, span, a.key_mask)) continue;
                    const bool o = marked_any<RB>(s_marks + BN * (RB / 16), r, 0, RB / 16);
                    spoilt[0] = spoilt[0] || o || marked_any<RB>(s_marks, r, 0, RB / 32);
                    spoilt[1] = spoilt[1] || o || marked_any<RB>(s_marks, r, RB / 32, RB / 16);
                }
            }
            if (spoilt[1]) sum = NAN;
        }
    }
    float share = live ? sum : 0.f;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) share += __shfl_xor(share, m);
    if (lane == 0) s_lam[wave] = share;
    __syncthreads();
    if (threadIdx.x == 0) {
        float x = 0.f;
        for (int w = 0; w < P::WAVES; ++w) x += s_lam[w];
        g.lam_part[(int64_t)tile * a.Hq + h] = x;
    }
    const uint32_t keep = (uint32_t)__ballot(i < a.Tq && (seq >= 0 || (a.flags & SGL_ATTN_ZERO_REST)));
    // (every wave's last look at the tiles lies before the barrier above)
    char* box = (wave & 1 ? s_b : s_a) + (wave >> 1) * (P::TILE / 2);
    constexpr int PIECE = RB / 2;                               // bytes of a row at a time
    const float f0 = g.scale, f1 = -lam * g.scale;
    store_rows<T, PIECE, S::DT, MODE == WHOLE_ROWS>([&](int d, int r) { return spoilt[0] ? NAN : live ? dq[0][d][r] * f0 : 0.f; }, box, lane, a.D, g.grain, row_out<T>(a.d_q, i0, 2 * h),
                                     a.d_q.row_stride, keep);
    store_rows<T, PIECE, S::DT, MODE == WHOLE_ROWS>([&](int d, int r) { return spoilt[1] ? NAN : live ? dq[1][d][r] * f1 : 0.f; }, box, lane, a.D, g.grain, row_out<T>(a.d_q, i0, 2 * h + 1),
                                     a.d_q.row_stride, keep);
}

// the query rows that may see key j0 + col, and its sequence; shown: some do
__device__ __forceinline__ Span rows_of(const sgl_diff_attn_args& a, int32_t B, int32_t j0, int32_t col, bool& shown, int32_t& seq) {
    const int32_t j = j0 + col;
    const int32_t at[1] = {col};
    int32_t found[1];
    find_seqs<1>(a.k_ptr, B, j0, at, found);
    seq = j >= a.Tk ? -1 : found[0];
    Span rows{0, 0};
    if (seq >= 0 && (a.key_mask == nullptr || a.key_mask[j])) {
        const int64_t q0 = a.q_ptr ? clamp_to(a.q_ptr[seq], a.Tq) : seq, q1 = a.q_ptr ? clamp_to(a.q_ptr[seq + 1], a.Tq) : seq + 1;
        int64_t from = q0, to = q1;
        if (a.causal) {
            const int64_t with = q1 - (clamp_to(a.k_ptr[seq + 1], a.Tk) - j);      // the query that stands where the key does
            if (with > from) from = with;
            if (a.window > 0 && with + a.window < to) to = with + a.window;
        }
        if (from < to) rows = Span{(int32_t)from, (int32_t)to};
    }
    shown = rows.lo < rows.hi;
    return rows;
}

// d_lam of a head: the row tiles' sums in their order
template <int NT>
__device__ __forceinline__ void sum_lam(const AttnArgs& g, int h, int32_t row_tiles, char* scratch) {
    float* s_sum = reinterpret_cast<float*>(scratch);
    float x = 0.f;
    for (int k = threadIdx.x; k < row_tiles; k += NT) x += g.lam_part[(int64_t)k * g.a.Hq + h];
    s_sum[threadIdx.x] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        float y = 0.f;
        for (int k = 0; k < NT; ++k) y += s_sum[k];
        g.a.d_lam[h] = -y;
    }
}

// ------------------------------------------------------------------------------------- owned: keys, rows up to 512 bytes
// A wave owns 32 keys: both maps' scores, dP, dV and dK of a tile of 32 query rows, nothing twice.  The products alternate with
// the vector instructions of the phase before (scores of the second map with the exponentials of the first, and so on), so
// that both kinds overlap within a wave; from 256-byte rows on one wave a SIMD has the registers for that.  At 512 bytes the
// sums of a wave take half of them; there two waves share the keys, take every other tile and add up at the end, and the keys
// of the first map and a quarter of the values come from LDS (or the sums are moved to memory and back in every step).
template <typename T, int DP>
struct Keys {
    static constexpr int RB = Shape<T, DP>::RB, SPLIT = RB > 256 ? 2 : 1, SUBS = 2, BQ = 32 * SUBS, TILE = 2 * BQ * RB, STAT = 3 * 256;
    static constexpr int BUF = TILE + SUBS * STAT;              // rows; per 32 of them lse and t of both maps, lam
    static constexpr int WAVES = 4, GROUPS = WAVES / SPLIT, ROWS = GROUPS * 32, OCC = RB < 256 ? 2 : 1, AHEAD = RB == 256 ? 4 : 2;
    static constexpr int KEY_LDS = RB > 256;           // maps whose keys are read from LDS
    static constexpr int OWN = KEY_LDS ? ROWS * RB / 2 * KEY_LDS : 16;
    static constexpr int VAL_LDS = RB > 256 ? Shape<T, DP>::VS / 4 : 0;     // fragments of the values, a lane's beside the next lane's
    static constexpr int VAL = VAL_LDS ? VAL_LDS * GROUPS * 1024 : 16;
};

template <typename T, int DP, int MODE>
__device__ __forceinline__ void keys_body(const AttnArgs& g, int32_t tiles, char* s_a, char* s_b, char* s_own, char* s_val, uint8_t* s_marks, int* s_lo, int* s_hi, int& s_bad) {
    typedef Shape<T, DP> S;
    typedef Keys<T, DP> P;
    typedef Mat<T> M;
    constexpr int RB = S::RB, NT = P::WAVES * 64, ROWS = P::ROWS, GROUPS = P::GROUPS, BQ = P::BQ, TILE = P::TILE, AHEAD = P::AHEAD;
    const sgl_diff_attn_args& a = g.a;
    const int G = a.Hq / a.Hk;
    const uint32_t n = (uint32_t)tiles * (uint32_t)a.Hk, item = xcd_item(g, n);
    if (item >= n) return;
    // key heads side by side; of a causal call the early keys, which most rows see, come first
    const int hk = (int)(item % (uint32_t)a.Hk);
    const int32_t tile = (int32_t)(item / (uint32_t)a.Hk);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = wave % GROUPS, half = lane >> 5, col = lane & 31;
    const int share = wave / GROUPS;                            // which of the tiles
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int32_t j0 = tile * ROWS + group * 32, j = j0 + col;
    bool shown;
    int32_t seq;
    const Span rows = rows_of(a, B, j0, col, shown, seq);
    // the wave's union, and the run of rows that see all its keys (if it has no key that none sees)
    Reach reach = reach_of(rows);
    if (!__all(shown)) reach.to = 0;
    if (lane == 0) s_lo[wave] = reach.lo, s_hi[wave] = reach.hi;
    if (threadIdx.x == 0) s_bad = 0;
    clear_image<MODE, TILE, NT>(s_a);
    clear_image<MODE, TILE, NT>(s_b);
    __syncthreads();
    int32_t lo = s_lo[0], hi = s_hi[0];
#pragma unroll
    for (int w = 1; w < GROUPS; ++w) lo = min(lo, s_lo[w]), hi = max(hi, s_hi[w]);
    constexpr int V_REGS = S::VS - P::VAL_LDS;
    typename M::Frag k[2][S::QS], v[V_REGS];
    int32_t by_val = group * 1024 + lane * 16;
    {
        const int64_t jj = j < a.Tk ? j : 0;
#pragma unroll
        for (int m = P::KEY_LDS; m < 2; ++m)
#pragma unroll
            for (int e = 0; e < S::QS; ++e) k[m][e] = global_frag<T, MODE == WHOLE_ROWS>(row<T>(a.k, jj, 2 * hk + m), (2 * e + half) * S::EP, a.D, g.grain);
        if constexpr (P::KEY_LDS == 2) Stager<T, DP, ROWS, NT, BY_REGISTERS, true>().load(s_own, halves<T>(a.k, hk, a.D), tile * ROWS, (int32_t)a.Tk - 1, g.grain);
        if constexpr (P::KEY_LDS == 1) Stager<T, DP / 2, ROWS, NT, BY_REGISTERS, false>().load(s_own, run<T>(a.k, 2 * hk, a.D), tile * ROWS, (int32_t)a.Tk - 1, g.grain);
#pragma unroll
        for (int e = 0; e < V_REGS; ++e) v[e] = global_frag<T, MODE == WHOLE_ROWS>(row<T>(a.v, jj, hk), (2 * e + half) * S::EP, a.Dv, g.grain);
        if (P::VAL_LDS && share == 0) {
#pragma unroll
            for (int e = 0; e < P::VAL_LDS; ++e)
                *reinterpret_cast<typename M::Frag*>(s_val + e * GROUPS * 1024 + by_val) = global_frag<T, MODE == WHOLE_ROWS>(row<T>(a.v, jj, hk), (2 * (V_REGS + e) + half) * S::EP, a.Dv, g.grain);
        }
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
    const float c2 = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(signed_c2(g))));
    const int32_t last = (int32_t)a.Tq - 1;
    const int32_t per_head = lo < hi ? (hi - lo + BQ - 1) / BQ : 0, steps = per_head * G;      // head by head, row tile by row tile
    Stager<T, DP, BQ, NT, MODE, true> stage_q;
    Stager<T, DP, BQ, NT, MODE, false> stage_go;
    stage_q.plan(halves<T>(a.q, 0, a.D));
    stage_go.plan(run<T>(a.d_out, 0, a.Dv));
    bool finite = false;        // the pass without what is not finite
    auto load = [&](char* buf, int h, int32_t i0) {
        if (finite) {
            stage_finite<T, DP, BQ, NT>(buf, s_marks, halves<T>(a.q, h, a.D), true, i0, last);
            stage_finite<T, DP, BQ, NT>(buf + BQ * RB, s_marks + BQ * (RB / 16), run<T>(a.d_out, h, a.Dv), false, i0, last);
        } else {
            stage_q.load(buf, halves<T>(a.q, h, a.D), i0, last, g.grain);
            stage_go.load(buf + BQ * RB, run<T>(a.d_out, h, a.Dv), i0, last, g.grain);
        }
        if (wave < 3) {
            // 64 numbers each: lse, t of the rows, map by map, and lam 64 times (a load of its own in a step would wait for the
            // tile that is on its way)
#pragma unroll
            for (int u = 0; u < P::SUBS; ++u) {
                const int32_t i = min(i0 + 32 * u + (lane & 31), last);
                const float* src = wave == 2 ? a.lam + h : (wave ? g.delta : a.lse) + pair_at(a, i, h) + (lane >> 5);
                const int at0 = __builtin_amdgcn_readfirstlane(u * P::STAT + wave * 256);
                __builtin_amdgcn_global_load_lds((SGL_GLOBAL void*)src, (SGL_LDS void*)(buf + TILE + at0), 4, 0, 0);
            }
        }
    };
    // The lane's parts of the addresses, fixed here (left alone the compiler keeps the sum of each with every buffer)
    int32_t by_row[4], by_key[4], by_col[2], by_stat = 16 * half + share * P::STAT;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (P::KEY_LDS) by_key[e] = lane_row<RB / 2 * P::KEY_LDS>(col, e, half) + group * 4 * (RB * P::KEY_LDS / 256) * 1024;
        by_row[e] = lane_row<RB>(col, e, half) + share * 4 * (RB / 128) * 1024;
        asm volatile("" : "+v"(by_row[e]), "+v"(by_key[e]));
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        by_col[e] = lane_col<T, RB>(e, lane) + share * 4 * (RB / 128) * 1024;
        asm volatile("" : "+v"(by_col[e]));
    }
    asm volatile("" : "+v"(by_stat), "+v"(by_val));
    auto of_row = [](const char* tile, const int32_t (&by)[4], int i) { return *reinterpret_cast<const typename M::Frag*>(tile + (i >> 2) * 1024 + by[i & 3]); };
    // 32 rows from i0, the first of which is row `sub` of the tile (beside the wave's share)
    auto sub_step = [&](const char* buf, int32_t i0, int sub, auto load_next) {
        i0 += 32 * share + sub;
        if (i0 >= reach.hi || i0 + 32 <= reach.lo) return load_next();
        constexpr int PS = Operand<T>::PS, QS = S::QS, NK = S::DT * PS;
        constexpr int N1 = QS, N2 = 2 * QS, N3 = N2 + S::VS, N4 = N3 + S::VT * PS, N5 = N4 + NK, N6 = N5 + NK;
        const char* go = buf + BQ * RB + sub * RB;
        const char* stat = buf + TILE + sub / 32 * P::STAT + by_stat;
        buf += sub * RB;
        f32x4 num[4];           // lse of the first map, then of the second, then t of either: a group is read a phase before its use
#pragma unroll
        for (int k = 0; k < 4; ++k) num[k] = *reinterpret_cast<const f32x4*>(stat + 32 * k);
        const float lam = *reinterpret_cast<const float*>(stat + 512);
        const bool some = !(i0 >= reach.from && i0 + 32 <= reach.to);
        uint32_t see = 0;
        if (some) see = span_bits(i0, rows) >> (4 * half);
        f32x16 s[2], dp;
        s[0] = s[1] = dp = zero16();
        Operand<T> p, ds[2];
        auto load_n = [&](int n) {
            if (n < N2) return of_row(buf, by_row, n);
            if (n < N3) return of_row(go, by_row, n - N2);
            if (n < N4) return col_at<T, RB>(go, by_col, 0, (n - N3) / S::VT, (n - N3) % S::VT);
            // dK of a map: the tiles of its half
            const int m = n < N5 ? 0 : 1, u = n - (m ? N5 : N4);
            return col_at<T, RB>(buf, by_col, 0, u / S::DT, m * S::DT + u % S::DT);
        };
        auto load_own = [&](int n) { return of_row(s_own, by_key, n); };
        // exponentials, d_score of registers r, r + 1 of a map
        auto exps = [&](int m, int r, float f) {
#pragma unroll
            for (int e = r; e < r + 2; ++e) s[m][e] = f * exp2_hw(__builtin_fmaf(s[m][e], c2, -num[r / 4][e % 4]));
            if (r % 4 == 2) num[r / 4] = *reinterpret_cast<const f32x4*>(stat + 128 * (m + 1) + 32 * (r / 4));
        };
        auto scores = [&](int m, int r) {
            ds[m].set2(r, s[m][r] * (dp[r] - num[r / 4][r % 4]), s[m][r + 1] * (dp[r + 1] - num[r / 4][r % 4 + 1]));
            if (r % 4 == 2 && m == 0) num[r / 4] = *reinterpret_cast<const f32x4*>(stat + 384 + 32 * (r / 4));
        };
        constexpr int FROM_LDS = P::KEY_LDS * QS;
        auto load_val = [&](int e) { return *reinterpret_cast<const typename M::Frag*>(s_val + e * GROUPS * 1024 + by_val); };
        Pipe<T, P::VAL_LDS, 2> values;
        Pipe<T, N6, AHEAD> ahead;
        Pipe<T, FROM_LDS, AHEAD> own;
        if constexpr (P::KEY_LDS) own.fill(load_own);
        ahead.fill(load_n);
        auto score = [&](int n, const typename M::Frag& x) {
            f32x16& to = s[n / QS];
            if (n < FROM_LDS) {
                to = M::mma(x, own.f[n % AHEAD], to);
                if (n + AHEAD < FROM_LDS) own.f[n % AHEAD] = load_own(n + AHEAD);
            } else {
                to = M::mma(x, k[n / QS][n % QS], to);
            }
        };
        ahead.template part<0, N1>(load_n, [&](int n, const typename M::Frag& x) { score(n, x); });
        ahead.template part<N1, N2>(load_n, [&](int n, const typename M::Frag& x) {
            score(n, x);
#pragma unroll
            for (int r = 8 * (n - N1) / QS * 2; r < 8 * (n - N1 + 1) / QS * 2; r += 2) exps(0, r, 1.f);
        });
        ahead.template part<N2, N3>(load_n, [&](int n, const typename M::Frag& x) {
            const int u = n - N2;
            if (P::VAL_LDS && u == V_REGS - 2) values.fill(load_val);
            if (u < V_REGS) {
                dp = M::mma(x, v[u], dp);
            } else {
                dp = M::mma(x, values.f[(u - V_REGS) % 2], dp);
                if (u + 2 < S::VS) values.f[(u - V_REGS) % 2] = load_val(u + 2 - V_REGS);
            }
#pragma unroll
            for (int r = 8 * (n - N2) / S::VS * 2; r < 8 * (n - N2 + 1) / S::VS * 2; r += 2) {
                exps(1, r, -lam);
                p.set2(r, s[0][r] + s[1][r], s[0][r + 1] + s[1][r + 1]);
            }
        });
        // (what the registers do not hold is read back in the phases above, where it would wait for these loads: at 512 bytes a
        // row the kernel above takes 985 us with them in front)
        load_next();
        if (some) p.mask(see);
        ahead.template part<N3, N4>(load_n, [&](int n, const typename M::Frag& x) {
            constexpr int N = N4 - N3;
            const int u = n - N3;
            dv[u % S::VT] = M::mma(x, p.f[u / S::VT], dv[u % S::VT]);
#pragma unroll
            for (int r = 8 * u / N * 2; r < 8 * (u + 1) / N * 2; r += 2) scores(0, r);
        });
        if (some) ds[0].mask(see);
        ahead.template part<N4, N5>(load_n, [&](int n, const typename M::Frag& x) {
            const int u = n - N4;
            dk[0][u % S::DT] = M::mma(x, ds[0].f[u / S::DT], dk[0][u % S::DT]);
#pragma unroll
            for (int r = 8 * u / NK * 2; r < 8 * (u + 1) / NK * 2; r += 2) scores(1, r);
        });
        if (some) ds[1].mask(see);
        ahead.template part<N5, N6>(load_n, [&](int n, const typename M::Frag& x) {
            const int u = n - N5;
            dk[1][u % S::DT] = M::mma(x, ds[1].f[u / S::DT], dk[1][u % S::DT]);
        });
    };
    auto step = [&](const char* buf, int32_t i0, auto load_next) {
        if constexpr (P::SPLIT == 2) {
            sub_step(buf, i0, 0, load_next);
        } else {
            load_next();
            sub_step(buf, i0, 0, [] {});
            sub_step(buf, i0, 32, [] {});
        }
    };
    bool spoilt[2] = {false, false};        // a row with something not finite sees the key: NaN
    if (steps > 0) {
        int h, hn;                          // head and first row of the tile at work, and of the one being loaded
        int32_t i0, in;
        auto next = [&]() {
            in += BQ;
            if (in >= hi) in = lo, ++hn;
        };
#pragma unroll 1
        for (;;) {
            hn = hk * G, in = lo;
            load(s_a, hn, in);
            staged();
#pragma unroll 1
            for (int32_t s = 0; s < steps; s += 2) {
                h = hn, i0 = in;
                next();
                step(s_a, i0, [&] {
                    if (s + 1 < steps) load(s_b, hn, in);
                });
                staged();
                if (s + 1 >= steps) break;
                h = hn, i0 = in;
                next();
                step(s_b, i0, [&] {
                    if (s + 2 < steps) load(s_a, hn, in);
                });
                staged();
            }
            if (finite) break;
            if ((any_nan(dk[0]) || any_nan(dk[1]) || any_nan(dv)) && shown) s_bad = 1;
            __syncthreads();
            if (!s_bad) break;
            finite = true;
            clear();
        }
        if (finite) {
            // the keys that a row with something not finite sees get NaN
            hn = hk * G, in = lo;
#pragma unroll 1
            for (int32_t s = 0; s < steps; ++s) {
                __syncthreads();
                stage_finite<T, DP, BQ, NT>(s_a, s_marks, halves<T>(a.q, hn, a.D), true, in, last);
                stage_finite<T, DP, BQ, NT>(s_a + BQ * RB, s_marks + BQ * (RB / 16), run<T>(a.d_out, hn, a.Dv), false, in, last);
                __syncthreads();
#pragma unroll 1
                for (int r = 0; r < BQ; ++r) {
                    if (in + r < rows.lo || in + r >= rows.hi) continue;
                    const uint8_t* of_out = s_marks + BQ * (RB / 16);
                    const bool o = marked_any<RB>(of_out, r, 0, RB / 16);
                    spoilt[0] = spoilt[0] || o || marked_any<RB>(s_marks, r, 0, RB / 32);
                    spoilt[1] = spoilt[1] || o || marked_any<RB>(s_marks, r, RB / 32, RB / 16);
                    if (o) spoil<T, RB, S::VT>(dv, of_out, r, half);
                }
                next();
            }
            __syncthreads();
        }
    }
    const uint32_t keep = (uint32_t)__ballot(j < a.Tk && (seq >= 0 || (a.flags & SGL_ATTN_ZERO_REST)));
    // the tiles are free: the last barrier is behind every wave's last look at them
    if constexpr (P::SPLIT == 2) {
        // the first wave takes dK, the second dV; each hands the other's part over
        static_assert(2 * S::DT * 4096 * GROUPS <= TILE && S::VT * 4096 * GROUPS <= TILE, "parts fit");
        char* mine = s_a + group * (2 * S::DT * 4096) + lane * 16;
        char* other = s_b + group * (S::VT * 4096) + lane * 16;
        auto put = [&](char* box, const f32x16& x) {
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) *reinterpret_cast<f32x4*>(box + r4 * 1024) = f32x4{x[4 * r4], x[4 * r4 + 1], x[4 * r4 + 2], x[4 * r4 + 3]};
        };
        auto add = [&](const char* box, f32x16& x) {
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const f32x4 y = *reinterpret_cast<const f32x4*>(box + r4 * 1024);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * r4 + e] += y[e];
            }
        };
        // (the ends of the branches differ: merged, they would address the sums, and these would lie in memory from the start)
        if (share) {
#pragma unroll
            for (int d = 0; d < S::DT; ++d) put(mine + d * 4096, dk[0][d]), put(mine + (S::DT + d) * 4096, dk[1][d]);
            asm volatile("; keys handed over");
        } else {
#pragma unroll
            for (int d = 0; d < S::VT; ++d) put(other + d * 4096, dv[d]);
            asm volatile("; values handed over");
        }
        __syncthreads();
        if (share) {
#pragma unroll
            for (int d = 0; d < S::VT; ++d) add(other + d * 4096, dv[d]);
            asm volatile("; values joined");
        } else {
#pragma unroll
            for (int d = 0; d < S::DT; ++d) add(mine + d * 4096, dk[0][d]), add(mine + (S::DT + d) * 4096, dk[1][d]);
            asm volatile("; keys joined");
        }
        __syncthreads();
    }
    constexpr int PIECE = TILE / P::WAVES / 32;                 // bytes of a row at a time
    char* box = s_a + wave * (TILE / P::WAVES);
    if (P::SPLIT == 1 || !share) {
        store_rows<T, PIECE, S::DT, MODE == WHOLE_ROWS>([&](int t, int r) { return spoilt[0] ? NAN : shown ? dk[0][t][r] * g.scale : 0.f; }, box, lane, a.D, g.grain,
                                         row_out<T>(a.d_k, j0, 2 * hk), a.d_k.row_stride, keep);
        store_rows<T, PIECE, S::DT, MODE == WHOLE_ROWS>([&](int t, int r) { return spoilt[1] ? NAN : shown ? dk[1][t][r] * g.scale : 0.f; }, box, lane, a.D, g.grain,
                                         row_out<T>(a.d_k, j0, 2 * hk + 1), a.d_k.row_stride, keep);
    }
    if (P::SPLIT == 1 || share)
        store_rows<T, PIECE, S::VT, MODE == WHOLE_ROWS>([&](int t, int r) { return shown ? dv[t][r] : 0.f; }, box, lane, a.Dv, g.grain, row_out<T>(a.d_v, j0, hk), a.d_v.row_stride, keep);
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__((Keys<T, DP>::WAVES * 64), (Keys<T, DP>::OCC)) void bwd_keys_kernel(AttnArgs g, int32_t tiles, int32_t row_tiles) {
    typedef Keys<T, DP> P;
    __shared__ __align__(16) char s_a[P::BUF];
    __shared__ __align__(16) char s_b[P::BUF];
    __shared__ __align__(16) char s_own[P::OWN];
    __shared__ __align__(16) char s_val[P::VAL];
    __shared__ __align__(8) uint8_t s_marks[2 * P::BQ * (P::RB / 16)];
    __shared__ int s_lo[P::WAVES], s_hi[P::WAVES], s_bad;
    const int64_t blocks = ceil_div<int64_t>((int64_t)tiles * g.a.Hk, 8) * 8, block = g.first + blockIdx.x;
    if (block >= blocks) sum_lam<P::WAVES * 64>(g, (int)(block - blocks), row_tiles, s_a);
    else keys_body<T, DP, MODE>(g, tiles, s_a, s_b, s_own, s_val, s_marks, s_lo, s_hi, s_bad);
}

// -------------------------------------------------------------------- owned: keys, rows of 1024 bytes (fp32, heads over 64)
// Four waves share 32 keys: two sum a map's dK each, two half of dV's columns; each computes the scores that it needs, the former
// dP too (no wave's registers hold more of the sums).  Keys and values are read from LDS, whose rest holds one tile of rows.
// 8 sequences of 1024, 8 heads 128 wide, causal: 1306 us; two waves, one for dK and one for dV, 1834.
template <typename T, int DP>
struct Roles {
    static constexpr int RB = Shape<T, DP>::RB, WAVES = 4, ROWS = 32, BQ = 32, TILE = 2 * BQ * RB;
    static constexpr int STAT = 2 * 256;                        // lse and t of the rows, map by map
    static constexpr int BUF = TILE + STAT, OWN = 2 * ROWS * RB;
    static_assert(sizeof(T) == 4 && RB >= 256, "a tile of 32 values is a piece of the image");
};

// DK: this wave sums dK of map `part`; else half `part` of dV's columns
template <typename T, int DP, int MODE, bool DK>
__device__ __forceinline__ void roles_body(const AttnArgs& g, int32_t tiles, char* s_a, char* s_own, uint8_t* s_marks, int& s_bad, int part) {
    typedef Shape<T, DP> S;
    typedef Roles<T, DP> P;
    typedef Mat<T> M;
    constexpr int RB = S::RB, NT = P::WAVES * 64, ROWS = P::ROWS, BQ = P::BQ, TILE = P::TILE, AHEAD = 2;
    const sgl_diff_attn_args& a = g.a;
    const int G = a.Hq / a.Hk;
    const uint32_t n = (uint32_t)tiles * (uint32_t)a.Hk, item = xcd_item(g, n);
    if (item >= n) return;
    // key heads side by side; of a causal call the early keys, which most rows see, come first
    const int hk = (int)(item % (uint32_t)a.Hk);
    const int32_t tile = (int32_t)(item / (uint32_t)a.Hk);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
    const int32_t B = (int32_t)live_count(a.B_dev, a.B);
    const int32_t j0 = tile * ROWS, j = j0 + col;
    bool shown;
    int32_t seq;
    const Span rows = rows_of(a, B, j0, col, shown, seq);
    // the wave's union, and the run of rows that see all its keys (if it has no key that none sees)
    Reach reach = reach_of(rows);
    if (!__all(shown)) reach.to = 0;
    if (threadIdx.x == 0) s_bad = 0;
    clear_image<MODE, TILE, NT>(s_a);
    if (MODE == PADDED) __syncthreads();
    const int32_t lo = reach.lo, hi = reach.hi;                 // (the waves have the same keys)
    Stager<T, DP, ROWS, NT, BY_REGISTERS, true>().load(s_own, halves<T>(a.k, hk, a.D), j0, (int32_t)a.Tk - 1, g.grain);
    Stager<T, DP, ROWS, NT, BY_REGISTERS, false>().load(s_own + ROWS * RB, run<T>(a.v, hk, a.Dv), j0, (int32_t)a.Tk - 1, g.grain);
    constexpr int N = DK ? S::DT : S::VT / 2;                   // 32-wide tiles of the sum
    f32x16 acc[N];
    auto clear = [&]() {
#pragma unroll
        for (int d = 0; d < N; ++d) acc[d] = zero16();
    };
    clear();
    const int32_t last = (int32_t)a.Tq - 1;
    const float c2 = signed_c2(g);
    const int32_t per_head = lo < hi ? (hi - lo + BQ - 1) / BQ : 0, steps = per_head * G;      // head by head, row tile by row tile
    auto load_stats = [&](char* buf, int h, int32_t i0) {
        if (wave < 2) {
            const int32_t i = min(i0 + (lane & 31), last);
            const float* src = (wave ? g.delta : a.lse) + pair_at(a, i, h) + (lane >> 5);
            const int at0 = __builtin_amdgcn_readfirstlane(wave * 256);
            __builtin_amdgcn_global_load_lds((SGL_GLOBAL void*)src, (SGL_LDS void*)(buf + TILE + at0), 4, 0, 0);
        }
    };
    Stager<T, DP, BQ, NT, MODE, true> stage_q;
    Stager<T, DP, BQ, NT, MODE, false> stage_go;
    stage_q.plan(halves<T>(a.q, 0, a.D));
    stage_go.plan(run<T>(a.d_out, 0, a.Dv));
    bool finite = false;        // the pass without what is not finite
    auto load = [&](char* buf, int h, int32_t i0) {
        if (finite) {
            stage_finite<T, DP, BQ, NT>(buf, s_marks, halves<T>(a.q, h, a.D), true, i0, last);
            stage_finite<T, DP, BQ, NT>(buf + BQ * RB, s_marks + BQ * (RB / 16), run<T>(a.d_out, h, a.Dv), false, i0, last);
        } else {
            stage_q.load(buf, halves<T>(a.q, h, a.D), i0, last, g.grain);
            stage_go.load(buf + BQ * RB, run<T>(a.d_out, h, a.Dv), i0, last, g.grain);
        }
        load_stats(buf, h, i0);
    };
    auto step = [&](const char* buf, int h, int32_t i0) {
        if (i0 >= reach.hi || i0 + BQ <= reach.lo) return;
        const float lam = a.lam[h];
        const float* stat = reinterpret_cast<const float*>(buf + TILE) + 4 * half;
        const char* go = buf + BQ * RB;
        f32x16 s[2], dp;
        s[0] = s[1] = dp = zero16();
        // fragments of the walked rows: a half of the queries and d_out, or both halves; those of the owned rows ride along
        auto load = [&](const char* rows2, int n) {
            if (n >= S::QS && DK) return row_frag<T, RB>(rows2 + BQ * RB, 0, col, n - S::QS, half);
            return map_frag<T, RB>(rows2, 0, col, DK ? part : n / S::QS, n % S::QS, half);
        };
        auto load_row = [&](int n) { return load(buf, n); };
        auto load_own = [&](int n) { return load(s_own, n); };
        constexpr int FRAGS = S::QS + (DK ? S::VS : S::QS);
        Pipe<T, FRAGS, AHEAD> ahead, own;
        own.fill(load_own);
        ahead.fill(load_row);
        ahead.drain(load_row, [&](int n, const typename M::Frag& f) {
            f32x16& to = n < S::QS ? s[0] : DK ? dp : s[1];
            to = M::mma(f, own.f[n % AHEAD], to);
            if (n + AHEAD < FRAGS) own.f[n % AHEAD] = load_own(n + AHEAD);
        });
        // dS of the map (the second's times -lam), or P_1 - lam P_2
        const float weight = DK && part == 0 ? 1.f : -lam;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 l = *reinterpret_cast<const f32x4*>(stat + (DK ? 32 * part : 0) + 8 * r4);
            const f32x4 u = *reinterpret_cast<const f32x4*>(stat + (DK ? 64 + 32 * part : 32) + 8 * r4);      // t, or the second map's lse
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * r4 + e;
                const float p = exp2_hw(__builtin_fmaf(s[0][r], c2, -l[e]));
                if constexpr (DK) s[0][r] = weight * p * (dp[r] - u[e]);
                else s[0][r] = __builtin_fmaf(weight, exp2_hw(__builtin_fmaf(s[1][r], c2, -u[e])), p);
            }
        }
        if (!(i0 >= reach.from && i0 + BQ <= reach.to)) {
            const uint32_t see = span_bits(i0, rows) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = row_bit(see, r) ? s[0][r] : 0.f;
        }
        add_product<T, RB, N, AHEAD>(acc, (DK ? buf : go) + part * N * 1024, 0, 0, operand<T>(s[0]), lane);
    };
    bool spoilt = false;                    // (dK) a row with something not finite sees the key: NaN
    if (steps > 0) {
        int hn;                             // head and first row of the tile
        int32_t in;
        auto next = [&]() {
            in += BQ;
            if (in >= hi) in = lo, ++hn;
        };
#pragma unroll 1
        for (;;) {
            hn = hk * G, in = lo;
            load(s_a, hn, in);
            staged();
#pragma unroll 1
            for (int32_t s = 0; s < steps; ++s) {
                step(s_a, hn, in);
                __syncthreads();
                next();
                if (s + 1 < steps) load(s_a, hn, in);
                staged();
            }
            if (finite) break;
            if (any_nan(acc) && shown) s_bad = 1;
            __syncthreads();
            if (!s_bad) break;
            finite = true;
            clear();
        }
        if (finite) {
            // the keys that a row with something not finite sees get NaN
            hn = hk * G, in = lo;
#pragma unroll 1
            for (int32_t s = 0; s < steps; ++s) {
                __syncthreads();
                stage_finite<T, DP, BQ, NT>(s_a, s_marks, halves<T>(a.q, hn, a.D), true, in, last);
                stage_finite<T, DP, BQ, NT>(s_a + BQ * RB, s_marks + BQ * (RB / 16), run<T>(a.d_out, hn, a.Dv), false, in, last);
                __syncthreads();
#pragma unroll 1
                for (int r = 0; r < BQ; ++r) {
                    if (in + r < rows.lo || in + r >= rows.hi) continue;
                    const uint8_t* of_out = s_marks + BQ * (RB / 16);
                    const bool o = marked_any<RB>(of_out, r, 0, RB / 16);
                    if constexpr (DK) spoilt = spoilt || o || marked_any<RB>(s_marks, r, part * (RB / 32), (part + 1) * (RB / 32));
                    else if (o) spoil<T, RB, N>(acc, of_out + part * N * 8, r, half);
                }
                next();
            }
            __syncthreads();
        }
    }
    const uint32_t keep = (uint32_t)__ballot(j < a.Tk && (seq >= 0 || (a.flags & SGL_ATTN_ZERO_REST)));
    // the walked side's tiles are free: the last barrier is behind every wave's last look at them
    char* box = s_a + wave * (TILE / P::WAVES);
    constexpr int PIECE = TILE / P::WAVES / 32;               // bytes of a row at a time
    if constexpr (DK)
        store_rows<T, PIECE, N, MODE == WHOLE_ROWS>([&](int d, int r) { return spoilt ? NAN : shown ? acc[d][r] * g.scale : 0.f; }, box, lane, a.D, g.grain,
                                     row_out<T>(a.d_k, j0, 2 * hk + part), a.d_k.row_stride, keep);
    else
        store_rows<T, PIECE, N, MODE == WHOLE_ROWS>([&](int d, int r) { return shown ? acc[d][r] : 0.f; }, box, lane, a.Dv - part * N * 32, g.grain,
                                     row_out<T>(a.d_v, j0, hk) + part * N * 32, a.d_v.row_stride, keep);
}

template <typename T, int DP, int MODE>
__global__ __launch_bounds__((Roles<T, DP>::WAVES * 64), 1) void bwd_roles_kernel(AttnArgs g, int32_t tiles, int32_t row_tiles) {
    typedef Roles<T, DP> P;
    __shared__ __align__(16) char s_a[P::BUF];
    __shared__ __align__(16) char s_own[P::OWN];
    __shared__ __align__(8) uint8_t s_marks[2 * P::BQ * (P::RB / 16)];
    __shared__ int s_bad;
    const int64_t blocks = ceil_div<int64_t>((int64_t)tiles * g.a.Hk, 8) * 8, block = g.first + blockIdx.x;
    if (block >= blocks) return sum_lam<P::WAVES * 64>(g, (int)(block - blocks), row_tiles, s_a);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave < 2) roles_body<T, DP, MODE, true>(g, tiles, s_a, s_own, s_marks, s_bad, wave);
    else roles_body<T, DP, MODE, false>(g, tiles, s_a, s_own, s_marks, s_bad, wave - 2);
}

template <typename T, int DP>
void launch(const AttnArgs& g, hipStream_t st) {
    const sgl_diff_attn_args& a = g.a;
    typedef Shape<T, DP> S;
    const int32_t qt = (int32_t)ceil_div<int64_t>(a.Tq, QUERY_ROWS);
    auto go = [&](auto mode) {
        constexpr int MODE = decltype(mode)::value;
        if (qt > 0)
            in_parts(g, ceil_div<int64_t>((int64_t)qt * a.Hq, 8) * 8, [&](const AttnArgs& part, dim3 grid) {
                hipLaunchKernelGGL((bwd_rows_kernel<T, DP, MODE>), grid, dim3(Rows<T, DP>::WAVES * 64), 0, st, part, qt);
            });
        if constexpr (S::RB <= 512) {
            typedef Keys<T, DP> P;
            const int32_t kt = (int32_t)ceil_div<int64_t>(a.Tk, P::ROWS);
            in_parts(g, ceil_div<int64_t>((int64_t)kt * a.Hk, 8) * 8 + a.Hq, [&](const AttnArgs& part, dim3 grid) {
                hipLaunchKernelGGL((bwd_keys_kernel<T, DP, MODE>), grid, dim3(P::WAVES * 64), 0, st, part, kt, qt);
            });
        } else {
            typedef Roles<T, DP> P;
            const int32_t kt = (int32_t)ceil_div<int64_t>(a.Tk, P::ROWS);
            in_parts(g, ceil_div<int64_t>((int64_t)kt * a.Hk, 8) * 8 + a.Hq, [&](const AttnArgs& part, dim3 grid) {
                hipLaunchKernelGGL((bwd_roles_kernel<T, DP, MODE>), grid, dim3(P::WAVES * 64), 0, st, part, kt, qt);
            });
        }
    };
    const int mode = stage_mode(g, DP, {&a.k, &a.v, &a.q, &a.d_out});
    if (mode == WHOLE_ROWS) go(Int<WHOLE_ROWS>{});
    else if (mode == PADDED) go(Int<PADDED>{});
    else go(Int<BY_REGISTERS>{});
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
