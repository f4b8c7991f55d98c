// Rotary encoding of rows by their event times, and the per-head RMS norm of queries and keys with that rotation in
// the same pass, forward and backward, for gfx950.
//
// Rotation: pair (a, b) of a head becomes A (a cos t - b sin t, a sin t + b cos t), t = pos * freq[i] in fp64 (event
// times reach 2^40, where an fp32 angle is off by whole turns).  Norm: y = rotate(x r w), r = (mean x^2 + eps)^-1/2.
// Backward: d = rotate^T(dy), dw = sum d x r, dx = r d w - x r^3 mean(d w x).
//
// All of it is bound by the rows it moves (x read once, the result written once; backward: x and dy read, dx
// written), so the work per value is kept small: the angles of a row are formed once per block, reduced in fp64 and
// parked in LDS as (cos, sin), and every head of the row reads them from there.  Reached, of the bytes a step cannot do without:
// rotation 5.9 TB/s at 131072 rows of 4 KB, 3.2 at 120000 rows of 400 bytes; norm, forward and backward, 4.0 TB/s at 65536 rows
// of 5 KB (a copy of 1 GiB: 5.0).
#include <math.h>

#include "common.hpp"

namespace sgl {
namespace {

constexpr int BLOCK = 256;
constexpr int DIM_MAX = 1024;
constexpr int TABLE_MAX = 2048;            // (cos, sin) pairs of a tile in LDS: 16 KB
constexpr int NORM_BWD_BLOCKS = 1024;      // blocks of one side's backward: one row of partial weight gradients each

enum { OP_ROT, OP_NORM, OP_NORM_BWD };

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T e[N];
};

struct Side {
    const void* x;
    const void* y;          // backward: the incoming gradient
    void* out;              // forward: y; backward: dx
    int64_t x_row, x_head, y_row, y_head, o_row, o_head;
    const int64_t* pos;
    int64_t N_max;
    const int64_t* N_dev;
    const float* weight;
    int64_t w_stride;
    float* partial;         // backward: [blocks, w_stride ? heads * dim : dim]
    int32_t heads;
    int32_t rows;           // rows of a tile
    int32_t blocks;         // blocks of this side
    uint32_t heads_div;     // ceil(2^32 / heads), 0 for heads = 1
};

struct Args {
    Side s[2];
    int32_t blocks0;        // blocks of side 0; the others belong to side 1
    int32_t dim, half, pairs, inverse;
    float amplitude, eps;
    const double* freq;
};

// n / d for n < 2^16 from m = ceil(2^32 / d): the error n (m d - 2^32) / (d 2^32) is below 1 / d there (d < 2^16)
__device__ __forceinline__ int32_t fast_div(int32_t n, uint32_t m) { return m ? (int32_t)__umulhi((uint32_t)n, m) : n; }

// (cos a, sin a): a is reduced by multiples of pi/2 in fp64 (two-constant Cody-Waite through FMA), the remainder of at
// most pi/4 rounded to fp32 (3e-8) and put through the Taylor sums to r^11 and r^12 (next terms below 1e-9)
__device__ __forceinline__ float2 cos_sin(double a) {
    if (!(__builtin_fabs(a) < 1e15)) {      // also NaN; not reached by times below 2^49
        double s, c;
        sincos(a, &s, &c);
        return make_float2((float)c, (float)s);
    }
    constexpr double SHIFT = 6755399441055744.0;        // 1.5 * 2^52: the integer lands in the low mantissa bits
    const double t = __builtin_fma(a, 0.63661977236758134308, SHIFT);
    const uint32_t n = (uint32_t)__double_as_longlong(t) & 3u;
    const double k = t - SHIFT;
    double rd = __builtin_fma(-k, 1.57079632679489655800e+00, a);
    rd = __builtin_fma(-k, 6.12323399573676603587e-17, rd);
    const float r = (float)rd, r2 = r * r;
    float s = __builtin_fmaf(r2, -2.50521084e-8f, 2.75573192e-6f);
    s = __builtin_fmaf(s, r2, -1.98412698e-4f);
    s = __builtin_fmaf(s, r2, 8.33333333e-3f);
    s = __builtin_fmaf(s, r2, -1.66666667e-1f);
    s = __builtin_fmaf(s, r * r2, r);
    float c = __builtin_fmaf(r2, 2.08767570e-9f, -2.75573192e-7f);
    c = __builtin_fmaf(c, r2, 2.48015873e-5f);
    c = __builtin_fmaf(c, r2, -1.38888889e-3f);
    c = __builtin_fmaf(c, r2, 4.16666667e-2f);
    c = __builtin_fmaf(c, r2, -0.5f);
    c = __builtin_fmaf(c, r2, 1.0f);
    const float cc = (n & 1) ? s : c, ss = (n & 1) ? c : s;
    return make_float2((n == 1 || n == 2) ? -cc : cc, (n >= 2) ? -ss : ss);
}

// (a, b) -> A (a c - b s, a s + b c); the caller passes -s for the transpose
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float u = __builtin_fmaf(a, c, -(b * s)), w = __builtin_fmaf(a, s, b * c);
    a = u;
    b = w;
}

// A head's values lie in `pairs` pairs of vectors of VW values (A, B): the rotated part first, then the rest.
//   rotated, halves:               A at VW p,  B at VW p + half           (their values pair up across the vectors)
//   rotated, interleaved, VW > 1:  A at 2 VW p, B at 2 VW p + VW          (neighbours inside a vector pair up)
//   rotated, interleaved, VW = 1:  A at 2 p,   B at 2 p + 1               (as halves)
//   rest: two consecutive vectors; the last B may lie behind the head (b < 0)
template <int VW, bool INTER>
struct Where {
    int32_t a, b, t;        // offsets of A and B in the head, first table entry; t < 0: not rotated
    __device__ __forceinline__ Where(int32_t p, int32_t half, int32_t dim) {
        const int32_t rp = half / VW;
        if (p < rp) {
            a = INTER ? 2 * VW * p : VW * p;
            b = INTER ? a + VW : a + half;
            t = VW * p;
        } else {
            a = 2 * half + 2 * VW * (p - rp);
            b = a + VW < dim ? a + VW : -1;
            t = -1;
        }
    }
};

// LP lanes (a power of two, run-time) share a head; lane l of them holds the pairs l, l + 64, ... (NI of them; NI > 1
// only with LP = 64).  A block walks tiles of `rows` rows; the tile's (row, head) vectors are dealt to its groups.
template <typename T, int VW, bool INTER, int NI, int OP>
__global__ __launch_bounds__(BLOCK) void rows_kernel(Args g, int32_t lp_log2) {
    // Vectors on their way in a group.  Step (forward and gradient) of the rotation, 1, 2, 4 of them: 120000 rows of 2 heads of 50 in
    // fp32 (one value a lane) 73, 63, 60 us; 131072 rows of 16 heads of 128 in bf16, half rotated (16 bytes a lane) 396, 366, 403 us.  The
    // norm's registers are full with one: 65536 events, 40 heads of 64 in bf16, 331, 348, 387 us.
    constexpr int UN = NI > 1 || OP != OP_ROT ? 1 : VW * sizeof(T) <= 8 ? 4 : 2;
    extern __shared__ __align__(16) float2 s_cs[];
    const bool second = (int32_t)blockIdx.x >= g.blocks0;
    const Side& s = g.s[second];
    const int32_t block = (int32_t)blockIdx.x - (second ? g.blocks0 : 0);
    const int32_t lane = threadIdx.x & ((1 << lp_log2) - 1), group = threadIdx.x >> lp_log2, groups = BLOCK >> lp_log2;
    const int32_t half = g.half, dim = g.dim;
    const int64_t N = live_count(s.N_dev, s.N_max);
    const T* __restrict__ x = static_cast<const T*>(s.x);
    const T* __restrict__ y = static_cast<const T*>(s.y);
    T* __restrict__ out = static_cast<T*>(s.out);
    const float inv_dim = 1.0f / (float)dim;
    const bool per_head = s.w_stride != 0;
    // backward with weights of their own for every head: one pass over the rows for each head, so that a group's sum
    // belongs to one head
    const int32_t passes = OP == OP_NORM_BWD && per_head ? s.heads : 1;
    const bool one_head = OP == OP_NORM_BWD && per_head;

    for (int32_t pass = 0; pass < passes; ++pass) {
        float wa[NI][VW], wb[NI][VW], da[NI][VW], db[NI][VW];
        if (OP != OP_ROT) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
#pragma unroll
                for (int e = 0; e < VW; ++e) wa[i][e] = wb[i][e] = 1.0f, da[i][e] = db[i][e] = 0.0f;
                const int32_t p = lane + i * 64;
                if (s.weight != nullptr && p < g.pairs && (!per_head || one_head)) {
                    const Where<VW, INTER> w(p, half, dim);
                    const float* wp = s.weight + (one_head ? (int64_t)pass * s.w_stride : 0);
#pragma unroll
                    for (int e = 0; e < VW; ++e) {
                        wa[i][e] = wp[w.a + e];
                        if (w.b >= 0) wb[i][e] = wp[w.b + e];
                    }
                }
            }
        }
        for (int64_t row0 = (int64_t)block * s.rows; row0 < N; row0 += (int64_t)s.blocks * s.rows) {
            const int32_t rows = (int32_t)((N - row0) < s.rows ? (N - row0) : s.rows);
            if (half > 0) {
                __syncthreads();
                for (int32_t i = threadIdx.x; i < rows * half; i += BLOCK) {
                    const int32_t r = i / half;
                    float2 cs = cos_sin((double)s.pos[row0 + r] * g.freq[i - r * half]);
                    cs.x *= g.amplitude;
                    cs.y *= g.amplitude;
                    if (OP == OP_NORM_BWD || (OP == OP_ROT && g.inverse)) cs.y = -cs.y;
                    s_cs[i] = cs;
                }
                __syncthreads();
            }
            const int32_t vectors = one_head ? rows : rows * s.heads;
            // whole waves stay in the loop (the reductions below need the lanes of a group, which lie in one wave); a group has
            // UN vectors on their way at a time
            for (int32_t v0 = 0; v0 < vectors; v0 += UN * groups) {
                int32_t rr[UN], hh[UN];
                bool live[UN];
                float a[UN][NI][VW], b[UN][NI][VW], ga[UN][NI][VW], gb[UN][NI][VW];
                Vec<T, VW> va[UN][NI], vb[UN][NI], ya[UN][NI], yb[UN][NI];
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int32_t v = v0 + u * groups + group;
                    live[u] = v < vectors;
                    rr[u] = live[u] ? (one_head ? v : fast_div(v, s.heads_div)) : 0;
                    hh[u] = one_head ? pass : (live[u] ? v - rr[u] * s.heads : 0);
                    const T* __restrict__ xv = x + (row0 + rr[u]) * s.x_row + hh[u] * s.x_head;
                    const T* __restrict__ yv = OP == OP_NORM_BWD ? y + (row0 + rr[u]) * s.y_row + hh[u] * s.y_head : nullptr;
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const int32_t p = lane + i * 64;
#pragma unroll
                        for (int e = 0; e < VW; ++e) va[u][i].e[e] = vb[u][i].e[e] = ya[u][i].e[e] = yb[u][i].e[e] = (T)0.0f;
                        if (!live[u] || p >= g.pairs) continue;
                        const Where<VW, INTER> w(p, half, dim);
                        va[u][i] = *reinterpret_cast<const Vec<T, VW>*>(xv + w.a);
                        if (w.b >= 0) vb[u][i] = *reinterpret_cast<const Vec<T, VW>*>(xv + w.b);
                        if constexpr (OP == OP_NORM_BWD) {
                            ya[u][i] = *reinterpret_cast<const Vec<T, VW>*>(yv + w.a);
                            if (w.b >= 0) yb[u][i] = *reinterpret_cast<const Vec<T, VW>*>(yv + w.b);
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const int32_t r = rr[u], h = hh[u];
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < NI; ++i)
#pragma unroll
                        for (int e = 0; e < VW; ++e) {
                            a[u][i][e] = (float)va[u][i].e[e];
                            b[u][i][e] = (float)vb[u][i].e[e];
                            ga[u][i][e] = (float)ya[u][i].e[e];
                            gb[u][i][e] = (float)yb[u][i].e[e];
                            if (OP != OP_ROT) sum = __builtin_fmaf(a[u][i][e], a[u][i][e], __builtin_fmaf(b[u][i][e], b[u][i][e], sum));
                        }
                    float inv = 1.0f;
                    if constexpr (OP != OP_ROT) {
                        for (int32_t m = 1; m < (1 << lp_log2); m <<= 1) sum += __shfl_xor(sum, m);
                        inv = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum, inv_dim, g.eps));
                    }
                    float dot = 0.0f;
                    if constexpr (OP == OP_NORM_BWD) {
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            const int32_t p = lane + i * 64;
                            if (!live[u] || p >= g.pairs) continue;
                            const Where<VW, INTER> w(p, half, dim);
                            if (w.t >= 0) {
                                const float2* __restrict__ cs = s_cs + r * half + w.t;
                                if constexpr (INTER && VW > 1) {
#pragma unroll
                                    for (int e = 0; e < VW; e += 2) {
                                        turn(ga[u][i][e], ga[u][i][e + 1], cs[e / 2].x, cs[e / 2].y);
                                        turn(gb[u][i][e], gb[u][i][e + 1], cs[VW / 2 + e / 2].x, cs[VW / 2 + e / 2].y);
                                    }
                                } else {
#pragma unroll
                                    for (int e = 0; e < VW; ++e) turn(ga[u][i][e], gb[u][i][e], cs[e].x, cs[e].y);
                                }
                            }
#pragma unroll
                            for (int e = 0; e < VW; ++e) {
                                const float xa = a[u][i][e] * inv, xb = b[u][i][e] * inv;
                                da[i][e] = __builtin_fmaf(ga[u][i][e], xa, da[i][e]);
                                db[i][e] = __builtin_fmaf(gb[u][i][e], xb, db[i][e]);
                                ga[u][i][e] *= wa[i][e];
                                gb[u][i][e] *= wb[i][e];
                                dot = __builtin_fmaf(ga[u][i][e], xa, __builtin_fmaf(gb[u][i][e], xb, dot));
                                a[u][i][e] = xa;
                                b[u][i][e] = xb;
                            }
                        }
                        for (int32_t m = 1; m < (1 << lp_log2); m <<= 1) dot += __shfl_xor(dot, m);
                        dot *= inv_dim;
                    }
                    if (!live[u]) continue;
                    T* __restrict__ ov = out + (row0 + r) * s.o_row + h * s.o_head;
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const int32_t p = lane + i * 64;
                        if (p >= g.pairs) continue;
                        const Where<VW, INTER> w(p, half, dim);
                        if constexpr (OP == OP_NORM) {
                            if (per_head) {
                                const float* wp = s.weight + h * s.w_stride;
#pragma unroll
                                for (int e = 0; e < VW; ++e) {
                                    wa[i][e] = wp[w.a + e];
                                    if (w.b >= 0) wb[i][e] = wp[w.b + e];
                                }
                            }
#pragma unroll
                            for (int e = 0; e < VW; ++e) {
                                a[u][i][e] = a[u][i][e] * inv * wa[i][e];
                                b[u][i][e] = b[u][i][e] * inv * wb[i][e];
                            }
                        }
                        if constexpr (OP == OP_NORM_BWD) {
#pragma unroll
                            for (int e = 0; e < VW; ++e) {
                                a[u][i][e] = inv * __builtin_fmaf(-a[u][i][e], dot, ga[u][i][e]);
                                b[u][i][e] = inv * __builtin_fmaf(-b[u][i][e], dot, gb[u][i][e]);
                            }
                        } else if (w.t >= 0) {
                            const float2* __restrict__ cs = s_cs + r * half + w.t;
                            if constexpr (INTER && VW > 1) {
#pragma unroll
                                for (int e = 0; e < VW; e += 2) {
                                    turn(a[u][i][e], a[u][i][e + 1], cs[e / 2].x, cs[e / 2].y);
                                    turn(b[u][i][e], b[u][i][e + 1], cs[VW / 2 + e / 2].x, cs[VW / 2 + e / 2].y);
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < VW; ++e) turn(a[u][i][e], b[u][i][e], cs[e].x, cs[e].y);
                            }
                        }
                        Vec<T, VW> oa, ob;
#pragma unroll
                        for (int e = 0; e < VW; ++e) oa.e[e] = (T)a[u][i][e], ob.e[e] = (T)b[u][i][e];
                        *reinterpret_cast<Vec<T, VW>*>(ov + w.a) = oa;
                        if (w.b >= 0) *reinterpret_cast<Vec<T, VW>*>(ov + w.b) = ob;
                    }
                }
            }
        }
        if constexpr (OP == OP_NORM_BWD) {
            // the block's sum over its groups, in group order (a tree would need a barrier a level): s_cs is free here
            if (s.partial != nullptr) {
                float* s_w = reinterpret_cast<float*>(s_cs);            // [groups][dim] in slices of as many groups as fit
                const int32_t fit = TABLE_MAX * 2 / dim;                // >= 4
                const int64_t cols = per_head ? (int64_t)s.heads * dim : dim;
                float* dst = s.partial + (int64_t)block * cols + (one_head ? (int64_t)pass * dim : 0);
                for (int32_t g0 = 0; g0 < groups; g0 += fit) {
                    const int32_t in = groups - g0 < fit ? groups - g0 : fit;
                    __syncthreads();
                    if (group >= g0 && group < g0 + in) {
#pragma unroll
                        for (int i = 0; i < NI; ++i) {
                            const int32_t p = lane + i * 64;
                            if (p >= g.pairs) continue;
                            const Where<VW, INTER> w(p, half, dim);
#pragma unroll
                            for (int e = 0; e < VW; ++e) {
                                s_w[(group - g0) * dim + w.a + e] = da[i][e];
                                if (w.b >= 0) s_w[(group - g0) * dim + w.b + e] = db[i][e];
                            }
                        }
                    }
                    __syncthreads();
                    for (int32_t d = threadIdx.x; d < dim; d += BLOCK) {
                        float acc = g0 == 0 ? 0.0f : dst[d];
                        for (int32_t k = 0; k < in; ++k) acc += s_w[k * dim + d];
                        dst[d] = acc;
                    }
                }
                __syncthreads();
            }
        }
    }
}

// out[c] = sum over the blocks' rows of partial[b][c], rows of a column dealt to 16 threads, then in thread order
constexpr int SUM_ROWS = 16, SUM_COLS = 64;
struct SumArgs {
    const float* partial[2];
    float* out[2];
    int64_t cols[2];
    int32_t rows[2], blocks0;
};
__global__ __launch_bounds__(SUM_ROWS * SUM_COLS) void sum_rows_kernel(SumArgs a) {
    __shared__ float s_sum[SUM_ROWS][SUM_COLS];
    const int second = (int32_t)blockIdx.x >= a.blocks0;
    const int64_t c = (int64_t)((int32_t)blockIdx.x - (second ? a.blocks0 : 0)) * SUM_COLS + threadIdx.x % SUM_COLS;
    const int32_t r0 = threadIdx.x / SUM_COLS;
    const float* __restrict__ p = a.partial[second];
    const int64_t cols = a.cols[second];
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < cols) {
        int32_t r = r0;
        for (; r + 3 * SUM_ROWS < a.rows[second]; r += 4 * SUM_ROWS) {
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[u] += p[(int64_t)(r + u * SUM_ROWS) * cols + c];
        }
        for (; r < a.rows[second]; r += SUM_ROWS) acc[0] += p[(int64_t)r * cols + c];
    }
    s_sum[r0][threadIdx.x % SUM_COLS] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    __syncthreads();
    if (r0 == 0 && c < cols) {
        float t = 0.f;
        for (int k = 0; k < SUM_ROWS; ++k) t += s_sum[k][threadIdx.x];
        a.out[second][c] = t;
    }
}

int64_t item_bytes(int32_t dtype) { return dtype == SGL_DT_F32 ? 4 : (dtype == SGL_DT_BF16 || dtype == SGL_DT_F16) ? 2 : 0; }

int32_t check_params(const char* what, const sgl_rotary_params* p) {
    if (!p) return fail(SGL_EINVAL, "%s: params is NULL", what);
    if (!item_bytes(p->dtype)) return fail(SGL_EINVAL, "%s: bad dtype", what);
    if (p->dim < 1 || p->dim > DIM_MAX) return fail(SGL_ENOTSUP, "%s: dim must lie in [1, %d]", what, DIM_MAX);
    if (p->rot_dim < 0 || p->rot_dim > p->dim || p->rot_dim % 2) return fail(SGL_EINVAL, "%s: rot_dim must be even and in [0, dim]", what);
    if (p->rot_dim > 0 && !p->freq) return fail(SGL_EINVAL, "%s: freq is NULL", what);
    return SGL_OK;
}

// the widest vector (in values) that keeps every access of the rows aligned and inside one part of the head
struct Width {
    int32_t vw;
    Width(const sgl_rotary_params* p) : vw((int32_t)(16 / item_bytes(p->dtype))) {
        const int32_t half = p->rot_dim / 2;
        while (vw > 1 && (p->dim % vw || half % vw)) vw /= 2;
    }
    void rows(const void* base, int64_t row, int64_t head, int64_t item) {
        while (vw > 1 && (row % vw || head % vw || reinterpret_cast<uintptr_t>(base) % (uintptr_t)(vw * item))) vw /= 2;
    }
};

void set_args(Args& g, const sgl_rotary_params* p, double eps, int vw) {
    g.dim = p->dim;
    g.half = p->rot_dim / 2;
    g.inverse = p->inverse;
    g.amplitude = (float)p->amplitude;
    g.eps = (float)eps;
    g.freq = p->freq;
    const int32_t rest = p->dim - p->rot_dim;
    g.pairs = g.half / vw + (rest + 2 * vw - 1) / (2 * vw);
}

int lanes_log2(int32_t pairs) {
    int l = 0;
    while ((1 << l) < pairs && l < 6) ++l;
    return l;
}

// Rows of a tile: enough (row, head) vectors for every group to get `trips` of them, within the table and the range of
// fast_div.  Four trips amortise the barriers of a tile (120000 rows of 2 heads of 50, fp32, with 1, 4, 8 trips: 39, 27, 28
// us; norm of 65536 events, 40 heads of 64, bf16, forward: 187, 133 us with 1, 4); a call too small to give the chip's 256 CUs
// four blocks each at that size gets one trip.
void set_side(Side& s, int32_t heads, int64_t N_max, int lp_log2, int32_t half, int64_t max_blocks) {
    s.heads = heads;
    s.N_max = N_max;
    s.heads_div = heads == 1 ? 0 : (uint32_t)(((1ull << 32) + heads - 1) / heads);
    const int64_t groups = BLOCK >> lp_log2;
    auto rows_for = [&](int64_t trips) {
        int64_t r = groups * trips / heads;
        if (half > 0 && r > TABLE_MAX / half) r = TABLE_MAX / half;
        if (r * heads > 65535) r = 65535 / heads;
        return r < 1 ? (int64_t)1 : r;
    };
    int64_t rows = rows_for(4);
    if (ceil_div<int64_t>(N_max, rows) < 1024) rows = rows_for(1);
    s.rows = (int32_t)rows;
    int64_t blocks = ceil_div<int64_t>(N_max, rows);
    if (blocks > max_blocks) blocks = max_blocks;
    s.blocks = (int32_t)blocks;
}

template <typename T, int VW, int OP>
void launch(const Args& g, int64_t blocks, bool inter, hipStream_t st) {
    const int l = lanes_log2(g.pairs);
    const int32_t rows = g.s[0].rows > g.s[1].rows ? g.s[0].rows : g.s[1].rows;
    size_t lds = (size_t)rows * g.half * sizeof(float2);
    if (OP == OP_NORM_BWD) lds = TABLE_MAX * sizeof(float2);            // the sum of the groups uses all of it
    const dim3 grid((unsigned)blocks), block(BLOCK);
    if (g.pairs <= 64) {
        if (inter) hipLaunchKernelGGL((rows_kernel<T, VW, true, 1, OP>), grid, block, lds, st, g, l);
        else hipLaunchKernelGGL((rows_kernel<T, VW, false, 1, OP>), grid, block, lds, st, g, l);
    } else if constexpr (VW == 1) {
        if (inter) hipLaunchKernelGGL((rows_kernel<T, VW, true, 8, OP>), grid, block, lds, st, g, l);
        else hipLaunchKernelGGL((rows_kernel<T, VW, false, 8, OP>), grid, block, lds, st, g, l);
    } else if constexpr (sizeof(T) == 4 || VW <= 4) {
        if (inter) hipLaunchKernelGGL((rows_kernel<T, VW, true, 4, OP>), grid, block, lds, st, g, l);
        else hipLaunchKernelGGL((rows_kernel<T, VW, false, 4, OP>), grid, block, lds, st, g, l);
    }
}

template <typename T, int OP>
void launch_width(const Args& g, int64_t blocks, int vw, bool inter, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (vw == 8) return launch<T, 8, OP>(g, blocks, inter, st);
    }
    if (vw == 4) return launch<T, 4, OP>(g, blocks, inter, st);
    if (vw == 2) return launch<T, 2, OP>(g, blocks, inter, st);
    launch<T, 1, OP>(g, blocks, inter, st);
}

template <int OP>
void launch_op(const Args& g, int64_t blocks, int vw, const sgl_rotary_params* p, hipStream_t st) {
    const bool inter = p->interleaved != 0;
    if (p->dtype == SGL_DT_F32) launch_width<float, OP>(g, blocks, vw, inter, st);
    else if (p->dtype == SGL_DT_BF16) launch_width<__bf16, OP>(g, blocks, vw, inter, st);
    else launch_width<_Float16, OP>(g, blocks, vw, inter, st);
}

constexpr int64_t GRID_MAX = 0x3FFFFF;

int32_t check_side(const char* what, const sgl_rotary_params* p, const sgl_norm_side& s, bool backward) {
    if (s.N_max < 0 || s.heads < 1 || s.heads > 65535) return fail(SGL_EINVAL, "%s: N_max < 0 or heads outside [1, 65535]", what);
    if (s.weight_stride != 0 && s.weight_stride != p->dim) return fail(SGL_EINVAL, "%s: weight_stride must be 0 or dim", what);
    if (s.weight_stride != 0 && !s.weight) return fail(SGL_EINVAL, "%s: weight_stride without weights", what);
    if (s.N_max == 0) return SGL_OK;
    if (!s.x.data || !s.y.data || (backward && !s.dx.data)) return fail(SGL_EINVAL, "%s: rows are NULL", what);
    if (p->rot_dim > 0 && !s.pos) return fail(SGL_EINVAL, "%s: pos is NULL", what);
    return SGL_OK;
}

// the backward's tile and grid of one side (what the workspace is sized by too)
Side bwd_side(const sgl_rotary_params* p, const sgl_norm_side& n, int vw) {
    Args g{};
    set_args(g, p, 0.0, vw);
    Side s{};
    set_side(s, n.heads, n.N_max, lanes_log2(g.pairs), g.half, NORM_BWD_BLOCKS);
    return s;
}

int64_t weight_cols(const sgl_rotary_params* p, const sgl_norm_side& n) { return n.weight_stride ? (int64_t)n.heads * p->dim : p->dim; }

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" int32_t sgl_rotary(const sgl_rotary_params* p, int32_t heads, const sgl_rows* x, const int64_t* pos, int64_t N_max,
                              const int64_t* N_dev, const sgl_rows* out, void* stream) {
    if (int32_t rc = check_params("rotary", p)) return rc;
    if (N_max < 0 || heads < 1 || heads > 65535) return fail(SGL_EINVAL, "rotary: N_max < 0 or heads outside [1, 65535]");
    if (N_max == 0) return SGL_OK;
    if (!x || !out || !x->data || !out->data) return fail(SGL_EINVAL, "rotary: x/out is NULL");
    if (p->rot_dim > 0 && !pos) return fail(SGL_EINVAL, "rotary: pos is NULL");
    Width w(p);
    w.rows(x->data, x->row_stride, x->head_stride, item_bytes(p->dtype));
    w.rows(out->data, out->row_stride, out->head_stride, item_bytes(p->dtype));
    Args g{};
    set_args(g, p, 0.0, w.vw);
    Side& s = g.s[0];
    s.x = x->data, s.x_row = x->row_stride, s.x_head = x->head_stride;
    s.out = out->data, s.o_row = out->row_stride, s.o_head = out->head_stride;
    s.pos = pos, s.N_dev = N_dev;
    set_side(s, heads, N_max, lanes_log2(g.pairs), g.half, GRID_MAX);
    g.blocks0 = s.blocks;
    launch_op<OP_ROT>(g, s.blocks, w.vw, p, as_stream(stream));
    SGL_LAUNCH_CHECK();
    return SGL_OK;
}

extern "C" int32_t sgl_qk_norm_rotary(const sgl_rotary_params* p, double eps, int32_t num, const sgl_norm_side* sides, void* stream) {
    if (int32_t rc = check_params("qk_norm_rotary", p)) return rc;
    if (num < 1 || num > 2 || !sides) return fail(SGL_EINVAL, "qk_norm_rotary: one or two sides");
    if (p->inverse) return fail(SGL_EINVAL, "qk_norm_rotary: inverse is for sgl_rotary");
    Width w(p);
    for (int i = 0; i < num; ++i) {
        if (int32_t rc = check_side("qk_norm_rotary", p, sides[i], false)) return rc;
        if (sides[i].N_max == 0) continue;
        w.rows(sides[i].x.data, sides[i].x.row_stride, sides[i].x.head_stride, item_bytes(p->dtype));
        w.rows(sides[i].y.data, sides[i].y.row_stride, sides[i].y.head_stride, item_bytes(p->dtype));
    }
    Args g{};
    set_args(g, p, eps, w.vw);
    int64_t blocks = 0;
    for (int i = 0; i < num; ++i) {
        const sgl_norm_side& n = sides[i];
        Side& s = g.s[i];
        s.x = n.x.data, s.x_row = n.x.row_stride, s.x_head = n.x.head_stride;
        s.out = n.y.data, s.o_row = n.y.row_stride, s.o_head = n.y.head_stride;
        s.pos = n.pos, s.N_dev = n.N_dev, s.weight = n.weight, s.w_stride = n.weight_stride;
        set_side(s, n.heads, n.N_max, lanes_log2(g.pairs), g.half, GRID_MAX);
        if (i == 0) g.blocks0 = s.blocks;
        blocks += s.blocks;
    }
    if (blocks == 0) return SGL_OK;
    launch_op<OP_NORM>(g, blocks, w.vw, p, as_stream(stream));
    SGL_LAUNCH_CHECK();
    return SGL_OK;
}

extern "C" size_t sgl_qk_norm_rotary_backward_workspace_bytes(const sgl_rotary_params* p, int32_t num, const sgl_norm_side* sides) {
    if (check_params("qk_norm_rotary_backward", p) || num < 1 || num > 2 || !sides) return 0;
    size_t total = 0;
    for (int i = 0; i < num; ++i)
        total += align_up((size_t)NORM_BWD_BLOCKS * (size_t)weight_cols(p, sides[i]) * sizeof(float));
    return total;
}

extern "C" int32_t sgl_qk_norm_rotary_backward(const sgl_rotary_params* p, double eps, int32_t num, const sgl_norm_side* sides,
                                               void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t rc = check_params("qk_norm_rotary_backward", p)) return rc;
    if (num < 1 || num > 2 || !sides) return fail(SGL_EINVAL, "qk_norm_rotary_backward: one or two sides");
    if (p->inverse) return fail(SGL_EINVAL, "qk_norm_rotary_backward: inverse is for sgl_rotary");
    Width w(p);
    const int64_t item = item_bytes(p->dtype);
    for (int i = 0; i < num; ++i) {
        const sgl_norm_side& n = sides[i];
        if (int32_t rc = check_side("qk_norm_rotary_backward", p, n, true)) return rc;
        if (n.N_max == 0) continue;
        w.rows(n.x.data, n.x.row_stride, n.x.head_stride, item);
        w.rows(n.y.data, n.y.row_stride, n.y.head_stride, item);
        w.rows(n.dx.data, n.dx.row_stride, n.dx.head_stride, item);
    }
    Args g{};
    set_args(g, p, eps, w.vw);
    Arena ws(workspace, workspace_bytes);
    SumArgs sum{};
    int64_t blocks = 0, sum_blocks = 0;
    bool any = false;
    for (int i = 0; i < num; ++i) {
        const sgl_norm_side& n = sides[i];
        Side& s = g.s[i];
        s = bwd_side(p, n, w.vw);
        s.x = n.x.data, s.x_row = n.x.row_stride, s.x_head = n.x.head_stride;
        s.y = n.y.data, s.y_row = n.y.row_stride, s.y_head = n.y.head_stride;
        s.out = n.dx.data, s.o_row = n.dx.row_stride, s.o_head = n.dx.head_stride;
        s.pos = n.pos, s.N_dev = n.N_dev, s.weight = n.weight, s.w_stride = n.weight_stride;
        const int64_t cols = weight_cols(p, n);
        float* part = ws.take<float>((size_t)NORM_BWD_BLOCKS * (size_t)cols);
        if (n.dweight) {
            any = true;
            s.partial = part;
            sum.partial[i] = part, sum.out[i] = n.dweight, sum.cols[i] = cols, sum.rows[i] = s.blocks;
            sum_blocks += ceil_div<int64_t>(cols, SUM_COLS);
        }
        if (i == 0) g.blocks0 = s.blocks, sum.blocks0 = (int32_t)sum_blocks;
        blocks += s.blocks;
    }
    if (any && !ws.ok()) return fail(SGL_ENOMEM, "qk_norm_rotary_backward: workspace of %zu bytes, %zu needed", workspace_bytes, ws.used);
    if (blocks > 0) {
        launch_op<OP_NORM_BWD>(g, blocks, w.vw, p, as_stream(stream));
        SGL_LAUNCH_CHECK();
    }
    if (sum_blocks > 0) {       // (a side without rows has no partial rows: its gradient is zero)
        hipLaunchKernelGGL(sum_rows_kernel, dim3((unsigned)sum_blocks), dim3(SUM_ROWS * SUM_COLS), 0, as_stream(stream), sum);
        SGL_LAUNCH_CHECK();
    }
    return SGL_OK;
}
