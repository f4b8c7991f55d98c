// Shared parts of the differential attention kernels: argument block, the span of keys a query sees, and the 32 x 32
// matrix tiles (fragments, LDS images, staging).
#pragma once

#include <math.h>

#include "common.hpp"

namespace sgl {
namespace attn {

constexpr int BLOCK = 256;
constexpr float NEG_INF = -INFINITY;
constexpr float LOG2E = 1.44269504088896340736f;

struct AttnArgs {
    sgl_diff_attn_args a;
    float scale;                // of the scores
    float c2;                   // |scale| log2(e): scores enter exponentials of base 2
    int32_t negate;             // scale < 0: the operand that stays in registers changes its sign (exact)
    int32_t aligned;            // every row of q, k, v (and of the gradients read) is a whole number of 16-byte chunks
    int32_t parts;              // forward: partial results per (row, head, map), joined by a second kernel; 1: none
    float* part_ml;             // [parts, Tq * Hq, 2, 2]: running maximum (in powers of two) and sum
    float* part_o;              // [parts, Tq * Hq, 2, Dv]
    float* delta;               // backward [Tq, Hq, 2]: t_1, t_2
    int32_t* spans;             // backward [Tq, 2]: the keys that a row sees, before key_mask
    float* lam_part;            // backward [row tiles, Hq]: sums of t_2
};

inline AttnArgs attn_args(const sgl_diff_attn_args& a) {
    AttnArgs g{};
    g.a = a;
    g.scale = (float)a.scale;
    // a scale of zero must not turn the -inf of a hidden score into a NaN: with 1e-30 every visible score vanishes too
    g.c2 = fmaxf(fabsf(g.scale) * LOG2E, 1e-30f);
    g.negate = g.scale < 0.f;
    g.parts = 1;
    return g;
}

#if defined(__HIPCC__)

// the sequence of element i: the last b with ptr[b] <= i < ptr[b + 1], -1 if there is none
__device__ __forceinline__ int32_t find_seq(const int64_t* __restrict__ ptr, int32_t B, int64_t i) {
    if (B <= 0 || i < ptr[0] || i >= ptr[B]) return -1;
    int32_t lo = 0, hi = B;                       // ptr[lo] <= i < ptr[hi]
    while (hi - lo > 1) {
        const int32_t mid = lo + (hi - lo) / 2;
        if (ptr[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int32_t clamp_to(int64_t x, int64_t n) { return (int32_t)(x < 0 ? 0 : (x > n ? n : x)); }

struct Span {
    int32_t lo, hi;             // [lo, hi); lo == hi: nothing
};

// keys that query row i of sequence seq sees (before key_mask)
__device__ __forceinline__ Span keys_of(const sgl_diff_attn_args& a, int32_t seq, int64_t i) {
    Span s{0, 0};
    if (seq < 0) return s;
    const int32_t k0 = clamp_to(a.k_ptr[seq], a.Tk), k1 = clamp_to(a.k_ptr[seq + 1], a.Tk);
    int64_t lo = k0, hi = k1;
    if (a.causal) {
        const int64_t last = k1 - (a.q_ptr ? a.q_ptr[seq + 1] - i : 1);       // the key that stands where the query does
        if (last + 1 < hi) hi = last + 1;
        if (a.window > 0 && last + 1 - a.window > lo) lo = last + 1 - a.window;
    }
    if (hi <= lo) return s;
    s.lo = (int32_t)lo;
    s.hi = (int32_t)hi;
    return s;
}

template <typename T>
__device__ __forceinline__ const T* row(const sgl_rows& r, int64_t n, int64_t h) {
    return static_cast<const T*>(r.data) + n * r.row_stride + h * r.head_stride;
}
template <typename T>
__device__ __forceinline__ T* row_out(const sgl_rows& r, int64_t n, int64_t h) {
    return static_cast<T*>(r.data) + n * r.row_stride + h * r.head_stride;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }     // below 2^-126: 0

// the other half's value of a reduction over lanes l and l ^ 32
__device__ __forceinline__ float half_max(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return fmaxf(__int_as_float(s[0]), __int_as_float(s[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
    return __int_as_float(s[0]) + __int_as_float(s[1]);
}

// ------------------------------------------------------------------------------------------------- matrix tiles
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define SGL_LDS __attribute__((address_space(3)))
#define SGL_GLOBAL __attribute__((address_space(1)))

// A fragment is 16 bytes of one row of an operand: EP elements.  A step contracts over 2 EP of them (32 bytes of a row:
// lanes 0-31 hold its first half, lanes 32-63 the second).  In the fp32 form, whose instruction takes two elements, a
// step is four instructions; both operands order the elements the same way, so the order is free.
//   result: column l & 31, rows 8 (r / 4) + 4 (l >> 5) + r % 4 of register r
template <typename T>
struct Mat;
template <>
struct Mat<__bf16> {
    typedef bf16x8 Frag;
    static constexpr int EP = 8;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mat<_Float16> {
    typedef f16x8 Frag;
    static constexpr int EP = 8;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mat<float> {
    typedef f32x4 Frag;
    static constexpr int EP = 4;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

// fp32 results of rows (of the result above) 2 EP s .. 2 EP (s + 1) as the right operand of a step that contracts over
// them: the registers EP s .. EP s + EP - 1 of a lane, which stand for the rows `row_of(s, j, half)`
template <typename T>
__device__ __forceinline__ typename Mat<T>::Frag to_frag(const f32x16& x, int s) {
    typename Mat<T>::Frag f;
#pragma unroll
    for (int j = 0; j < Mat<T>::EP; ++j) f[j] = (T)x[s * Mat<T>::EP + j];
    return f;
}
template <typename T>
__device__ __forceinline__ int row_of(int s, int j, int half) {
    return 2 * Mat<T>::EP * s + 8 * (j / 4) + 4 * half + j % 4;
}

// LDS image of rows of RB bytes: pieces of 8 rows x 8 chunks (16 bytes each), 1 KB, the pieces of 8 rows side by side; chunk c
// of row r lies in its piece's row r % 8 at place (c ^ r) % 8.  Eight lanes that read one chunk column, and the sixteen that
// read two columns of four rows (the transposed reads), then meet different banks; a piece is what one wave brings in at a time
// (8 whole lines of 128 bytes); and an address is a lane's part plus a constant but for the two bits of the exchange.
template <int RB>
__device__ __forceinline__ int at(int r, int chunk) {
    return ((r >> 3) * (RB / 128) + (chunk >> 3)) * 1024 + (r & 7) * 128 + (((chunk ^ r) & 7) << 4);
}

// row fragment: row r, chunk 2 i + half
template <typename T, int RB>
__device__ __forceinline__ typename Mat<T>::Frag row_frag(const char* tile, int row0, int col, int i, int half) {
    return *reinterpret_cast<const typename Mat<T>::Frag*>(tile + (row0 >> 3) * (RB / 128) * 1024 + (i >> 2) * 1024 + (col >> 3) * (RB / 128) * 1024 +
                                                           (col & 7) * 128 + ((((2 * i) & 7) ^ (half ^ (col & 7))) << 4));
}

// column fragment: elements (row0 + row_of(s, j, half), 32 t + lane column): the transposed left operand whose 32 rows are
// the 32 elements from 32 t of the tile's rows
template <typename T, int RB>
__device__ __forceinline__ typename Mat<T>::Frag col_frag(const char* tile, int row0, int s, int t, int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        const int r = 4 * half + ((lane & 15) >> 2), c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);       // chunk 4 t + c
        const int base = (row0 / 8 + 2 * s) * (RB / 128) * 1024 + (t >> 1) * 1024 + r * 128 + ((((4 * t) & 7) ^ (c ^ r)) << 4) + (lane & 1) * 8;
        typedef SGL_LDS s16x4 lds4;
        union {
            s16x8 v;
            typename Mat<T>::Frag f;
        } u;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + base));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(tile + base + (RB / 128) * 1024));
        u.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return u.f;
    } else {
        typename Mat<T>::Frag f;
        const int c = (lane & 31) >> 2;                                                                      // chunk 8 t + c
#pragma unroll
        for (int j = 0; j < 4; ++j)
            f[j] = *reinterpret_cast<const float*>(tile + ((row0 / 8 + s) * (RB / 128) + t) * 1024 + (4 * half + j) * 128 + ((c ^ (4 * half + j)) << 4) + (lane & 3) * 4);
        return f;
    }
}

// where chunk c of a staged row comes from: the two halves of a head ([2][D], D <= DP each), or one head of Dv <= 2 DP
struct Source {
    const void* data;
    int64_t row_stride;
    int64_t half_stride;        // elements from the first half to the second; 0: one run
    int32_t len;                // valid elements of a half (D), or of the run (Dv)
};

template <typename T>
__device__ __forceinline__ Source halves(const sgl_rows& r, int head, int D) {
    return Source{static_cast<const T*>(r.data) + (int64_t)(2 * head) * r.head_stride, r.row_stride, r.head_stride, D};
}
template <typename T>
__device__ __forceinline__ Source run(const sgl_rows& r, int head, int Dv) {
    return Source{static_cast<const T*>(r.data) + (int64_t)head * r.head_stride, r.row_stride, 0, Dv};
}

// Stage ROWS rows from row0 (rows beyond `last` repeat it: their columns are hidden) into the image of RB-byte rows, by
// NT threads.  DMA: every chunk is whole and aligned, and goes from memory to LDS without passing through registers (a
// wave's 64 chunks land side by side, so the swizzle is applied to what each lane fetches); complete after
// staged().  Otherwise through registers, with zeros behind a row's valid elements.
template <typename T, int DP, int ROWS, int NT, bool DMA>
__device__ __forceinline__ void stage(char* tile, const Source& s, bool two, int32_t row0, int32_t last, int aligned) {
    constexpr int RB = 2 * DP * (int)sizeof(T), CH = RB / 16, EP = 16 / (int)sizeof(T);
    const T* __restrict__ base = static_cast<const T*>(s.data);
    if constexpr (DMA) {
#pragma unroll
        for (int i0 = 0; i0 < ROWS * CH; i0 += NT) {
            const int i = i0 + threadIdx.x, piece = i >> 6;
            const int r = piece / (CH / 8) * 8 + ((i >> 3) & 7), c = piece % (CH / 8) * 8 + ((i ^ (i >> 3)) & 7);
            const int32_t n = row0 + r < last ? row0 + r : last;
            const T* src = base + (int64_t)n * s.row_stride + (two ? (c / (CH / 2)) * s.half_stride + (c % (CH / 2)) * EP : c * EP);
            const int wave0 = __builtin_amdgcn_readfirstlane(i0 + ((int)threadIdx.x & ~63));
            __builtin_amdgcn_global_load_lds((SGL_GLOBAL void*)src, (SGL_LDS void*)(tile + wave0 * 16), 16, 0, 0);
        }
    } else {
        typedef typename Mat<T>::Frag Frag;
        for (int i = threadIdx.x; i < ROWS * CH; i += NT) {
            const int r = i / CH, c = i % CH;
            const int32_t n = row0 + r < last ? row0 + r : last;
            const int e = two ? (c % (CH / 2)) * EP : c * EP;
            const T* src = base + (int64_t)n * s.row_stride + (two ? (c / (CH / 2)) * s.half_stride : 0) + e;
            Frag f;
            if (aligned && e + EP <= s.len) {
                f = *reinterpret_cast<const Frag*>(src);
            } else {
#pragma unroll
                for (int j = 0; j < EP; ++j) f[j] = e + j < s.len ? src[j] : (T)0.0f;
            }
            *reinterpret_cast<Frag*>(tile + at<RB>(r, c)) = f;
        }
    }
}

// this wave's DMA has landed and every wave's has once the block is past the barrier
__device__ __forceinline__ void staged() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// fragment `chunk` (of EP elements) of a row kept in registers; zero where the row is not live or beyond len
template <typename T>
__device__ __forceinline__ typename Mat<T>::Frag global_frag(const T* src, int e, int len, bool live, int aligned, bool negate) {
    typename Mat<T>::Frag f;
    constexpr int EP = Mat<T>::EP;
    if (live && aligned && e + EP <= len) {
        f = *reinterpret_cast<const typename Mat<T>::Frag*>(src + e);
    } else {
#pragma unroll
        for (int j = 0; j < EP; ++j) f[j] = live && e + j < len ? src[e + j] : (T)0.0f;
    }
    if (negate) {
#pragma unroll
        for (int j = 0; j < EP; ++j) f[j] = -f[j];
    }
    return f;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

// Work item of a block: consecutive items of one XCD (blocks go to the 8 of them in turn) are neighbours, so that what they
// share lies in one L2.  The grid is a multiple of 8; items >= n do nothing.
__device__ __forceinline__ int64_t xcd_item(int64_t n) {
    const int64_t per = ceil_div<int64_t>(n, 8), b = blockIdx.x;
    return (b % 8) * per + b / 8;
}

// smallest and largest over a wave
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = min(x, __shfl_xor(x, m));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) { return -wave_min(-x); }

// 32 keys [j0, j0 + 32) of a lane's column that it does not see become -inf: column span [lo, hi), key mask
__device__ __forceinline__ void hide(f32x16& s, int32_t j0, int half, Span span, const uint8_t* __restrict__ mask, int32_t last) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int32_t j = j0 + 8 * (r / 4) + 4 * half + r % 4;
        bool see = j >= span.lo && j < span.hi;
        if (mask != nullptr) see = see && mask[j < last ? j : last];
        s[r] = see ? s[r] : NEG_INF;
    }
}
__device__ __forceinline__ bool sees(int32_t j, Span span, const uint8_t* __restrict__ mask) {
    return j >= span.lo && j < span.hi && (mask == nullptr || mask[j]);
}

#endif  // __HIPCC__

// Host side.  Forward on the matrix units: tiles of query rows, or (without q_ptr) of the heads of a group.
struct FwdWork {
    int64_t items;              // blocks with work
    int32_t tiles;              // row tiles, or sequences
    int32_t groups;             // without q_ptr: column tiles of a head group
    int32_t splits;             // parts of a key range
};
FwdWork forward_work(const sgl_diff_attn_args& a);
// the narrower of the three widths 32, 64, 128 that holds D and half of Dv is the matrix kernels' head width
inline int heads_width(const sgl_diff_attn_args& a) { return a.D > (a.Dv + 1) / 2 ? a.D : (a.Dv + 1) / 2; }
// one query per sequence without matrix units
template <int N>
struct Int {
    static constexpr int value = N;
};
int64_t seg_blocks(const sgl_diff_attn_args& a);
void seg_forward(const AttnArgs& g, hipStream_t st);
void seg_backward(const AttnArgs& g, hipStream_t st);
template <typename T>
void forward_type(const AttnArgs& g, hipStream_t st);
template <typename T>
void backward_type(const AttnArgs& g, hipStream_t st);

}  // namespace attn
}  // namespace sgl
