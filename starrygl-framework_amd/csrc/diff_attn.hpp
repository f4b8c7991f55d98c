// Shared parts of the differential attention kernels: argument block, the span of keys a query sees, and the 32 x 32
// matrix tiles (fragments, LDS images, staging).
#pragma once

#include <math.h>

#include <initializer_list>

#include "common.hpp"

namespace sgl {
namespace attn {

constexpr int BLOCK = 256;
constexpr float NEG_INF = -INFINITY;
constexpr float LOG2E = 1.44269504088896340736f;

constexpr int64_t GRID_PART = 1 << 22;      // blocks of a launch, a multiple of 8 (a launch takes less than 2^32 threads)
constexpr int QUERY_ROWS = 128;     // query rows of a block of the backward pass (a sum of t_2 in the workspace each)

// How rows come into LDS: through registers, whole (as wide as the image), or padded (narrower, in whole 16-byte chunks)
enum { BY_REGISTERS, WHOLE_ROWS, PADDED };

struct AttnArgs {
    sgl_diff_attn_args a;
    float scale;                // of the scores
    float c2;                   // |scale| log2(e): scores enter exponentials of base 2
    int32_t negate;             // scale < 0: the operand that stays in registers changes its sign (exact)
    int32_t grain;              // bytes, 16 at most, that divide the address of every row and the length of every row's head
    int32_t map_grain;          // the same of the rows of `maps`
    int32_t parts;              // forward: partial results per (row, head, map), joined by a second kernel; 1: none
    int64_t first;              // first block of a launch: large grids go out in parts
    float* part_ml;             // [parts, Tq * Hq, 2, 2]: running maximum (in powers of two) and sum
    float* part_o;              // [parts, Tq * Hq, 2, Dv]
    float* delta;               // backward [Tq, Hq, 2]: t_1, t_2
    float* lam_part;            // backward [row tiles, Hq]: sums of t_2
};

inline AttnArgs attn_args(const sgl_diff_attn_args& a) {
    AttnArgs g{};
    g.a = a;
    if (a.window > 0x7FFFFFFF) g.a.window = 0;      // wider than any sequence
    g.scale = (float)a.scale;
    // a scale of zero must not turn the -inf of a hidden score into a NaN: with 2^-149 every visible score vanishes too
    g.c2 = fmaxf(fabsf(g.scale) * LOG2E, 0x1p-149f);
    g.negate = g.scale < 0.f;
    g.map_grain = a.Dv % 4 == 0 ? 16 : a.Dv % 2 == 0 ? 8 : 4;
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

// The sequences of N elements per lane, first + at[0 .. N), 0 <= at < 64, of one wave (`first` the same in all lanes).  A search
// by halves waits for one load after the other; here the wave looks at 64 entries at a time (one load up to 63 sequences,
// three up to 250000) and the lanes find their own among the 64 that follow.
template <int N>
__device__ __forceinline__ void find_seqs(const int64_t* __restrict__ ptr, int32_t B, int64_t first, const int32_t (&at)[N], int32_t (&seq)[N]) {
    const int lane = threadIdx.x & 63;
    int32_t lo = 0, len = B + 1;                  // the entries at hand: [lo, lo + len)
    while (len > 64) {
        const int32_t step = (len + 63) / 64;
        const int c = __popcll(__ballot(lane * step < len && ptr[lo + min(lane * step, len - 1)] <= first));
        if (c == 0) {
            len = 1;                              // all behind `first`
            break;
        }
        lo += (c - 1) * step;
        len = min(step, B + 1 - lo);
    }
    const int c = __popcll(__ballot(lane < len && ptr[lo + min(lane, len - 1)] <= first));
    const int32_t s0 = lo + c - 1;                // the last entry <= first, -1: none
    // how far the next 64 entries lie behind `first`
    const int32_t k = s0 + 1 + lane;
    const int64_t far = k <= B ? ptr[k] - first : 64;
    const int32_t next = (int32_t)min(far, (int64_t)64);
#pragma unroll
    for (int n = 0; n < N; ++n) seq[n] = s0;
    if (__builtin_amdgcn_readfirstlane(next) < 64) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            int32_t pos = 0;                      // entries <= first + at
#pragma unroll
            for (int w = 32; w > 0; w >>= 1)
                if (__shfl(next, pos + w - 1) <= at[n]) pos += w;
            if (__shfl(next, pos) <= at[n]) ++pos;
            seq[n] = pos < 64 ? s0 + pos : find_seq(ptr, B, first + at[n]);      // (64 empty sequences in a row)
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (seq[n] >= B) seq[n] = -1;
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
        const int64_t last = k1 - (a.q_ptr ? clamp_to(a.q_ptr[seq + 1], a.Tq) - i : 1);       // the key that stands where the query does
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

// where the two numbers of (row, head) lie in lse and delta: rows times heads may need all of 31 bits
__device__ __forceinline__ int64_t pair_at(const sgl_diff_attn_args& a, int64_t i, int h) { return (i * a.Hq + h) * 2; }

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
// them: the registers EP s .. EP s + EP - 1 of a lane, which stand for the rows
// row(s, j, half) = 2 EP s + 8 (j / 4) + 4 half + j % 4
template <typename T>
__device__ __forceinline__ typename Mat<T>::Frag to_frag(const f32x16& x, int s) {
    typename Mat<T>::Frag f;
#pragma unroll
    for (int j = 0; j < Mat<T>::EP; ++j) f[j] = (T)x[s * Mat<T>::EP + j];
    return f;
}

// LDS image of rows of RB bytes: pieces of 8 rows x 8 chunks (16 bytes each), 1 KB, the pieces of 8 rows side by side.  Row r is
// line r & 7 of its pieces, its chunk c lies at place (c ^ mix(r)) & 7 of the line.  A 128-bit read serves 16 lanes a cycle, of
// 32 consecutive rows those with an even (then those with an odd) number of ones in bits 2-4: bits 0-3 tell them apart, and
// one chunk column meets all 64 banks once.  So do the transposed reads (4 columns of 4 rows, whose bit 1 moves the place
// by 4).  A piece is what one wave brings in at a time (8 whole lines of memory); an address is a lane's part plus a
// constant but for the bits of the exchange.
__device__ __forceinline__ constexpr int mix(int r) { return ((r & 2) << 1) | ((r >> 2) & 1) | ((r >> 2) & 2); }
template <int RB>
__device__ __forceinline__ int at(int r, int chunk) {
    return ((r >> 3) * (RB / 128) + (chunk >> 3)) * 1024 + ((r & 7) << 7) + (((chunk ^ mix(r)) & 7) << 4);
}

// row fragment: row row0 + col (row0 a multiple of 16), chunk 2 i + half
template <typename T, int RB>
__device__ __forceinline__ typename Mat<T>::Frag row_frag(const char* tile, int row0, int col, int i, int half) {
    return *reinterpret_cast<const typename Mat<T>::Frag*>(tile + (row0 >> 3) * (RB / 128) * 1024 + (i >> 2) * 1024 + (col >> 3) * (RB / 128) * 1024 +
                                                           ((col & 7) << 7) + ((((2 * i) & 7) ^ (half ^ mix(col))) << 4));
}

// row fragment of half `map` of a head: RB / 32 chunks, whole pieces of 8 or (64-byte halves) half a piece
template <typename T, int RB>
__device__ __forceinline__ typename Mat<T>::Frag map_frag(const char* tile, int row0, int col, int map, int i, int half) {
    if constexpr (RB >= 256) return row_frag<T, RB>(tile + map * (RB / 256) * 1024, row0, col, i, half);
    else return map ? row_frag<T, RB>(tile, row0, col, i + 2, half) : row_frag<T, RB>(tile, row0, col, i, half);
}

// column fragment: elements (row0 + row(s, j, half), 32 t + lane column), row0 a multiple of 16: the transposed left operand
// whose 32 rows are the 32 elements from 32 t of the tile's rows
template <typename T, int RB>
__device__ __forceinline__ typename Mat<T>::Frag col_frag(const char* tile, int row0, int s, int t, int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        const int r = 4 * half + ((lane & 15) >> 2), c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);       // row of a piece, chunk 4 t + c
        const int place = ((((4 * t) & 7) ^ (c ^ mix(r))) << 4) + (lane & 1) * 8;
        const char* base = tile + ((row0 / 8 + 2 * s) * (RB / 128) + (t >> 1)) * 1024;
        typedef SGL_LDS s16x4 lds4;
        union {
            s16x8 v;
            typename Mat<T>::Frag f;
        } u;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(base + (r * 128 + place)));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(base + (RB / 128) * 1024 + (r * 128 + (place ^ 32))));
        u.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return u.f;
    } else {
        typename Mat<T>::Frag f;
        const int c = (lane & 31) >> 2;                                                                      // chunk 8 t + c
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = 4 * half + j;
            f[j] = *reinterpret_cast<const float*>(tile + ((row0 / 8 + s) * (RB / 128) + t) * 1024 + (r << 7) + ((c ^ mix(r + 8 * (s & 1))) << 4) + (lane & 3) * 4);
        }
        return f;
    }
}

// The same by the lane's part of the address, which the caller keeps: of row `col` and chunk 2 i + half (tile + 1024 (i / 4) + part
// i % 4), of the transposed fragment of elements 32 t (part t % 2; fp32: part of rows 8 s, s odd or even).
template <int RB>
__device__ __forceinline__ int32_t lane_row(int col, int i, int half) {
    return (col >> 3) * (RB / 128) * 1024 + ((col & 7) << 7) + ((((2 * i) & 7) ^ (half ^ mix(col))) << 4);
}
template <typename T, int RB>
__device__ __forceinline__ int32_t lane_col(int e, int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        const int r = 4 * half + ((lane & 15) >> 2), c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
        return r * 128 + ((((4 * e) & 7) ^ (c ^ mix(r))) << 4) + (lane & 1) * 8;
    } else {
        const int r = 4 * half, c = (lane & 31) >> 2;
        return (r << 7) + ((c ^ mix(r + 8 * e)) << 4) + (lane & 3) * 4;
    }
}
template <typename T, int RB>
__device__ __forceinline__ typename Mat<T>::Frag col_at(const char* tile, const int32_t (&by)[2], int32_t off, int s, int t) {
    if constexpr (sizeof(T) == 2) {
        const char* base = tile + (2 * s * (RB / 128) + (t >> 1)) * 1024;
        typedef SGL_LDS s16x4 lds4;
        union {
            s16x8 v;
            typename Mat<T>::Frag f;
        } u;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(base + (by[t & 1] + off)));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(base + (RB / 128) * 1024 + ((by[t & 1] ^ 32) + off)));
        u.v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return u.f;
    } else {
        typename Mat<T>::Frag f;
        const char* base = tile + (s * (RB / 128) + t) * 1024;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(base + (j << 7) + ((by[s & 1] ^ (mix(j) << 4)) + off));
        return f;
    }
}

// Fragments 0 .. N - 1 from LDS, `use`d in turn with the next DEPTH on their way.  The order is fixed: left to itself the
// compiler, short of registers, reads each fragment into the same four and waits for it (a read takes as long as four
// products).
template <typename T, int N, int DEPTH>
struct Pipe {
    typename Mat<T>::Frag f[DEPTH];
    template <typename Load>
    __device__ __forceinline__ void fill(Load load) {
#pragma unroll
        for (int n = 0; n < DEPTH && n < N; ++n) f[n] = load(n);
        __builtin_amdgcn_sched_barrier(0);
    }
    template <typename Load, typename Use>
    __device__ __forceinline__ void drain(Load load, Use use) {
        part<0, N>(load, use);
    }
    template <int FROM, int TO, typename Load, typename Use>
    __device__ __forceinline__ void part(Load load, Use use) {
#pragma unroll
        for (int n = FROM; n < TO; ++n) {
            use(n, f[n % DEPTH]);
            if (n + DEPTH < N) f[n % DEPTH] = load(n + DEPTH);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// A chunk of 16 bytes of which `left` elements are a row's (none, where left <= 0), the others zero; rows of other widths than whole
// chunks move in pieces of `grain` bytes (a training step of 8 sequences of 1024, 8 heads, causal: 50 wide in bf16, pieces of 4
// bytes, 466 us; 100 wide in fp16, pieces of 8, 1040 us; element by element 532 and 1407).
template <typename T>
__device__ __forceinline__ typename Mat<T>::Frag load_chunk(const T* src, int left, int grain) {
    constexpr int EP = Mat<T>::EP;
    union {
        typename Mat<T>::Frag f;
        uint4 w16;
        uint2 w8[2];
        uint32_t w4[4];
    } u;
    u.w16 = uint4{0, 0, 0, 0};
    if (grain == 16) {
        if (left > 0) u.w16 = *reinterpret_cast<const uint4*>(src);
    } else if (grain == 8) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (left > k * (EP / 2)) u.w8[k] = reinterpret_cast<const uint2*>(src)[k];
    } else if (grain == 4 || sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (left > k * (EP / 4)) u.w4[k] = reinterpret_cast<const uint32_t*>(src)[k];
    } else {
        typename Mat<T>::Frag f;
#pragma unroll
        for (int k = 0; k < EP; ++k) f[k] = left > k ? src[k] : (T)0.0f;
        return f;
    }
    return u.f;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* dst, const typename Mat<T>::Frag& f, int left, int grain) {
    constexpr int EP = Mat<T>::EP;
    union {
        typename Mat<T>::Frag f;
        uint4 w16;
        uint2 w8[2];
        uint32_t w4[4];
    } u;
    u.f = f;
    if (grain == 16) {
        if (left > 0) *reinterpret_cast<uint4*>(dst) = u.w16;
    } else if (grain == 8) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (left > k * (EP / 2)) reinterpret_cast<uint2*>(dst)[k] = u.w8[k];
    } else if (grain == 4 || sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (left > k * (EP / 4)) reinterpret_cast<uint32_t*>(dst)[k] = u.w4[k];
    } else {
#pragma unroll
        for (int k = 0; k < EP; ++k)
            if (left > k) dst[k] = u.f[k];
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

// whether bit `bits` of register r's row is set, bits shifted by 4 half before
__device__ __forceinline__ bool row_bit(uint32_t bits, int r) { return (bits >> (8 * (r / 4) + r % 4)) & 1; }

// Staging of ROWS rows from row0 (rows beyond `last` repeat it: their columns are hidden) into the image of RB-byte rows by NT
// threads.  DMA: every chunk is whole and aligned, and goes from memory to LDS without passing through registers (a
// wave's 64 chunks land side by side, a piece, so the exchange is applied to what each lane fetches); complete after
// staged().  PADDED: lanes whose chunk lies behind a row's valid elements bring nothing, and what they would write has been zero
// since the caller cleared the image.  Otherwise through registers, with zeros behind a row's valid elements.
template <typename T, int DP, int ROWS, int NT, int MODE, bool TWO>
struct Stager {
    static constexpr bool DMA = MODE != BY_REGISTERS, PAD = MODE == PADDED;
    static constexpr int RB = 2 * DP * (int)sizeof(T), CH = RB / 16, EP = 16 / (int)sizeof(T);
    static constexpr int NW = NT / 64, PG = CH / 8;             // waves; pieces side by side
    static_assert(NW % PG == 0 || PG % NW == 0, "a wave covers whole columns or walks whole rows of pieces");
    // the thread's own part of an address (fits 32 bits: dma_rows); the rest is the same for all lanes
    static constexpr int COLS = PG > NW ? PG / NW : 1;          // columns of pieces that a wave walks through
    static constexpr int KINDS = PG >= NW ? 2 : 1;              // rows of pieces of both parities, or of the wave's own
    int32_t off[COLS][KINDS];
    bool on[COLS][KINDS];

    // row in its tile and chunk of what lane `lane` of piece `piece` brings
    static __device__ __forceinline__ void of_piece(int piece, int lane, int& r, int& c) {
        const int rows8 = piece / PG;
        r = rows8 * 8 + (lane >> 3);
        c = piece % PG * 8 + ((lane ^ mix(r)) & 7);
    }
    static __device__ __forceinline__ int64_t element(const Source& s, int r, int c) {
        return r * s.row_stride + (TWO ? c / (CH / 2) * s.half_stride + c % (CH / 2) * EP : c * EP);
    }
    static __device__ __forceinline__ bool valid(const Source& s, int c) { return (TWO ? c % (CH / 2) : c) * EP < s.len; }
    __device__ __forceinline__ void plan(const Source& s) {
        if constexpr (DMA) {
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
            for (int p = 0; p < COLS; ++p)
#pragma unroll
                for (int q = 0; q < KINDS; ++q) {
                    int r, c;
                    of_piece(q * PG + p * NW + wave, lane, r, c);           // (PG > NW: wave < NW; else p = 0)
                    off[p][q] = (int32_t)((element(s, r, c) - q * 8 * s.row_stride) * (int64_t)sizeof(T));
                    on[p][q] = !PAD || valid(s, c);
                }
        }
    }
    __device__ __forceinline__ void load(char* tile, const Source& s, int32_t row0, int32_t last, int grain) const {
        if constexpr (DMA) {
            const int wave = threadIdx.x >> 6;
            if (row0 + ROWS - 1 <= last) {
                // a descriptor for the tile's rows: the thread's part of an address is one register, the rest is scalar (the
                // descriptor's type exists in the device pass only)
#if defined(__HIP_DEVICE_COMPILE__)
                const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(static_cast<const T*>(s.data) + (int64_t)row0 * s.row_stride), 0, 0x7FFFFFFF, 0x00027000);
                const int32_t step = (int32_t)s.row_stride * (int32_t)sizeof(T) * (PG > NW ? 8 : NW / PG * 8);
#pragma unroll
                for (int k = 0; k < ROWS * CH / NT; ++k) {
                    const int at0 = __builtin_amdgcn_readfirstlane((k * NW + wave) * 1024);
                    if (!PAD || on[k % COLS][KINDS == 2 ? k / COLS & 1 : 0]) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (SGL_LDS void*)(tile + at0), 16, off[k % COLS][KINDS == 2 ? k / COLS & 1 : 0], k / COLS * step, 0, 0);
                }
#endif
            } else {
                const int lane = threadIdx.x & 63;
#pragma unroll 1
                for (int k = 0; k < ROWS * CH / NT; ++k) {
                    const int piece = k * NW + wave;
                    int r, c;
                    of_piece(piece, lane, r, c);
                    const int32_t n = row0 + r < last ? row0 + r : last;
                    const T* src = static_cast<const T*>(s.data) + (int64_t)n * s.row_stride + element(s, 0, c);
                    const int at0 = __builtin_amdgcn_readfirstlane(piece * 1024);
                    if (!PAD || valid(s, c)) __builtin_amdgcn_global_load_lds((SGL_GLOBAL void*)src, (SGL_LDS void*)(tile + at0), 16, 0, 0);
                }
            }
        } else {
            typedef typename Mat<T>::Frag Frag;
            const T* __restrict__ base = static_cast<const T*>(s.data);
            for (int i = threadIdx.x; i < ROWS * CH; i += NT) {
                const int r = i / CH, c = i % CH;
                const int32_t n = row0 + r < last ? row0 + r : last;
                const int e = TWO ? (c % (CH / 2)) * EP : c * EP;
                const T* src = base + (int64_t)n * s.row_stride + (TWO ? (c / (CH / 2)) * s.half_stride : 0) + e;
                const Frag f = load_chunk<T>(src, s.len - e, grain);
                *reinterpret_cast<Frag*>(tile + at<RB>(r, c)) = f;
            }
        }
    }
};

// Staging for a pass in which something that is not finite has turned up: such elements become zero, and byte (row, chunk) of
// `marks` has their bits.  What a column does not see then no longer reaches it as 0 * NaN; what it sees is put back as NaN
// by the caller from the marks.
template <typename T, int DP, int ROWS, int NT>
__device__ __forceinline__ void stage_finite(char* tile, uint8_t* marks, const Source& s, bool two, int32_t row0, int32_t last) {
    constexpr int RB = 2 * DP * (int)sizeof(T), CH = RB / 16, EP = 16 / (int)sizeof(T);
    const T* __restrict__ base = static_cast<const T*>(s.data);
#pragma unroll 1
    for (int i = threadIdx.x; i < ROWS * CH; i += NT) {
        const int r = i / CH, c = i % CH;
        const int32_t n = row0 + r < last ? row0 + r : last;
        const int e = two ? (c % (CH / 2)) * EP : c * EP;
        const T* src = base + (int64_t)n * s.row_stride + (two ? (c / (CH / 2)) * s.half_stride : 0) + e;
        T* to = reinterpret_cast<T*>(tile + at<RB>(r, c));
        uint32_t bits = 0;
#pragma unroll 1
        for (int j = 0; j < EP; ++j) {
            const T x = e + j < s.len ? src[j] : (T)0.0f;
            const float y = (float)x;
            const bool bad = !(y - y == 0.f);
            to[j] = bad ? (T)0.0f : x;
            bits |= bad ? 1u << j : 0u;
        }
        marks[i] = (uint8_t)bits;
    }
}

// marks of the elements 32 t .. 32 t + 31 of staged row r, a bit each
template <typename T, int RB>
__device__ __forceinline__ uint32_t marked(const uint8_t* marks, int r, int t) {
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const uint32_t*>(marks + r * (RB / 16) + 4 * t);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(marks + r * (RB / 16) + 8 * t);
        auto pack = [](uint32_t x) { return (x & 0xF) | (x >> 4 & 0xF0) | (x >> 8 & 0xF00) | (x >> 12 & 0xF000); };
        return pack(w.x) | pack(w.y) << 16;
    }
}
// any of chunks [c0, c1)
template <int RB>
__device__ __forceinline__ bool marked_any(const uint8_t* marks, int r, int c0, int c1) {
    uint32_t x = 0;
#pragma unroll 1
    for (int c = c0; c < c1; ++c) x |= marks[r * (RB / 16) + c];
    return x != 0;
}
// the results of a column at the marked elements become NaN
template <typename T, int RB, int N>
__device__ __forceinline__ void spoil(f32x16 (&x)[N], const uint8_t* marks, int r, int half) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
        const uint32_t bits = marked<T, RB>(marks, r, t) >> (4 * half);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[t][e] = row_bit(bits, e) ? NAN : x[t][e];
    }
}

// this wave's DMA has landed and every wave's has once the block is past the barrier
__device__ __forceinline__ void staged() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// clears an image whose padding no load will write
template <int MODE, int BYTES, int NT>
__device__ __forceinline__ void clear_image(char* tile) {
    if constexpr (MODE == PADDED) {
        for (int i = threadIdx.x * 16; i < BYTES; i += NT * 16) *reinterpret_cast<uint4*>(tile + i) = uint4{0, 0, 0, 0};
    }
}

// EP elements from element e of a row, kept in registers; zero beyond len.  WHOLE: every chunk is whole and aligned.
template <typename T, bool WHOLE>
__device__ __forceinline__ typename Mat<T>::Frag global_frag(const T* src, int e, int len, int grain) {
    if constexpr (WHOLE) return *reinterpret_cast<const typename Mat<T>::Frag*>(src + e);
    else return load_chunk<T>(src + e, len - e, grain);
}

// of map m of (row i, head h)
__device__ __forceinline__ float* map_row(const sgl_diff_attn_args& a, int64_t i, int h, int m) { return a.maps + (pair_at(a, i, h) + m) * a.Dv; }
// sum += x . (the same elements of a row of `maps`, from element e)
template <typename T, bool WHOLE>
__device__ __forceinline__ float dot_map(const typename Mat<T>::Frag& x, const float* src, int e, int len, int grain, float sum) {
#pragma unroll
    for (int u = 0; u < Mat<T>::EP; u += 4) {
        const f32x4 y = global_frag<float, WHOLE>(src, e + u, len, grain);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum = __builtin_fmaf((float)x[u + j], y[j], sum);
    }
    return sum;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

// 32 rows of results, one a lane of either half (the layout of the products), to memory through the wave's own piece of LDS (32
// rows of PIECE bytes): a row's elements lie in registers of two lanes, eight bytes here and there; from LDS they go out as
// whole 16-byte chunks side by side.  val(t, r): register r of the 32 elements from 32 t; row k goes to base + k * stride
// where bit k of `keep` is set.  The order is fixed, a few values at a time: a spilled register here would be read back behind the stores (loads
// and stores return through one counter), which cost 28000 cycles a block.
template <typename T, int PIECE, int N, bool WHOLE, typename Val>
__device__ __forceinline__ void store_rows(Val val, char* box, int lane, int len, int grain, T* base, int64_t stride, uint32_t keep) {
    constexpr int FIT = PIECE / (32 * (int)sizeof(T)), AT = FIT >= N ? N : FIT >= 2 ? 2 : 1;           // 32-wide pieces at a time
    static_assert(FIT >= 1, "one piece fits");
    constexpr int BYTES = AT * 32 * (int)sizeof(T), CH = BYTES / 16, EP = 16 / (int)sizeof(T);
    struct alignas(4 * sizeof(T)) Four {
        T e[4];
    };
    const int half = lane >> 5, col = lane & 31, c = lane % CH;
#pragma unroll
    for (int t0 = 0; t0 < N; t0 += AT) {
#pragma unroll
        for (int u = 0; u < AT; ++u) {
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                Four y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y.e[e] = (T)val(t0 + u, 4 * r4 + e);
                const int b = (u * 32 + 8 * r4 + 4 * half) * (int)sizeof(T);
                *reinterpret_cast<Four*>(box + col * BYTES + ((((b >> 4) ^ col) & (CH - 1)) << 4) + (b & 15)) = y;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        T* to = base + (lane / CH) * stride + t0 * 32 + c * EP;
        const int left = len - t0 * 32 - c * EP;
#pragma unroll
        for (int i = 0; i < 32 * CH / 64; ++i) {
            const int r = i * (64 / CH) + lane / CH;
            const typename Mat<T>::Frag f = *reinterpret_cast<const typename Mat<T>::Frag*>(box + r * BYTES + (((c ^ r) & (CH - 1)) << 4));
            if ((keep >> r) & 1) {
                if constexpr (WHOLE) *reinterpret_cast<typename Mat<T>::Frag*>(to) = f;
                else store_chunk<T>(to, f, left, grain);
            }
            to += (64 / CH) * stride;
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// Work item of a block: consecutive items of one XCD (blocks go to the 8 of them in turn) are neighbours, so that what they
// share lies in one L2.  The grid is a multiple of 8; items >= n do nothing.
__device__ __forceinline__ uint32_t xcd_item(const AttnArgs& g, uint32_t n) {
    const uint32_t first = (uint32_t)g.first, here = min(n - first, (uint32_t)GRID_PART);
    return first + (blockIdx.x % 8) * ((here + 7) / 8) + blockIdx.x / 8;
}

// The spans of 32 columns (lanes l and l + 32 hold the same one): their union, and what all of them see.  Spans of ascending rows
// ascend, so the first and the last that are not empty say it.
struct Reach {
    int32_t lo, hi;             // the union
    int32_t from, to;           // seen by all
};
__device__ __forceinline__ Reach reach_of(Span span) {
    const uint32_t live = (uint32_t)__ballot(span.lo < span.hi);
    if (live == 0) return Reach{0x7FFFFFFF, 0, 0, 0};
    const int first = __builtin_ctz(live), last = 31 - __builtin_clz(live);
    return Reach{__builtin_amdgcn_readlane(span.lo, first), __builtin_amdgcn_readlane(span.hi, last), __builtin_amdgcn_readlane(span.lo, last),
                 __builtin_amdgcn_readlane(span.hi, first)};
}

// bit k: element base + k lies in [lo, hi)
__device__ __forceinline__ uint32_t span_bits(int32_t base, Span span) {
    const int32_t from = min(max(span.lo - base, 0), 32), to = min(max(span.hi - base, 0), 32);
    return (uint32_t)((1ull << to) - 1) & ~(uint32_t)((1ull << from) - 1);
}
// the key mask of the keys [j0, j0 + 32), the same in all lanes; keys beyond `last` repeat it
__device__ __forceinline__ uint32_t mask_bits(const uint8_t* __restrict__ mask, int32_t j0, int lane, int32_t last) {
    if (mask == nullptr) return ~0u;
    return (uint32_t)__ballot(mask[min(j0 + (lane & 31), last)] != 0);
}
// whether a column sees key j
__device__ __forceinline__ bool sees(int32_t j, Span span, const uint8_t* __restrict__ mask) {
    return j >= span.lo && j < span.hi && (mask == nullptr || mask[j]);
}

#endif  // __HIPCC__

// Host side.  A launch of any number of blocks, in parts (one, but for calls of millions of row tiles or rows).
template <typename Launch>
void in_parts(AttnArgs g, int64_t blocks, Launch launch) {
    for (g.first = 0; g.first < blocks; g.first += GRID_PART) launch(g, dim3((unsigned)(blocks - g.first < GRID_PART ? blocks - g.first : GRID_PART)));
}

// Forward on the matrix units: tiles of query rows, or (without q_ptr) of the heads of a group.
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
// rows whose offsets inside a tile of 64 fit 31 bits: up to 2^21 elements from row to row, 2^24 from half to half
inline bool dma_rows(const sgl_rows& r) { return r.row_stride >= 0 && r.row_stride <= (1 << 21) && r.head_stride >= 0 && r.head_stride <= (1 << 24); }
// How the matrix kernels of head width DP bring their rows in.  Training step of 8 sequences of 1024, 8 heads of 100 in fp32, causal:
// padded rows 3170 us, the same through registers 4230.
inline int stage_mode(const AttnArgs& g, int DP, std::initializer_list<const sgl_rows*> staged) {
    bool direct = g.grain == 16;
    for (const sgl_rows* r : staged) direct = direct && dma_rows(*r);
    return !direct ? BY_REGISTERS : g.a.D == DP && g.a.Dv == 2 * DP ? WHOLE_ROWS : PADDED;
}
template <typename T>
void forward_type(const AttnArgs& g, hipStream_t st);
template <typename T>
void backward_type(const AttnArgs& g, hipStream_t st);

}  // namespace attn
}  // namespace sgl
