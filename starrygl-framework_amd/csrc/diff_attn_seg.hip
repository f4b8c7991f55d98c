// Differential attention of one query per sequence over few keys (a root over its sampled neighbours) without matrix units,
// forward and backward.
//
// A wave takes one (sequence, head).  L lanes share a key row, 16 bytes each: the first L / 2 hold the first half of the
// head's key, the others the second, all of them the value; 64 / L keys are looked at side by side.  Nothing is read twice
// and nothing waits for another wave: a backward wave has a key's scores, probabilities and d_out v product at hand, and
// writes dK and dV as it goes.  Bound by the rows it moves: 2 D + Dv products a key and head stand against as many elements
// read (and written, backward).  12000 roots with up to 10 neighbours, 2 heads over 2, 32 wide, fp32: forward 26 us, backward 38
// us and 4 to sum d_lam (29, 45 and 4 without fetching the next keys before the present ones are worked on): the calls are short,
// and a wave waits for its one or two rounds of loads.
#include "diff_attn.hpp"

namespace sgl {
namespace attn {
namespace {

constexpr int WAVES = BLOCK / 64;

template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int m = 1; m < L; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

// EP values of a row as floats; zeros beyond len
template <typename T>
__device__ __forceinline__ void load_part(float (&f)[Mat<T>::EP], const T* src, int e, int len, bool live, int grain) {
    typename Mat<T>::Frag x = {};
    if (live) x = global_frag<T, false>(src, e, len, grain);
#pragma unroll
    for (int j = 0; j < Mat<T>::EP; ++j) f[j] = (float)x[j];
}
template <typename T>
__device__ __forceinline__ void store_part(T* dst, const float (&f)[Mat<T>::EP], float scale, int e, int len, int grain) {
    typename Mat<T>::Frag x;
#pragma unroll
    for (int j = 0; j < Mat<T>::EP; ++j) x[j] = (T)(f[j] * scale);
    store_chunk<T>(dst + e, x, len - e, grain);
}

// what a lane holds of a key and its value, still as it came: the next keys' are fetched before the present ones are worked on
template <typename T>
struct KeyPart {
    typename Mat<T>::Frag k, v;
    bool in, see;               // a key of the sequence; one that the query sees
};
template <typename T>
__device__ __forceinline__ void widen(float (&f)[Mat<T>::EP], const typename Mat<T>::Frag& x) {
#pragma unroll
    for (int j = 0; j < Mat<T>::EP; ++j) f[j] = (float)x[j];
}

struct Lanes {
    int slot, half, e, ev;      // key of a pass, half of the head, first element of the half, first of the value
    template <int L, int EP>
    static __device__ __forceinline__ Lanes make(int lane) {
        Lanes s;
        const int l = lane & (L - 1);
        s.slot = lane / L;
        s.half = l / (L / 2);
        s.e = (l & (L / 2 - 1)) * EP;
        s.ev = l * EP;
        return s;
    }
};

template <typename T>
__device__ __forceinline__ KeyPart<T> fetch(const sgl_diff_attn_args& a, Span span, int32_t j, int hk, const Lanes& ln, int grain) {
    KeyPart<T> x = {};
    x.in = j < span.hi;
    x.see = x.in && (a.key_mask == nullptr || a.key_mask[j]);
    if (x.see) {
        x.k = global_frag<T, false>(row<T>(a.k, j, 2 * hk + ln.half), ln.e, a.D, grain);
        x.v = global_frag<T, false>(row<T>(a.v, j, hk), ln.ev, a.Dv, grain);
    }
    return x;
}

template <typename T, int L>
__global__ __launch_bounds__(BLOCK) void seg_fwd_kernel(AttnArgs g) {
    constexpr int EP = Mat<T>::EP, SLOTS = 64 / L;
    const sgl_diff_attn_args& a = g.a;
    const int lane = threadIdx.x & 63;
    const int64_t w = (g.first + blockIdx.x) * WAVES + (threadIdx.x >> 6);
    if (w >= a.B * a.Hq) return;
    const int64_t i = w / a.Hq;
    const int h = (int)(w - i * a.Hq), hk = h / (a.Hq / a.Hk);
    const int64_t B = live_count(a.B_dev, a.B);
    if (i >= B && !(a.flags & SGL_ATTN_ZERO_REST)) return;
    const Span span = keys_of(a, i < B ? (int32_t)i : -1, i);
    const Lanes ln = Lanes::make<L, EP>(lane);
    const float c2 = g.scale < 0.f ? -g.c2 : g.c2;
    float q[EP], o[2][EP], m[2] = {NEG_INF, NEG_INF}, l[2] = {0.f, 0.f};
    KeyPart<T> next = fetch<T>(a, span, span.lo + ln.slot, hk, ln, g.grain);
    load_part<T>(q, row<T>(a.q, i, 2 * h + ln.half), ln.e, a.D, true, g.grain);
#pragma unroll
    for (int j = 0; j < EP; ++j) o[0][j] = o[1][j] = 0.f;
    for (int32_t j0 = span.lo; j0 < span.hi; j0 += SLOTS) {
        const KeyPart<T> key = next;
        next = fetch<T>(a, span, j0 + SLOTS + ln.slot, hk, ln, g.grain);
        const bool see = key.see;
        float k[EP], v[EP];
        widen<T>(k, key.k);
        widen<T>(v, key.v);
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < EP; ++e) x = __builtin_fmaf(q[e], k[e], x);
        x = lanes_sum<L / 2>(x) * c2;
        x = see ? x : NEG_INF;
        const float y = __shfl_xor(x, L / 2);
        const float s[2] = {ln.half ? y : x, ln.half ? x : y};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float mn = fmaxf(m[t], s[t]), ms = mn == NEG_INF ? 0.f : mn;
            const float f = exp2_hw(m[t] - ms), p = exp2_hw(s[t] - ms);
            m[t] = mn;
            l[t] = __builtin_fmaf(l[t], f, p);
#pragma unroll
            for (int e = 0; e < EP; ++e) o[t][e] = __builtin_fmaf(o[t][e], f, p * v[e]);
        }
    }
    // the slots' results joined
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float top = m[t];
#pragma unroll
        for (int k = L; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
        const float f = m[t] == NEG_INF && l[t] == 0.f ? 0.f : exp2_hw(m[t] - top);
        l[t] *= f;
#pragma unroll
        for (int k = L; k < 64; k <<= 1) l[t] += __shfl_xor(l[t], k);
        const bool none = l[t] == 0.f;
        const float inv = none ? 0.f : 1.f / l[t];
#pragma unroll
        for (int e = 0; e < EP; ++e) {
            float x = o[t][e] * f;          // (NaN stays, whatever the slot's weight)
#pragma unroll
            for (int k = L; k < 64; k <<= 1) x += __shfl_xor(x, k);
            o[t][e] = none ? 0.f : x * inv;
        }
        if (a.lse && lane == t) a.lse[w * 2 + t] = none ? INFINITY : top + __builtin_amdgcn_logf(l[t]);
    }
    if (ln.slot != 0) return;
    const float lam = a.lam[h];
    if (a.maps) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < EP; u += 4)
                store_chunk<float>(map_row(a, i, h, t) + ln.ev + u, f32x4{o[t][u], o[t][u + 1], o[t][u + 2], o[t][u + 3]}, a.Dv - ln.ev - u, g.map_grain);
    }
    if (a.o2.data) store_part<T>(row_out<T>(a.o2, i, h), o[1], 1.f, ln.ev, a.Dv, g.grain);
#pragma unroll
    for (int e = 0; e < EP; ++e) o[0][e] = __builtin_fmaf(-lam, o[1][e], o[0][e]);
    store_part<T>(row_out<T>(a.out, i, h), o[0], 1.f, ln.ev, a.Dv, g.grain);
}

// DQ: a wave's unit is (sequence, query head), it sums dQ and d_lam's share.  DKV: (sequence, key head), it writes dK and dV,
// summed over the heads of the group; it reads the row sums t_m that the former leaves.  Groups of one head do both at once.
template <typename T, int L, bool DQ, bool DKV>
__global__ __launch_bounds__(BLOCK) void seg_bwd_kernel(AttnArgs g) {
    constexpr int EP = Mat<T>::EP, SLOTS = 64 / L;
    __shared__ float s_lam[WAVES];
    const sgl_diff_attn_args& a = g.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, G = a.Hq / a.Hk;
    const int head = blockIdx.y;                    // DQ: query head (with one head a group also the key head)
    const int hk = DQ ? head / G : head;
    const int64_t B = live_count(a.B_dev, a.B);
    const int64_t first = (int64_t)blockIdx.x * WAVES + wave, stride = (int64_t)gridDim.x * WAVES;
    const bool zero = a.flags & SGL_ATTN_ZERO_REST;
    const Lanes ln = Lanes::make<L, EP>(lane);
    const float c2 = g.scale < 0.f ? -g.c2 : g.c2;
    float share = 0.f;
    for (int64_t i = first; i < a.B; i += stride) {
        if (i >= B && !(zero && DQ)) break;
        const Span span = keys_of(a, i < B ? (int32_t)i : -1, i);
        float q[EP], go[EP], t[2], lse[2], dq[EP], lam = 0.f;
        auto of_head = [&](int h) {
            lam = a.lam[h];
            load_part<T>(q, row<T>(a.q, i, 2 * h + ln.half), ln.e, a.D, true, g.grain);
            const typename Mat<T>::Frag x = global_frag<T, false>(row<T>(a.d_out, i, h), ln.ev, a.Dv, g.grain);
            widen<T>(go, x);
            lse[0] = a.lse[pair_at(a, i, h)];
            lse[1] = a.lse[pair_at(a, i, h) + 1];
            if (!DQ) {
                t[0] = g.delta[pair_at(a, i, h)];
                t[1] = g.delta[pair_at(a, i, h) + 1];
                return;
            }
            t[0] = t[1] = 0.f;
            if (a.maps) {
#pragma unroll
                for (int m = 0; m < 2; ++m) t[m] = dot_map<T, false>(x, map_row(a, i, h, m), ln.ev, a.Dv, g.map_grain, 0.f);
            } else {
                float y[EP], y2[EP];
                load_part<T>(y, row<T>(a.out, i, h), ln.ev, a.Dv, true, g.grain);
                load_part<T>(y2, row<T>(a.o2, i, h), ln.ev, a.Dv, true, g.grain);
#pragma unroll
                for (int e = 0; e < EP; ++e) {
                    t[1] = __builtin_fmaf(go[e], y2[e], t[1]);
                    t[0] = __builtin_fmaf(go[e], __builtin_fmaf(lam, y2[e], y[e]), t[0]);
                }
            }
            t[0] = lanes_sum<L>(t[0]);
            t[1] = lanes_sum<L>(t[1]);
            if (!DKV && lane == 0) g.delta[pair_at(a, i, h)] = t[0], g.delta[pair_at(a, i, h) + 1] = t[1];
        };
#pragma unroll
        for (int e = 0; e < EP; ++e) dq[e] = 0.f;
        KeyPart<T> next = fetch<T>(a, span, span.lo + ln.slot, hk, ln, g.grain);
        if (DQ || G == 1) of_head(head);
        for (int32_t j0 = span.lo; j0 < span.hi; j0 += SLOTS) {
            const int32_t j = j0 + ln.slot;
            const KeyPart<T> key = next;
            next = fetch<T>(a, span, j0 + SLOTS + ln.slot, hk, ln, g.grain);
            const bool in = key.in, see = key.see;
            float k[EP], v[EP], dk[EP], dv[EP];
            widen<T>(k, key.k);
            widen<T>(v, key.v);
#pragma unroll
            for (int e = 0; e < EP; ++e) dk[e] = dv[e] = 0.f;
            for (int hg = 0; hg < (DQ ? 1 : G); ++hg) {
                if (!DQ && G > 1) of_head(hk * G + hg);
                float x = 0.f, dp = 0.f;
#pragma unroll
                for (int e = 0; e < EP; ++e) {
                    x = __builtin_fmaf(q[e], k[e], x);
                    dp = __builtin_fmaf(go[e], v[e], dp);
                }
                x = lanes_sum<L / 2>(x);
                dp = lanes_sum<L>(dp);
                float p = see ? exp2_hw(__builtin_fmaf(x, c2, -(ln.half ? lse[1] : lse[0]))) : 0.f;
                const float other = __shfl_xor(p, L / 2), p2 = ln.half ? p : other;
                if (!see) dp = 0.f;
                if (DQ) share += ln.e == 0 && ln.half == 0 && see ? p2 * dp : 0.f;
                const float ds = see ? p * (dp - (ln.half ? t[1] : t[0])) * (ln.half ? -lam : 1.f) : 0.f;
                if (DKV) {
                    const float wgt = __builtin_fmaf(-lam, p2, ln.half ? other : p);
#pragma unroll
                    for (int e = 0; e < EP; ++e) {
                        dk[e] = see ? __builtin_fmaf(ds, q[e], dk[e]) : 0.f;
                        dv[e] = see ? __builtin_fmaf(wgt, go[e], dv[e]) : 0.f;
                    }
                }
                if (DQ) {
#pragma unroll
                    for (int e = 0; e < EP; ++e) dq[e] = __builtin_fmaf(ds, k[e], dq[e]);
                }
            }
            if (DKV && in) {
                store_part<T>(row_out<T>(a.d_k, j, 2 * hk + ln.half), dk, g.scale, ln.e, a.D, g.grain);
                store_part<T>(row_out<T>(a.d_v, j, hk), dv, 1.f, ln.ev, a.Dv, g.grain);
            }
        }
        if (DKV && a.window > 0) {
            // keys of the sequence in front of the window
            const float none[EP] = {};
            for (int32_t j = clamp_to(a.k_ptr[i], a.Tk) + ln.slot; j < span.lo; j += SLOTS) {
                store_part<T>(row_out<T>(a.d_k, j, 2 * hk + ln.half), none, 1.f, ln.e, a.D, g.grain);
                store_part<T>(row_out<T>(a.d_v, j, hk), none, 1.f, ln.ev, a.Dv, g.grain);
            }
        }
        if (DQ) {
#pragma unroll
            for (int e = 0; e < EP; ++e) {
#pragma unroll
                for (int k = L; k < 64; k <<= 1) dq[e] += __shfl_xor(dq[e], k);
            }
            if (ln.slot == 0) store_part<T>(row_out<T>(a.d_q, i, 2 * head + ln.half), dq, span.lo < span.hi ? g.scale : 0.f, ln.e, a.D, g.grain);
        }
    }
    if (DKV && zero) {
        // keys of no sequence
        const int64_t k0 = B > 0 ? clamp_to(a.k_ptr[0], a.Tk) : a.Tk, k1 = B > 0 ? clamp_to(a.k_ptr[B], a.Tk) : a.Tk;
        const float none[EP] = {};
        for (int64_t r = first * SLOTS + ln.slot; r < k0 + (a.Tk - k1); r += stride * SLOTS) {
            const int64_t j = r < k0 ? r : r - k0 + k1;
            store_part<T>(row_out<T>(a.d_k, j, 2 * hk + ln.half), none, 1.f, ln.e, a.D, g.grain);
            store_part<T>(row_out<T>(a.d_v, j, hk), none, 1.f, ln.ev, a.Dv, g.grain);
        }
    }
    if (DQ) {
        share = lanes_sum<64>(share);
        if (lane == 0) s_lam[wave] = share;
        __syncthreads();
        if (threadIdx.x == 0) {
            float x = 0.f;
            for (int w = 0; w < WAVES; ++w) x += s_lam[w];
            g.lam_part[(int64_t)head * gridDim.x + blockIdx.x] = x;
        }
    }
}

// d_lam[h] = -sum of the blocks' shares, in a fixed order
__global__ __launch_bounds__(BLOCK) void lam_kernel(const float* __restrict__ part, int32_t n, float* __restrict__ out) {
    __shared__ float s_sum[BLOCK];
    float acc = 0.f;
    for (int32_t i = threadIdx.x; i < n; i += BLOCK) acc += part[(int64_t)blockIdx.x * n + i];
    s_sum[threadIdx.x] = acc;
    __syncthreads();
#pragma unroll
    for (int k = BLOCK / 2; k > 0; k /= 2) {
        if ((int)threadIdx.x < k) s_sum[threadIdx.x] += s_sum[threadIdx.x + k];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[blockIdx.x] = -s_sum[0];
}

template <typename T, int L>
void launch_fwd(const AttnArgs& g, hipStream_t st) {
    in_parts(g, ceil_div<int64_t>(g.a.B * g.a.Hq, WAVES),
             [&](const AttnArgs& part, dim3 grid) { hipLaunchKernelGGL((seg_fwd_kernel<T, L>), grid, dim3(BLOCK), 0, st, part); });
}

template <typename T, int L>
void launch_bwd(const AttnArgs& g, hipStream_t st) {
    const int64_t n = seg_blocks(g.a);
    const dim3 block(BLOCK);
    if (g.a.Hq == g.a.Hk) {
        hipLaunchKernelGGL((seg_bwd_kernel<T, L, true, true>), dim3((unsigned)n, (unsigned)g.a.Hq), block, 0, st, g);
    } else {
        hipLaunchKernelGGL((seg_bwd_kernel<T, L, true, false>), dim3((unsigned)n, (unsigned)g.a.Hq), block, 0, st, g);
        hipLaunchKernelGGL((seg_bwd_kernel<T, L, false, true>), dim3((unsigned)n, (unsigned)g.a.Hk), block, 0, st, g);
    }
    hipLaunchKernelGGL(lam_kernel, dim3((unsigned)g.a.Hq), block, 0, st, g.lam_part, (int32_t)n, g.a.d_lam);
}

// lanes of a key row: a power of two that holds both halves of a key and the value, 16 bytes a lane
int lanes_of(const sgl_diff_attn_args& a) {
    const int ep = a.dtype == SGL_DT_F32 ? 4 : 8;
    int half = 2;
    while (half * ep < a.D) half *= 2;
    int l = 2 * half;
    while (l * ep < a.Dv) l *= 2;
    return l;
}

template <typename T, bool BWD>
void launch_lanes(const AttnArgs& g, hipStream_t st) {
    auto go = [&](auto l) {
        constexpr int L = decltype(l)::value;
        if constexpr (BWD) launch_bwd<T, L>(g, st);
        else launch_fwd<T, L>(g, st);
    };
    switch (lanes_of(g.a)) {
        case 4: return go(Int<4>{});
        case 8: return go(Int<8>{});
        case 16: return go(Int<16>{});
        case 32: return go(Int<32>{});
        default: return go(Int<64>{});
    }
}

}  // namespace

// waves walk the sequences of a head in turn: at most 8 blocks a CU in all, so that the shares of d_lam stay few
int64_t seg_blocks(const sgl_diff_attn_args& a) {
    int64_t n = ceil_div<int64_t>(a.B, WAVES);
    const int64_t most = ceil_div<int64_t>(2048, a.Hq);
    return n > most ? most : n < 1 ? 1 : n;
}

void seg_forward(const AttnArgs& g, hipStream_t st) {
    if (g.a.dtype == SGL_DT_F32) launch_lanes<float, false>(g, st);
    else if (g.a.dtype == SGL_DT_BF16) launch_lanes<__bf16, false>(g, st);
    else launch_lanes<_Float16, false>(g, st);
}

void seg_backward(const AttnArgs& g, hipStream_t st) {
    if (g.a.dtype == SGL_DT_F32) launch_lanes<float, true>(g, st);
    else if (g.a.dtype == SGL_DT_BF16) launch_lanes<__bf16, true>(g, st);
    else launch_lanes<_Float16, true>(g, st);
}

}  // namespace attn
}  // namespace sgl
