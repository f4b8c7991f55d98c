// Differential attention over ragged sequences for gfx950: out = softmax(S_1) v - lam softmax(S_2) v.
//
// Forward, one pass over a query's keys: the running maximum m and sum l of both maps, o_m <- o_m exp(m - m') + p v.
// Backward: P_m = exp(S_m - lse_m), dP = d_out v^T (one product for both maps), t_m = sum_j P_m dP,
//   dS_1 = P_1 (dP - t_1), dS_2 = -lam P_2 (dP - t_2), d_lam = -sum t_2,
//   dV = (P_1 - lam P_2)^T d_out, dK_m = scale dS_m^T q_m, dQ_m = scale dS_m k_m.
#include <math.h>

#include "common.hpp"

namespace sgl {
namespace {

constexpr int BLOCK = 256;
constexpr float NEG_INF = -INFINITY;

struct AttnArgs {
    sgl_diff_attn_args a;
    float scale;
};

// the sequence of element i: the last b with ptr[b] <= i < ptr[b + 1], -1 if there is none
__device__ __forceinline__ int64_t find_seq(const int64_t* __restrict__ ptr, int64_t B, int64_t i) {
    if (B <= 0 || i < ptr[0] || i >= ptr[B]) return -1;
    int64_t lo = 0, hi = B;                       // ptr[lo] <= i < ptr[hi]
    while (hi - lo > 1) {
        const int64_t mid = lo + (hi - lo) / 2;
        if (ptr[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

struct Span {
    int64_t lo, hi;
};

__device__ __forceinline__ int64_t clamp_to(int64_t x, int64_t n) { return x < 0 ? 0 : (x > n ? n : x); }

// keys that query row i sees (before key_mask); seq: its sequence
__device__ __forceinline__ Span keys_of(const sgl_diff_attn_args& a, int64_t seq, int64_t i) {
    Span s{0, 0};
    if (seq < 0) return s;
    const int64_t k0 = clamp_to(a.k_ptr[seq], a.Tk), k1 = clamp_to(a.k_ptr[seq + 1], a.Tk);
    s.lo = k0;
    s.hi = k1;
    if (a.causal) {
        const int64_t q1 = a.q_ptr ? a.q_ptr[seq + 1] : i + 1;
        const int64_t last = k1 - (q1 - i);       // the key that stands where the query does
        if (last + 1 < s.hi) s.hi = last + 1;
        if (a.window > 0 && last + 1 - a.window > s.lo) s.lo = last + 1 - a.window;
    }
    if (s.hi < s.lo) s.hi = s.lo;
    return s;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

template <typename T>
__device__ __forceinline__ const T* row(const sgl_rows& r, int64_t n, int64_t h) {
    return static_cast<const T*>(r.data) + n * r.row_stride + h * r.head_stride;
}
template <typename T>
__device__ __forceinline__ T* row_out(const sgl_rows& r, int64_t n, int64_t h) {
    return static_cast<T*>(r.data) + n * r.row_stride + h * r.head_stride;
}

// one wave per (query row, query head)
template <typename T>
__global__ __launch_bounds__(BLOCK) void fwd_row_kernel(AttnArgs g) {
    const sgl_diff_attn_args& a = g.a;
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= a.Tq * a.Hq) return;
    const int64_t i = w / a.Hq;
    const int h = (int)(w % a.Hq), hk = h / (a.Hq / a.Hk);
    const int64_t B = live_count(a.B_dev, a.B);
    const int64_t seq = a.q_ptr ? find_seq(a.q_ptr, B, i) : (i < B ? i : -1);
    if (seq < 0 && !(a.flags & SGL_ATTN_ZERO_REST)) return;
    const Span s = keys_of(a, seq, i);
    float q[2][2], o[2][4] = {}, m[2] = {NEG_INF, NEG_INF}, l[2] = {0.f, 0.f};
    for (int t = 0; t < 2; ++t)
        for (int u = 0; u < 2; ++u) {
            const int d = lane + u * 64;
            q[t][u] = seq >= 0 && d < a.D ? (float)row<T>(a.q, i, 2 * h + t)[d] * g.scale : 0.f;
        }
    for (int64_t j = s.lo; j < s.hi; ++j) {
        if (a.key_mask && !a.key_mask[j]) continue;
        float p[2];
        for (int t = 0; t < 2; ++t) {
            const T* k = row<T>(a.k, j, 2 * hk + t);
            float x = 0.f;
            for (int u = 0; u < 2; ++u) {
                const int d = lane + u * 64;
                if (d < a.D) x = __builtin_fmaf(q[t][u], (float)k[d], x);
            }
            x = wave_sum(x);
            const float mn = fmaxf(m[t], x), ms = mn == NEG_INF ? 0.f : mn;
            const float c = __expf(m[t] - ms);
            p[t] = __expf(x - ms);
            l[t] = l[t] * c + p[t];
            for (int u = 0; u < 4; ++u) o[t][u] *= c;
            m[t] = mn;
        }
        const T* v = row<T>(a.v, j, hk);
        for (int u = 0; u < 4; ++u) {
            const int d = lane + u * 64;
            if (d < a.Dv)
                for (int t = 0; t < 2; ++t) o[t][u] = __builtin_fmaf(p[t], (float)v[d], o[t][u]);
        }
    }
    const float lam = a.lam[h];
    const float i0 = l[0] == 0.f ? 0.f : 1.f / l[0], i1 = l[1] == 0.f ? 0.f : 1.f / l[1];
    for (int u = 0; u < 4; ++u) {
        const int d = lane + u * 64;
        if (d >= a.Dv) continue;
        const float o1 = o[0][u] * i0, o2 = o[1][u] * i1;
        row_out<T>(a.out, i, h)[d] = (T)(o1 - lam * o2);
        if (a.o2.data) row_out<T>(a.o2, i, h)[d] = (T)o2;
    }
    if (a.lse && lane < 2) a.lse[(i * a.Hq + h) * 2 + lane] = l[lane] == 0.f ? INFINITY : m[lane] + __logf(l[lane]);
}

// P_1, P_2 and dP of one (query, key); scores as the forward kernel forms them
template <typename T>
__device__ __forceinline__ void pair_of(const AttnArgs& g, int64_t i, int h, int64_t j, int hk, int lane, float p[2], float& dp) {
    const sgl_diff_attn_args& a = g.a;
    for (int t = 0; t < 2; ++t) {
        const T* q = row<T>(a.q, i, 2 * h + t);
        const T* k = row<T>(a.k, j, 2 * hk + t);
        float x = 0.f;
        for (int d = lane; d < a.D; d += 64) x = __builtin_fmaf((float)q[d] * g.scale, (float)k[d], x);
        x = wave_sum(x);
        const float lse = a.lse[(i * a.Hq + h) * 2 + t];
        p[t] = lse == INFINITY ? 0.f : __expf(x - lse);
    }
    const T* go = row<T>(a.d_out, i, h);
    const T* v = row<T>(a.v, j, hk);
    dp = 0.f;
    for (int d = lane; d < a.Dv; d += 64) dp = __builtin_fmaf((float)go[d], (float)v[d], dp);
    dp = wave_sum(dp);
}

// t_1, t_2 (delta [Tq, Hq, 2]) in a first pass over the keys, dQ in a second; one wave per (query row, query head)
template <typename T>
__global__ __launch_bounds__(BLOCK) void bwd_q_kernel(AttnArgs g, float* __restrict__ delta) {
    const sgl_diff_attn_args& a = g.a;
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= a.Tq * a.Hq) return;
    const int64_t i = w / a.Hq;
    const int h = (int)(w % a.Hq), hk = h / (a.Hq / a.Hk);
    const int64_t B = live_count(a.B_dev, a.B);
    const int64_t seq = a.q_ptr ? find_seq(a.q_ptr, B, i) : (i < B ? i : -1);
    const Span s = keys_of(a, seq, i);
    float tt[2] = {0.f, 0.f};
    for (int64_t j = s.lo; j < s.hi; ++j) {
        if (a.key_mask && !a.key_mask[j]) continue;
        float p[2], dp;
        pair_of<T>(g, i, h, j, hk, lane, p, dp);
        for (int t = 0; t < 2; ++t) tt[t] = __builtin_fmaf(p[t], dp, tt[t]);
    }
    if (lane < 2) delta[w * 2 + lane] = tt[lane];
    if (seq < 0 && !(a.flags & SGL_ATTN_ZERO_REST)) return;
    const float lam = a.lam[h];
    float dq[2][2] = {};
    for (int64_t j = s.lo; j < s.hi; ++j) {
        if (a.key_mask && !a.key_mask[j]) continue;
        float p[2], dp;
        pair_of<T>(g, i, h, j, hk, lane, p, dp);
        for (int t = 0; t < 2; ++t) {
            const float ds = p[t] * (dp - tt[t]) * (t ? -lam : 1.f);
            const T* k = row<T>(a.k, j, 2 * hk + t);
            for (int u = 0; u < 2; ++u)
                if (lane + u * 64 < a.D) dq[t][u] = __builtin_fmaf(ds, (float)k[lane + u * 64], dq[t][u]);
        }
    }
    for (int t = 0; t < 2; ++t)
        for (int u = 0; u < 2; ++u)
            if (lane + u * 64 < a.D) row_out<T>(a.d_q, i, 2 * h + t)[lane + u * 64] = (T)(dq[t][u] * g.scale);
}

// dK, dV; one wave per (key, key head), its sequence's queries in order
template <typename T>
__global__ __launch_bounds__(BLOCK) void bwd_kv_kernel(AttnArgs g, const float* __restrict__ delta) {
    const sgl_diff_attn_args& a = g.a;
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= a.Tk * a.Hk) return;
    const int64_t j = w / a.Hk;
    const int hk = (int)(w % a.Hk), G = a.Hq / a.Hk;
    const int64_t B = live_count(a.B_dev, a.B);
    const int64_t seq = find_seq(a.k_ptr, B, j);
    if (seq < 0 && !(a.flags & SGL_ATTN_ZERO_REST)) return;
    float dk[2][2] = {}, dv[4] = {};
    if (seq >= 0 && (!a.key_mask || a.key_mask[j])) {
        const int64_t q0 = a.q_ptr ? clamp_to(a.q_ptr[seq], a.Tq) : seq, q1 = a.q_ptr ? clamp_to(a.q_ptr[seq + 1], a.Tq) : seq + 1;
        for (int64_t i = q0; i < q1; ++i) {
            const Span s = keys_of(a, seq, i);
            if (j < s.lo || j >= s.hi) continue;
            for (int h = hk * G; h < (hk + 1) * G; ++h) {
                float p[2], dp;
                pair_of<T>(g, i, h, j, hk, lane, p, dp);
                const float lam = a.lam[h];
                const T* go = row<T>(a.d_out, i, h);
                for (int u = 0; u < 4; ++u)
                    if (lane + u * 64 < a.Dv) dv[u] = __builtin_fmaf(p[0] - lam * p[1], (float)go[lane + u * 64], dv[u]);
                for (int t = 0; t < 2; ++t) {
                    const float ds = p[t] * (dp - delta[(i * a.Hq + h) * 2 + t]) * (t ? -lam : 1.f);
                    const T* q = row<T>(a.q, i, 2 * h + t);
                    for (int u = 0; u < 2; ++u)
                        if (lane + u * 64 < a.D) dk[t][u] = __builtin_fmaf(ds, (float)q[lane + u * 64], dk[t][u]);
                }
            }
        }
    }
    for (int t = 0; t < 2; ++t)
        for (int u = 0; u < 2; ++u)
            if (lane + u * 64 < a.D) row_out<T>(a.d_k, j, 2 * hk + t)[lane + u * 64] = (T)(dk[t][u] * g.scale);
    for (int u = 0; u < 4; ++u)
        if (lane + u * 64 < a.Dv) row_out<T>(a.d_v, j, hk)[lane + u * 64] = (T)dv[u];
}

// d_lam[h] = -sum over rows of t_2, in a fixed order
__global__ __launch_bounds__(BLOCK) void lam_kernel(const float* __restrict__ delta, int64_t Tq, int32_t Hq, float* __restrict__ out) {
    __shared__ float s_sum[BLOCK];
    const int h = blockIdx.x;
    float acc = 0.f;
    for (int64_t i = threadIdx.x; i < Tq; i += BLOCK) acc += delta[(i * Hq + h) * 2 + 1];
    s_sum[threadIdx.x] = acc;
    __syncthreads();
    for (int n = BLOCK / 2; n > 0; n /= 2) {
        if ((int)threadIdx.x < n) s_sum[threadIdx.x] += s_sum[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[h] = -s_sum[0];
}

constexpr int64_t GRID_MAX = 0x7FFFFFFF;

int32_t check_args(const char* what, const sgl_diff_attn_args* a, bool backward) {
    if (!a) return fail(SGL_EINVAL, "%s: args is NULL", what);
    if (a->dtype != SGL_DT_F32 && a->dtype != SGL_DT_BF16 && a->dtype != SGL_DT_F16) return fail(SGL_EINVAL, "%s: bad dtype", what);
    if (a->D < 1 || a->D > 128 || a->Dv < 1 || a->Dv > 256) return fail(SGL_ENOTSUP, "%s: D must lie in [1, 128] and Dv in [1, 256]", what);
    if (a->Hk < 1 || a->Hq < 1 || a->Hq % a->Hk || a->Hq > 65535) return fail(SGL_EINVAL, "%s: Hq must be a multiple of Hk (both in [1, 65535])", what);
    if (a->B < 0 || a->Tq < 0 || a->Tk < 0 || a->window < 0) return fail(SGL_EINVAL, "%s: negative size", what);
    if (a->Tq > 0x7FFFFFFF || a->Tk > 0x7FFFFFFF || a->B > 0x7FFFFFFF) return fail(SGL_ENOTSUP, "%s: Tq, Tk and B must lie below 2^31", what);
    if (a->window > 0 && !a->causal) return fail(SGL_EINVAL, "%s: a window needs causal", what);
    if (!a->q_ptr && a->Tq != a->B) return fail(SGL_EINVAL, "%s: without q_ptr there is one query per sequence (Tq = B)", what);
    if (!a->k_ptr || !a->lam) return fail(SGL_EINVAL, "%s: k_ptr/lam is NULL", what);
    if (!(a->scale > -INFINITY && a->scale < INFINITY)) return fail(SGL_EINVAL, "%s: scale is not finite", what);
    if (a->Tq > 0 && (!a->q.data || !a->out.data)) return fail(SGL_EINVAL, "%s: q/out is NULL", what);
    if (a->Tk > 0 && (!a->k.data || !a->v.data)) return fail(SGL_EINVAL, "%s: k/v is NULL", what);
    if ((a->lse == nullptr) != (a->o2.data == nullptr)) return fail(SGL_EINVAL, "%s: lse and o2 come together", what);
    if (backward) {
        if (!a->d_lam || (a->Tq > 0 && (!a->lse || !a->d_out.data || !a->d_q.data)) || (a->Tk > 0 && (!a->d_k.data || !a->d_v.data)))
            return fail(SGL_EINVAL, "%s: lse, o2 or a gradient is NULL", what);
    }
    if (ceil_div<int64_t>(a->Tq * a->Hq, 4) > GRID_MAX || ceil_div<int64_t>(a->Tk * a->Hk, 4) > GRID_MAX)
        return fail(SGL_ENOTSUP, "%s: too many rows times heads", what);
    return SGL_OK;
}

template <typename T>
void forward(const AttnArgs& g, hipStream_t st) {
    hipLaunchKernelGGL(fwd_row_kernel<T>, dim3((unsigned)ceil_div<int64_t>(g.a.Tq * g.a.Hq, 4)), dim3(BLOCK), 0, st, g);
}

template <typename T>
void backward(const AttnArgs& g, float* delta, hipStream_t st) {
    if (g.a.Tq > 0) hipLaunchKernelGGL(bwd_q_kernel<T>, dim3((unsigned)ceil_div<int64_t>(g.a.Tq * g.a.Hq, 4)), dim3(BLOCK), 0, st, g, delta);
    if (g.a.Tk > 0) hipLaunchKernelGGL(bwd_kv_kernel<T>, dim3((unsigned)ceil_div<int64_t>(g.a.Tk * g.a.Hk, 4)), dim3(BLOCK), 0, st, g, delta);
    hipLaunchKernelGGL(lam_kernel, dim3((unsigned)g.a.Hq), dim3(BLOCK), 0, st, delta, g.a.Tq, g.a.Hq, g.a.d_lam);
}

}  // namespace
}  // namespace sgl

using namespace sgl;

extern "C" size_t sgl_diff_attn_workspace_bytes(const sgl_diff_attn_args* a) { return 0; }

extern "C" int32_t sgl_diff_attn(const sgl_diff_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t rc = check_args("diff_attn", a, false)) return rc;
    if (a->Tq == 0) return SGL_OK;
    const AttnArgs g{*a, (float)a->scale};
    if (a->dtype == SGL_DT_F32) forward<float>(g, as_stream(stream));
    else if (a->dtype == SGL_DT_BF16) forward<__bf16>(g, as_stream(stream));
    else forward<_Float16>(g, as_stream(stream));
    SGL_LAUNCH_CHECK();
    return SGL_OK;
}

extern "C" size_t sgl_diff_attn_backward_workspace_bytes(const sgl_diff_attn_args* a) {
    return check_args("diff_attn_backward", a, false) ? 0 : align_up((size_t)a->Tq * (size_t)a->Hq * 2 * sizeof(float));
}

extern "C" int32_t sgl_diff_attn_backward(const sgl_diff_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t rc = check_args("diff_attn_backward", a, true)) return rc;
    const size_t need = sgl_diff_attn_backward_workspace_bytes(a);
    if (need > 0 && (!workspace || workspace_bytes < need)) return fail(SGL_ENOMEM, "diff_attn_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const AttnArgs g{*a, (float)a->scale};
    float* delta = static_cast<float*>(workspace);
    if (a->dtype == SGL_DT_F32) backward<float>(g, delta, as_stream(stream));
    else if (a->dtype == SGL_DT_BF16) backward<__bf16>(g, delta, as_stream(stream));
    else backward<_Float16>(g, delta, as_stream(stream));
    SGL_LAUNCH_CHECK();
    return SGL_OK;
}
