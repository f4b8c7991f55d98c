// Differential attention over ragged sequences for gfx950: out = softmax(S_1) v - lam softmax(S_2) v.  Host side: argument
// checks, the choice of kernels, workspaces.
//
// Forward, one pass over a query's keys: the running maximum and sum of both maps, o_m <- o_m 2^(m - m') + p v.
// Backward: P_m = 2^(S_m - lse_m), dP = d_out v^T (one product for both maps), t_m = sum_j P_m dP = d_out o_m,
//   dS_1 = P_1 (dP - t_1), dS_2 = -lam P_2 (dP - t_2), d_lam = -sum t_2,
//   dV = (P_1 - lam P_2)^T d_out, dK_m = scale dS_m^T q_m, dQ_m = scale dS_m k_m.
// t_m is taken from o_m, for which a call that a backward one follows keeps both maps' results as they are, in fp32 (`maps`): the
// scores' gradients are differences P (dP - t) that mostly cancel where one key has all the weight, so a t that is off by a
// rounding to 16 bits shows in dQ and dK whole (off by 0.005 to 0.007 in bf16 over rows of 10 to 200 keys with scores of a few
// tens, 0.0024 from rounding dS alone; not zero where one key is seen).  It costs 6 bytes more an element written and 4 more
// read: 8 sequences of 2048, 16 heads over 4, 64 wide, causal, bf16, forward 268 -> 318 us (50 us; through LDS 351, past the caches
// 364), rows of the backward 297 -> 318.  In fp32 out and o_2 do (t_1 from out + lam o_2).  d_lam sums P_2 dP.
#include "diff_attn.hpp"

namespace sgl {
namespace attn {

FwdWork forward_work(const sgl_diff_attn_args& a) {
    FwdWork w{};
    const int G = a.Hq / a.Hk;
    int64_t units, keys;        // blocks without splitting, keys of one of them on average
    if (!a.q_ptr) {
        w.tiles = (int32_t)a.Tq;
        w.groups = ceil_div(G, 32);
        units = a.Tq * a.Hk * w.groups;
        keys = a.B > 0 ? a.Tk / a.B : 0;
    } else {
        const int rows = 128;                   // of a block
        w.tiles = (int32_t)ceil_div<int64_t>(a.Tq, rows);
        w.groups = 1;
        units = (int64_t)w.tiles * a.Hq;
        keys = a.Tk / (a.B > 0 && a.B < w.tiles ? a.B : (w.tiles > 0 ? w.tiles : 1));
    }
    // A call of fewer blocks than the chip holds side by side splits its key ranges, down to 256 keys a block.  16 histories of up to
    // 32768 keys, 16 heads over 4: 1024 blocks 117 us and 9 to join them, 2048 116 and 13, 4096 126 and 23.  Row tiles, whose
    // partial results are as large as 2 x 128 rows of fp32, are split only when they would leave half of the chip idle.
    int64_t splits = units > 0 ? (a.q_ptr ? 256 : 1024) / units : 1;
    if (splits > keys / 256) splits = keys / 256;
    w.splits = (int32_t)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
    w.items = units * w.splits;
    return w;
}

namespace {

constexpr int64_t PAIRS_MAX = 0x7FFFFFFF, COUNT_MAX = 0x7FFFFF00;

// SIZES: of a backward call whose gradients need not be there yet
enum Call { FORWARD, SIZES, BACKWARD };

int32_t check_args(const char* what, const sgl_diff_attn_args* a, Call call) {
    if (!a) return fail(SGL_EINVAL, "%s: args is NULL", what);
    if (a->dtype != SGL_DT_F32 && a->dtype != SGL_DT_BF16 && a->dtype != SGL_DT_F16) return fail(SGL_EINVAL, "%s: bad dtype", what);
    if (a->D < 1 || a->D > 128 || a->Dv < 1 || a->Dv > 256) return fail(SGL_ENOTSUP, "%s: D must lie in [1, 128] and Dv in [1, 256]", what);
    if (a->Hk < 1 || a->Hq < 1 || a->Hq % a->Hk || a->Hq > 65535) return fail(SGL_EINVAL, "%s: Hq must be a multiple of Hk (both in [1, 65535])", what);
    if (a->B < 0 || a->Tq < 0 || a->Tk < 0 || a->window < 0) return fail(SGL_EINVAL, "%s: negative size", what);
    // (rows are counted in 32 bits, and the last tile may reach past the last row)
    if (a->Tq > COUNT_MAX || a->Tk > COUNT_MAX || a->B > COUNT_MAX) return fail(SGL_ENOTSUP, "%s: Tq, Tk and B must not exceed 2^31 - 256", what);
    if (a->window > 0 && !a->causal) return fail(SGL_EINVAL, "%s: a window needs causal", what);
    if (!a->q_ptr && a->Tq != a->B) return fail(SGL_EINVAL, "%s: without q_ptr there is one query per sequence (Tq = B)", what);
    if (!a->k_ptr || !a->lam) return fail(SGL_EINVAL, "%s: k_ptr/lam is NULL", what);
    if (!(fabs(a->scale) * LOG2E <= 3.4e38)) return fail(SGL_EINVAL, "%s: scale is not finite in 32 bits", what);
    if (a->Tq > 0 && (!a->q.data || (!a->out.data && !(call != FORWARD && a->maps)))) return fail(SGL_EINVAL, "%s: q/out is NULL", what);
    if (a->Tk > 0 && (!a->k.data || !a->v.data)) return fail(SGL_EINVAL, "%s: k/v is NULL", what);
    if ((a->lse == nullptr) != (a->o2.data == nullptr && a->maps == nullptr)) return fail(SGL_EINVAL, "%s: lse comes with o2 or maps", what);
    if (reinterpret_cast<uintptr_t>(a->maps) % 16) return fail(SGL_EINVAL, "%s: maps is not aligned to 16 bytes", what);
    if (call == BACKWARD) {
        if (!a->d_lam || (a->Tq > 0 && (!a->lse || !a->d_out.data || !a->d_q.data)) || (a->Tk > 0 && (!a->d_k.data || !a->d_v.data)))
            return fail(SGL_EINVAL, "%s: lse, o2 and maps, or a gradient is NULL", what);
    }
    // (blocks are counted in 32 bits)
    if (a->Tq * a->Hq > PAIRS_MAX || a->Tk * a->Hk > PAIRS_MAX) return fail(SGL_ENOTSUP, "%s: Tq * Hq and Tk * Hk must stay below 2^31", what);
    return SGL_OK;
}

// Without q_ptr: sequences of few keys on average go without matrix units, a wave per query and head, which reads a key once for
// every query head of its group and walks it alone.  131072 keys in sequences of n, forward, matrix units against segments (us):
//   16 heads over 4, 64 wide, bf16   n = 32: 260, 148   48: 187, 130   64: 145, 122   96: 115, 120   128: 91, 119
//    8 heads over 8, 64 wide, bf16   n = 64: 196, 110   128: 142, 102   256: 124, 93   512: 107, 137
//    2 heads over 2, 32 wide, fp32   n = 64: 64, 25   128: 49, 28   256: 43, 48   512: 44, 84
//    2 heads over 1, 32 wide, fp32   n = 64: 37, 18    96: 39, 22   128: 29, 26   192: 33, 37   256: 25, 47
//   16 heads over 8, 64 wide, bf16   n = 64: 228, 192  96: 185, 192 128: 157, 198 192: 141, 214
// so groups of one or two heads stay there longer, if there is a wave for every SIMD (groups of two wide heads lose by it from about
// 96 keys on).  The rule knows the average length only: one long sequence among short ones is walked by a wave a head (12000 roots of
// 10 keys, 2 heads, 32 wide, fp32: 29 us; one of them with 1000 more 179, with 10000 more 1683).
bool by_segments(const sgl_diff_attn_args& a) {
    const int64_t keys = a.Hq / a.Hk <= 2 && a.B * a.Hq >= 1024 ? 192 : 64;
    return !a.q_ptr && a.Tk < keys * a.B;
}

// the widest pieces, of 16 bytes at most, that all rows divide into
int32_t grain_of(const sgl_diff_attn_args& a) {
    const int64_t item = a.dtype == SGL_DT_F32 ? 4 : 2;
    uint64_t bits = 16 | (uint64_t)(a.D * item) | (uint64_t)(a.Dv * item);
    auto rows = [&](const sgl_rows& r, int64_t heads) {
        if (r.data) bits |= reinterpret_cast<uintptr_t>(r.data) | (uint64_t)(r.row_stride * item) | (heads > 1 ? (uint64_t)(r.head_stride * item) : 0);
    };
    for (const sgl_rows* r : {&a.q, &a.k, &a.d_q, &a.d_k}) rows(*r, 2);
    for (const sgl_rows* r : {&a.out, &a.o2, &a.d_out}) rows(*r, a.Hq);
    for (const sgl_rows* r : {&a.v, &a.d_v}) rows(*r, a.Hk);
    return (int32_t)(bits & (~bits + 1));       // the lowest bit
}

int32_t forward_parts(const sgl_diff_attn_args& a) {
    if (a.Tq == 0 || by_segments(a)) return 1;
    const FwdWork w = forward_work(a);
    return a.q_ptr ? w.splits : 2 * w.splits;
}
size_t forward_need(const sgl_diff_attn_args& a, int32_t parts) {
    const size_t n = (size_t)parts * (size_t)a.Tq * (size_t)a.Hq * 2;
    return parts > 1 ? align_up(n * 2 * sizeof(float)) + align_up(n * (size_t)a.Dv * sizeof(float)) : 0;
}

int64_t backward_row_tiles(const sgl_diff_attn_args& a) { return ceil_div<int64_t>(a.Tq, QUERY_ROWS); }
size_t backward_need(const sgl_diff_attn_args& a) {
    const size_t sums = align_up((size_t)a.Tq * (size_t)a.Hq * 2 * sizeof(float));
    if (!a.q_ptr) return align_up((size_t)seg_blocks(a) * (size_t)a.Hq * sizeof(float)) + (a.Hq == a.Hk ? 0 : sums);
    return sums + align_up((size_t)backward_row_tiles(a) * (size_t)a.Hq * sizeof(float)) + 256;
}

}  // namespace
}  // namespace attn
}  // namespace sgl

using namespace sgl;
using namespace sgl::attn;

extern "C" size_t sgl_diff_attn_workspace_bytes(const sgl_diff_attn_args* a) {
    return check_args("diff_attn", a, FORWARD) ? 0 : forward_need(*a, forward_parts(*a));
}

extern "C" int32_t sgl_diff_attn(const sgl_diff_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t rc = check_args("diff_attn", a, FORWARD)) return rc;
    if (a->Tq == 0) return SGL_OK;
    AttnArgs g = attn_args(*a);
    g.grain = grain_of(*a);
    g.parts = forward_parts(*a);
    const size_t need = forward_need(*a, g.parts);
    if (need > 0) {
        if (!workspace || workspace_bytes < need) return fail(SGL_ENOMEM, "diff_attn: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        Arena ws(workspace, workspace_bytes);
        const size_t n = (size_t)g.parts * (size_t)a->Tq * (size_t)a->Hq * 2;
        g.part_ml = ws.take<float>(2 * n);
        g.part_o = ws.take<float>(n * (size_t)a->Dv);
    }
    if (by_segments(*a)) seg_forward(g, as_stream(stream));
    else if (a->dtype == SGL_DT_F32) forward_type<float>(g, as_stream(stream));
    else if (a->dtype == SGL_DT_BF16) forward_type<__bf16>(g, as_stream(stream));
    else forward_type<_Float16>(g, as_stream(stream));
    SGL_LAUNCH_CHECK();
    return SGL_OK;
}

extern "C" size_t sgl_diff_attn_backward_workspace_bytes(const sgl_diff_attn_args* a) {
    return check_args("diff_attn_backward", a, SIZES) ? 0 : backward_need(*a);
}

extern "C" int32_t sgl_diff_attn_backward(const sgl_diff_attn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (int32_t rc = check_args("diff_attn_backward", a, BACKWARD)) return rc;
    const size_t need = backward_need(*a);
    if (!workspace || workspace_bytes < need) return fail(SGL_ENOMEM, "diff_attn_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    AttnArgs g = attn_args(*a);
    g.grain = grain_of(*a);
    Arena ws(workspace, workspace_bytes);
    if (!a->q_ptr) {
        g.lam_part = ws.take<float>((size_t)seg_blocks(*a) * (size_t)a->Hq);
        if (a->Hq != a->Hk) g.delta = ws.take<float>((size_t)a->Tq * (size_t)a->Hq * 2);
        seg_backward(g, as_stream(stream));
    } else {
        g.delta = ws.take<float>((size_t)a->Tq * (size_t)a->Hq * 2);
        g.lam_part = ws.take<float>((size_t)backward_row_tiles(*a) * (size_t)a->Hq);
        if (a->dtype == SGL_DT_F32) backward_type<float>(g, as_stream(stream));
        else if (a->dtype == SGL_DT_BF16) backward_type<__bf16>(g, as_stream(stream));
        else backward_type<_Float16>(g, as_stream(stream));
    }
    SGL_LAUNCH_CHECK();
    return SGL_OK;
}
