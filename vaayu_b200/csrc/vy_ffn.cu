// vy_ffn.cu -- dense gated feed-forward block in bf16 / fp16, forward and backward.
//
//   forward   gate/up product with the activation in its epilogue -> h; down product
//   backward  dh = dy Wd with the gate's derivative in its epilogue -> dg, du, h; then dx and the
//             three weight gradients as one launch of four GEMMs
//
// Bounds.  Forward 6 T H I flops on 6 H I bytes of weights: HBM below about 250 tokens, the tensor
// cores above.  Backward 12 T H I flops.
#include "vy_stream.cuh"
#include "vy_tile.cuh"

namespace vy {
namespace {

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// The longest sum of one output tile, in values of K: 2^21 blocks of 64, each 0.24 us at the tensor cores'
// rate and 0.75 us where every block comes from HBM.  Beyond it a tile could take longer than the 2 s after
// which a wait for its sums gives up.
constexpr int64_t kMaxFfnK = int64_t(1) << 27;

// Elements of one part of a hidden row's matrix, and bytes of the matrix.
int64_t h_elems(const vy_ffn_call* c) { return c->n_tokens * int64_t(c->inter); }
int h_parts(const vy_ffn_call* c) { return c->n_tokens <= kPartTokens ? 2 : 1; }
size_t h_bytes(const vy_ffn_call* c) { return align256(size_t(h_elems(c)) * 2 * h_parts(c)); }

int check_ffn(const vy_ffn_call* c, bool backward) {
    if (!c) return fail(VY_ERR_INVALID, "null call");
    if (c->act_dtype != VY_BF16 && c->act_dtype != VY_F16)
        return fail(VY_ERR_UNSUPPORTED, "activation dtype code %d (bf16 or fp16)", c->act_dtype);
    if (c->activation != VY_ACT_SILU && c->activation != VY_ACT_GELU_TANH)
        return fail(VY_ERR_UNSUPPORTED, "activation code %d", c->activation);
    if (c->n_tokens < 0 || c->hidden <= 0 || c->inter <= 0)
        return fail(VY_ERR_INVALID, "n_tokens %lld, hidden %d, inter %d", (long long)c->n_tokens, c->hidden, c->inter);
    if (c->n_tokens > (int64_t(1) << 30)) return fail(VY_ERR_UNSUPPORTED, "n_tokens %lld", (long long)c->n_tokens);
    if (c->hidden % 8 || c->inter % 8)
        return fail(VY_ERR_UNSUPPORTED, "hidden %d and inter %d must be multiples of 8", c->hidden, c->inter);
    const bool by_token = backward && (c->d_w_gate || c->d_w_up || c->d_w_down);      // sums over the tokens
    if (c->hidden > kMaxFfnK || 2 * int64_t(c->inter) > kMaxFfnK || (by_token && c->n_tokens > kMaxFfnK))
        return fail(VY_ERR_UNSUPPORTED, "n_tokens %lld, hidden %d, inter %d: a sum of more than 2^27 products",
                    (long long)c->n_tokens, c->hidden, c->inter);
    const bool empty = c->n_tokens == 0;
    const void* need[] = {empty ? c->w_gate : c->x, c->w_gate, c->w_up, c->w_down};
    for (const void* q : need) {
        if (!q) return fail(VY_ERR_INVALID, "null operand");
        if (!aligned16(q)) return fail(VY_ERR_ALIGNMENT, "operands must be 16-byte aligned");
    }
    if (!aligned16(c->saved)) return fail(VY_ERR_ALIGNMENT, "saved must be 16-byte aligned");      // moved as float4
    if (c->x_row_stride < c->hidden || c->x_row_stride % 8)
        return fail(VY_ERR_ALIGNMENT, "x row stride %lld", (long long)c->x_row_stride);
    if (!backward) {
        if (!empty && !c->out) return fail(VY_ERR_INVALID, "null out");
        if (!aligned16(c->out) || c->out_row_stride % 8 || c->out_row_stride < c->hidden)
            return fail(VY_ERR_ALIGNMENT, "out %p, row stride %lld", c->out, (long long)c->out_row_stride);
    } else {
        if (!empty && (!c->d_out || !c->saved)) return fail(VY_ERR_INVALID, "backward needs d_out and saved");
        if (!aligned16(c->d_out) || c->d_out_row_stride % 8 || c->d_out_row_stride < c->hidden)
            return fail(VY_ERR_ALIGNMENT, "d_out %p, row stride %lld", c->d_out, (long long)c->d_out_row_stride);
        if (!aligned16(c->d_x) || !aligned16(c->d_w_gate) || !aligned16(c->d_w_up) || !aligned16(c->d_w_down) ||
            (c->d_x && (c->d_x_row_stride % 8 || c->d_x_row_stride < c->hidden)))
            return fail(VY_ERR_ALIGNMENT, "gradients must be 16-byte aligned (d_x row stride %lld)",
                        (long long)c->d_x_row_stride);
    }
    const size_t bytes = vy_gated_ffn_workspace_size(c, backward);
    if (!empty && (!c->workspace || c->workspace_bytes < bytes))
        return fail(VY_ERR_WORKSPACE, "workspace %zu bytes, %zu needed", c->workspace_bytes, bytes);
    return VY_OK;
}

int epi_store(TileProblem* q, int act_dtype, void* out, int64_t ldo) {
    q->epi.out = out;
    q->epi.ldo = ldo;
    return make_map_2d(&q->out, act_dtype, out, q->m, q->n, ldo, 64, 32);
}

#define VY_TRY(expr)                         \
    do {                                     \
        const int vy_st = (expr);            \
        if (vy_st != VY_OK) return vy_st;    \
    } while (0)

int k_blocks(int64_t k) { return static_cast<int>((k + 63) / 64); }

template <int ACT>
int forward(const vy_ffn_call* c, const ClusterCaps& caps, cudaStream_t s) {
    const int64_t T = c->n_tokens, H = c->hidden, I = c->inter;
    uint16_t* h = reinterpret_cast<uint16_t*>((reinterpret_cast<uintptr_t>(c->workspace) + 255) & ~uintptr_t(255));
    EpiParams e{};
    e.out = h;
    e.ldo = I;
    e.act = c->activation;
    e.saved = c->saved;
    e.saved_bands = saved_bands(T);
    e.part = h_parts(c) == 2 ? h_elems(c) : 0;
    const int t = static_cast<int>(T), parts = h_parts(c);
    if (T <= kStreamMaxGate) {
        const StreamCall gate{c->w_gate, c->w_up, c->x, c->x_row_stride, t, 1, c->inter, c->hidden, false, nullptr, 0, nullptr};
        VY_TRY((stream_launch<EPI_GATE, ACT>(gate, e, c->flags, caps, s)));
    } else {
        TileParams p{};
        TileProblem& q = tile_add(&p, T, I, k_blocks(H));
        tile_layout(&p, true, caps);
        VY_TRY(tile_operand(&q.a[0], ACT, c->x, T, H, c->x_row_stride, false, 128));
        VY_TRY(tile_operand(&q.b[0], ACT, c->w_gate, I, H, H, false, q.bn / 2));
        VY_TRY(tile_operand(&q.b[1], ACT, c->w_up, I, H, H, false, q.bn / 2));
        q.epi = e;
        p.flags = c->flags;
        VY_TRY((tile_launch<EPI_GATE, ACT>(p, caps, s)));
    }
    if (T <= kStreamMaxPlain) {
        EpiParams d{};
        d.out = c->out;
        d.ldo = c->out_row_stride;
        const StreamCall down{c->w_down, nullptr, h, I, t * parts, parts, c->hidden, c->inter, true, nullptr, 0, nullptr};
        return stream_launch<EPI_STORE, ACT>(down, d, c->flags, caps, s);
    }
    TileParams p{};
    TileProblem& q = tile_add(&p, T, H, k_blocks(I));
    tile_layout(&p, false, caps);
    VY_TRY(tile_operand(&q.a[0], ACT, h, T, I, I, false, 128));
    VY_TRY(tile_operand(&q.b[0], ACT, c->w_down, H, I, I, false, q.bn / 2));
    VY_TRY(epi_store(&q, ACT, c->out, c->out_row_stride));
    p.flags = c->flags;
    return tile_launch<EPI_STORE, ACT>(p, caps, s);
}

template <int ACT>
int backward(const vy_ffn_call* c, const ClusterCaps& caps, cudaStream_t s) {
    const int64_t T = c->n_tokens, H = c->hidden, I = c->inter;
    char* base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(c->workspace) + 255) & ~uintptr_t(255));
    const size_t each = h_bytes(c);
    const int parts = h_parts(c);
    const int64_t part = parts == 2 ? h_elems(c) : 0;
    uint16_t* dg = reinterpret_cast<uint16_t*>(base);
    uint16_t* du = reinterpret_cast<uint16_t*>(base + each);
    uint16_t* h = reinterpret_cast<uint16_t*>(base + 2 * each);
    const int t = static_cast<int>(T);
    EpiParams e{};
    e.act = c->activation;
    e.saved = c->saved;
    e.saved_bands = saved_bands(T);
    e.part = part;
    e.ldo = I;
    e.dg = dg;
    e.du = du;
    e.h = h;
    // dh streams Wd while its epilogue, a value at a time there, is short; d_x streams Wg and Wu as long
    // as the forward call would
    if (T <= kPartTokens) {
        const StreamCall dh{c->w_down, nullptr, c->d_out, c->d_out_row_stride, t, 1, c->inter, c->hidden, false,
                            nullptr, 0, nullptr};
        VY_TRY((stream_launch<EPI_DGATE, ACT, SRC_TMA, true>(dh, e, c->flags, caps, s)));
    } else {
        TileParams p{};
        TileProblem& q = tile_add(&p, T, I, k_blocks(H));
        tile_layout(&p, false, caps);
        q.b_mn = 1;
        VY_TRY(tile_operand(&q.a[0], ACT, c->d_out, T, H, c->d_out_row_stride, false, 128));
        VY_TRY(tile_operand(&q.b[0], ACT, c->w_down, I, H, I, true, 0));
        q.epi = e;
        p.flags = c->flags;
        VY_TRY((tile_launch<EPI_DGATE, ACT>(p, caps, s)));
    }
    TileParams p{};
    p.flags = c->flags;
    if (c->d_x && T <= kStreamMaxPlain) {
        EpiParams d{};
        d.out = c->d_x;
        d.ldo = c->d_x_row_stride;
        const StreamCall dx{c->w_gate, c->w_up, dg, I, t * parts, parts, c->hidden, c->inter, true, nullptr, 0, du};
        VY_TRY((stream_launch<EPI_STORE, ACT, SRC_TMA, true>(dx, d, c->flags, caps, s)));
    } else if (c->d_x) {      // K segments: dg with Wg, du with Wu
        TileProblem& q = tile_add(&p, T, H, k_blocks(I), 2);
        q.b_mn = 1;
        for (int i = 0; i < 2; ++i) {
            q.a_of[i] = q.b_of[i] = static_cast<uint8_t>(i);
            VY_TRY(tile_operand(&q.a[i], ACT, i ? du : dg, T, I, I, false, 128));
            VY_TRY(tile_operand(&q.b[i], ACT, i ? c->w_up : c->w_gate, H, I, H, true, 0));
        }
        VY_TRY(epi_store(&q, ACT, c->d_x, c->d_x_row_stride));
    }
    struct Grad {
        void* out;
        const void *a, *b;
        int64_t m, n, lda, ldb;
        bool b_parts;      // the hidden row's matrix is b (else a)
    };
    const Grad grads[3] = {{c->d_w_gate, dg, c->x, I, H, I, c->x_row_stride, false},
                           {c->d_w_up, du, c->x, I, H, I, c->x_row_stride, false},
                           {c->d_w_down, c->d_out, h, H, I, c->d_out_row_stride, I, true}};
    for (const Grad& g : grads) {
        if (!g.out) continue;
        TileProblem& q = tile_add(&p, g.m, g.n, k_blocks(T), parts);
        q.a_mn = q.b_mn = 1;
        for (int i = 0; i < parts; ++i) {
            uint8_t* of = g.b_parts ? q.b_of : q.a_of;
            of[i] = static_cast<uint8_t>(i);
            const int64_t at = i * part;
            if (i == 0 || !g.b_parts)
                VY_TRY(tile_operand(&q.a[i], ACT, static_cast<const uint16_t*>(g.a) + at, g.m, T, g.lda, true, 0));
            if (i == 0 || g.b_parts)
                VY_TRY(tile_operand(&q.b[i], ACT, static_cast<const uint16_t*>(g.b) + at, g.n, T, g.ldb, true, 0));
        }
        VY_TRY(epi_store(&q, ACT, g.out, g.n));
    }
    if (p.n_problems == 0) return VY_OK;
    tile_layout(&p, false, caps);
    return tile_launch<EPI_STORE, ACT>(p, caps, s);
}

}  // namespace
}  // namespace vy

using namespace vy;

extern "C" int64_t vy_gated_ffn_saved_floats(int64_t n_tokens, int32_t inter) {
    return n_tokens < 0 || inter < 0 ? 0 : saved_bands(n_tokens) * ((int64_t(inter) + 15) / 16) * kSavedBlock;
}

extern "C" size_t vy_gated_ffn_workspace_size(const vy_ffn_call* c, int32_t backward) {
    if (!c || c->n_tokens <= 0 || c->inter <= 0) return 0;
    return (backward ? 3 : 1) * h_bytes(c) + 256;
}

extern "C" int vy_gated_ffn_forward(const vy_ffn_call* c, void* stream) {
    int st;
    if ((st = check_ffn(c, false)) != VY_OK) return st;
    if (!device_info(&st)) return st;
    const ClusterCaps* caps = cluster_caps(&st);
    if (!caps) return st;
    if (c->n_tokens == 0) return ok();
    st = c->act_dtype == VY_BF16 ? forward<VY_BF16>(c, *caps, as_stream(stream)) : forward<VY_F16>(c, *caps, as_stream(stream));
    return st != VY_OK ? st : check_launch("vy_gated_ffn_forward");
}

extern "C" int vy_gated_ffn_backward(const vy_ffn_call* c, void* stream) {
    int st;
    if ((st = check_ffn(c, true)) != VY_OK) return st;
    if (!device_info(&st)) return st;
    const ClusterCaps* caps = cluster_caps(&st);
    if (!caps) return st;
    if (c->n_tokens == 0) {      // no token, no contribution: the weight gradients are zero
        const size_t bytes = size_t(c->hidden) * size_t(c->inter) * 2;
        for (void* w : {c->d_w_gate, c->d_w_up, c->d_w_down})
            if (w && cudaMemsetAsync(w, 0, bytes, as_stream(stream)) != cudaSuccess)
                return check_launch("vy_gated_ffn_backward");
        return ok();
    }
    st = c->act_dtype == VY_BF16 ? backward<VY_BF16>(c, *caps, as_stream(stream)) : backward<VY_F16>(c, *caps, as_stream(stream));
    return st != VY_OK ? st : check_launch("vy_gated_ffn_backward");
}
