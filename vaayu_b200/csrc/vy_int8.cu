// vy_int8.cu -- 8-bit integer linears: per-token quantisation, the scaled int8 product, and the
// gated feed-forward block on int8 weights.
//
// Bounds.  Quantisation: HBM (each value read once, kept in registers between the row maximum and
// the rounding).  The products: the weights' bytes for few tokens, the tensor cores' int8 rate
// (twice the bf16 rate) for many.
#include "vy_quant.cuh"
#include "vy_stream.cuh"
#include "vy_tile.cuh"

namespace vy {
namespace {

constexpr int kMaxK = 131072;      // 128 * 128 * k stays below 2^31
constexpr int kMaxN = 0x7FFFFF00;      // rounded up to whole tiles it is still an int
size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// ── quantisation ────────────────────────────────────────────────────────────────────────────

struct QuantParams {
    const void* x;
    int64_t x_stride, rows, cols;
    int8_t* codes;
    float* scales;
    bool vec;      // rows take 16-byte loads, codes the stores that go with them
};

// One block per row; the row stays in registers between its maximum and its codes.
template <int DT, int THREADS, int UNITS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) quantize_kernel(QuantParams p) {
    using P = Piece<DT>;
    __shared__ uint32_t part[THREADS / 32];
    grid_dependency_wait();
    grid_dependents_launch();
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const int64_t size = DT == VY_F32 ? 4 : 2;
    const unsigned char* src = reinterpret_cast<const unsigned char*>(p.x) + row * p.x_stride * size;
    const uint4* pieces = reinterpret_cast<const uint4*>(src);
    const int64_t n = p.vec ? p.cols / P::N : 0;
    const bool fits = n <= int64_t(UNITS) * THREADS;
    uint4 keep[UNITS];
    uint32_t top = 0;
    if (fits) {
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int64_t at = tid + i * THREADS;
            keep[i] = at < n ? ld_piece(pieces + at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < UNITS; ++i) top = P::top(top, keep[i]);
    } else {
        for (int64_t at = tid; at < n; at += THREADS) top = P::top(top, ld_piece(pieces + at));
    }
    top = P::wide(top);
    for (int64_t k = n * P::N + tid; k < p.cols; k += THREADS)
        top = max(top, __float_as_uint(load_as_float(src, DT, k)) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((tid & 31) == 0) part[tid >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, part[(tid & 31) % (THREADS / 32)]);

    const RowScale r = row_scale(top);
    if (tid == 0) p.scales[row] = r.s;
    int8_t* out = p.codes + row * p.cols;
    if (fits) {
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int64_t at = tid + i * THREADS;
            if (at < n) put_piece<DT>(out, at, keep[i], r);
        }
    } else {
        for (int64_t at = tid; at < n; at += THREADS) put_piece<DT>(out, at, ld_piece(pieces + at), r);
    }
    put_tail<DT>(out, src, n * P::N + tid, p.cols, THREADS, r);
}

template <int DT>
int launch_quantize_as(const QuantParams& p, int sm_count, cudaStream_t s) {
    const int64_t n = p.cols / Piece<DT>::N;
    // Threads of a row's block, and 16-byte pieces each keeps in registers.  Many rows: few threads
    // with many pieces, so that several blocks share an SM and one's loads run under another's
    // arithmetic.  Fewer rows than SMs: as many threads as the row can use, since one block's latency
    // is the call's.  (A row past 8192 pieces is read twice.)  Device time in us, threads x pieces:
    //   5 x 7168 (896 pieces)          64x2 4.5   256x2 2.8   1024x2 2.0   256x8 2.1   1024x8 2.8
    //   128 x 2048 (256)               64x2 3.0   256x2 1.8   1024x2 2.0
    //   64 x 14336 (1792)              256x2 4.8  1024x2 2.8  256x8 3.5    512x8 3.2
    //   4096 x 1024 (128)              64x2 5.1   128x4 7.0   256x2 9.7
    //   4096 x 4096 (512)              64x2 13.8  128x4 12.0  256x2 14.5   256x8 19.8
    //   4096 x 14336 (1792)            128x4 45   256x8 36    512x8 50     1024x8 85
    //   2048 x 32768 (4096)            256x8 50   512x8 41    1024x8 59
    //   1024 x 65536 (8192)            256x8 63   512x8 53    1024x8 46
    // Rows that take no 16-byte loads (an odd length, an odd start) go value by value in blocks of 64:
    // 4096 x 14335 103 us in bf16 and 123 in fp32, where 14336 takes 36 and 47.
    const bool few = p.rows <= sm_count;
    void (*kern)(QuantParams) = quantize_kernel<DT, 1024, 8, 1>;
    int threads = 1024;
    if (few ? n <= 64 : n <= 128)
        kern = quantize_kernel<DT, 64, 2, 8>, threads = 64;
    else if (few && n <= 256)
        kern = quantize_kernel<DT, 256, 2, 4>, threads = 256;
    else if (!few && n <= 512)
        kern = quantize_kernel<DT, 128, 4, 8>, threads = 128;
    else if (few && n <= 2048)
        kern = quantize_kernel<DT, 1024, 2, 1>, threads = 1024;
    else if (n <= 2048)
        kern = quantize_kernel<DT, 256, 8, 4>, threads = 256;
    else if (n <= 4096)
        kern = quantize_kernel<DT, 512, 8, 2>, threads = 512;
    const cudaError_t e = launch_chained(kern, dim3(static_cast<unsigned>(p.rows)), dim3(threads), 0, s, p);
    return e == cudaSuccess ? VY_OK : fail(VY_ERR_CUDA, "int8 quantise launch: %s", cudaGetErrorString(e));
}

int launch_quantize(const void* x, int dtype, int64_t stride, int64_t rows, int64_t cols, int8_t* codes, float* scales,
                    int sm_count, cudaStream_t s) {
    QuantParams p{x, stride, rows, cols, codes, scales, false};
    const int64_t size = dtype == VY_F32 ? 4 : 2;
    p.vec = aligned16(x) && (rows == 1 || (stride * size) % 16 == 0) && aligned16(codes) && (rows == 1 || cols % 8 == 0);
    return dtype == VY_F32   ? launch_quantize_as<VY_F32>(p, sm_count, s)
           : dtype == VY_F16 ? launch_quantize_as<VY_F16>(p, sm_count, s)
                             : launch_quantize_as<VY_BF16>(p, sm_count, s);
}

// ── products ────────────────────────────────────────────────────────────────────────────────

#define VY_TRY(expr)                         \
    do {                                     \
        const int vy_st = (expr);            \
        if (vy_st != VY_OK) return vy_st;    \
    } while (0)

// out = scaled codes x weight^T (`first`: no kernel of the same call runs in front of it); gate: w[0], w[1] are gate and up and out is h (fp32).
struct Product {
    const int8_t* codes;
    int64_t codes_ld;
    const float* scales;
    const int8_t* w[2];
    const float* ws[2];
    int64_t tokens;
    int k, n;
    void* out;
    int64_t ldo;
    int out_dtype, act;
    const void* bias;
    int bias_dtype;
    int32_t* flags;
    uint32_t* maxima;      // GATE, few tokens: the largest |h| of each CTA's columns, for the down product
    int n_maxima;
};

template <bool GATE>
int launch_product(const Product& a, bool first, const ClusterCaps& caps, cudaStream_t s) {
    EpiParams e{};
    e.out = a.out;
    e.ldo = a.ldo;
    e.out_dtype = a.out_dtype;
    e.vec = aligned16(a.out) && (a.ldo * (a.out_dtype == VY_F32 ? 4 : 2)) % 16 == 0;
    e.act = a.act;
    e.row_scale = a.scales;
    e.col_scale[0] = a.ws[0];
    e.col_scale[1] = a.ws[1];
    e.bias = a.bias;
    e.bias_dtype = a.bias_dtype;
    constexpr int EPI = GATE ? EPI_I8GATE : EPI_I8;
    if (a.tokens <= (GATE ? kStreamMaxGate : kStreamMaxPlain)) {
        const StreamCall c{a.w[0], a.w[1], a.codes, a.codes_ld, static_cast<int>(a.tokens), 1, a.n, a.k, !first,
                           a.maxima, a.n_maxima, nullptr};
        return stream_launch<EPI, VY_BF16>(c, e, a.flags, caps, s);
    }
    TileParams p{};
    TileProblem& q = tile_add(&p, a.tokens, a.n, (a.k + 127) / 128);
    tile_layout(&p, GATE, caps);
    VY_TRY(tile_operand(&q.a[0], VY_E4M3, a.codes, a.tokens, a.k, a.codes_ld, false, 128));
    VY_TRY(tile_operand(&q.b[0], VY_E4M3, a.w[0], a.n, a.k, a.k, false, q.bn / 2));
    if (GATE) VY_TRY(tile_operand(&q.b[1], VY_E4M3, a.w[1], a.n, a.k, a.k, false, q.bn / 2));
    q.epi = e;
    p.flags = a.flags;
    return tile_launch<EPI, VY_BF16>(p, caps, s);
}

bool float_dtype(int d) { return d == VY_BF16 || d == VY_F16 || d == VY_F32; }

int check_linear(const vy_int8_linear_call* c) {
    if (!c) return fail(VY_ERR_INVALID, "null call");
    if (c->n_tokens < 0 || c->k <= 0 || c->n <= 0)
        return fail(VY_ERR_INVALID, "n_tokens %lld, k %d, n %d", (long long)c->n_tokens, c->k, c->n);
    if (c->n_tokens > (int64_t(1) << 30)) return fail(VY_ERR_UNSUPPORTED, "n_tokens %lld", (long long)c->n_tokens);
    if (c->k % 16 || c->k >= kMaxK) return fail(VY_ERR_UNSUPPORTED, "k %d must be a multiple of 16 below %d", c->k, kMaxK);
    if (c->n > kMaxN) return fail(VY_ERR_UNSUPPORTED, "n %d above %d", c->n, kMaxN);
    if (!float_dtype(c->out_dtype) || (c->bias && !float_dtype(c->bias_dtype)))
        return fail(VY_ERR_UNSUPPORTED, "out / bias dtype code %d / %d", c->out_dtype, c->bias_dtype);
    if (c->n_tokens == 0) return VY_OK;
    if (!c->codes || !c->scales || !c->weight || !c->weight_scales || !c->out) return fail(VY_ERR_INVALID, "null operand");
    if (!aligned16(c->codes) || !aligned16(c->weight) || c->codes_row_stride % 16 || c->codes_row_stride < c->k)
        return fail(VY_ERR_ALIGNMENT, "codes and weight must have 16-byte aligned rows (row stride %lld)",
                    (long long)c->codes_row_stride);
    if (c->out_row_stride < c->n) return fail(VY_ERR_INVALID, "out row stride %lld", (long long)c->out_row_stride);
    return VY_OK;
}

// Buffers of the int8 block inside its workspace.
struct FfnLayout {
    int8_t *x_codes, *h_codes;
    float *x_scales, *h_scales, *h;
    uint32_t* maxima;
    size_t bytes;
};
FfnLayout ffn_layout(const vy_int8_ffn_call* c, char* base) {
    FfnLayout L{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* p = base ? base + at : nullptr;
        at += align256(bytes);
        return p;
    };
    const size_t T = size_t(c->n_tokens);
    L.x_codes = reinterpret_cast<int8_t*>(take(T * c->hidden));
    L.x_scales = reinterpret_cast<float*>(take(T * 4));
    L.h = reinterpret_cast<float*>(take(T * c->inter * 4));
    L.h_codes = reinterpret_cast<int8_t*>(take(T * c->inter));
    L.h_scales = reinterpret_cast<float*>(take(T * 4));
    if (c->n_tokens <= kSourceTokens)      // at most 8 CTAs a unit
        L.maxima = reinterpret_cast<uint32_t*>(take(size_t((c->inter + kStreamRows - 1) / kStreamRows) * 8 * T * 4));
    L.bytes = at + 256;
    return L;
}

int check_ffn(const vy_int8_ffn_call* c) {
    if (!c) return fail(VY_ERR_INVALID, "null call");
    if (c->act_dtype != VY_BF16 && c->act_dtype != VY_F16)
        return fail(VY_ERR_UNSUPPORTED, "activation dtype code %d (bf16 or fp16)", c->act_dtype);
    if (c->activation != VY_ACT_SILU && c->activation != VY_ACT_GELU_TANH)
        return fail(VY_ERR_UNSUPPORTED, "activation code %d", c->activation);
    if (c->n_tokens < 0 || c->hidden <= 0 || c->inter <= 0)
        return fail(VY_ERR_INVALID, "n_tokens %lld, hidden %d, inter %d", (long long)c->n_tokens, c->hidden, c->inter);
    if (c->n_tokens > (int64_t(1) << 30)) return fail(VY_ERR_UNSUPPORTED, "n_tokens %lld", (long long)c->n_tokens);
    if (c->hidden % 16 || c->inter % 16 || c->hidden >= kMaxK || c->inter >= kMaxK)
        return fail(VY_ERR_UNSUPPORTED, "hidden %d and inter %d must be multiples of 16 below %d", c->hidden, c->inter, kMaxK);
    if (c->n_tokens == 0) return VY_OK;
    if (!c->x || !c->w_gate || !c->w_up || !c->w_down || !c->gate_scales || !c->up_scales || !c->down_scales || !c->out)
        return fail(VY_ERR_INVALID, "null operand");
    if (!aligned16(c->w_gate) || !aligned16(c->w_up) || !aligned16(c->w_down))
        return fail(VY_ERR_ALIGNMENT, "weights must be 16-byte aligned");
    if (c->x_row_stride < c->hidden || c->out_row_stride < c->hidden)
        return fail(VY_ERR_INVALID, "row strides %lld, %lld", (long long)c->x_row_stride, (long long)c->out_row_stride);
    const size_t bytes = vy_int8_gated_ffn_workspace_size(c);
    if (!c->workspace || c->workspace_bytes < bytes)
        return fail(VY_ERR_WORKSPACE, "workspace %zu bytes, %zu needed", c->workspace_bytes, bytes);
    return VY_OK;
}

}  // namespace
}  // namespace vy

using namespace vy;

extern "C" int vy_int8_quantize(const void* x, int32_t x_dtype, int64_t x_row_stride, int64_t rows, int64_t cols,
                                int8_t* codes, float* scales, void* stream) {
    int st;
    if (!float_dtype(x_dtype)) return fail(VY_ERR_UNSUPPORTED, "x dtype code %d (bf16, fp16 or fp32)", x_dtype);
    if (rows < 0 || cols <= 0) return fail(VY_ERR_INVALID, "rows %lld, cols %lld", (long long)rows, (long long)cols);
    if (rows > 0x7FFFFFFFll) return fail(VY_ERR_UNSUPPORTED, "rows %lld", (long long)rows);
    if (rows == 0) return ok();
    if (!x || !codes || !scales) return fail(VY_ERR_INVALID, "null operand");
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    st = launch_quantize(x, x_dtype, x_row_stride, rows, cols, codes, scales, dev->sm_count, as_stream(stream));
    return st != VY_OK ? st : check_launch("vy_int8_quantize");
}

extern "C" int vy_int8_linear(const vy_int8_linear_call* c, void* stream) {
    int st;
    if ((st = check_linear(c)) != VY_OK) return st;
    if (!device_info(&st)) return st;
    const ClusterCaps* caps = cluster_caps(&st);
    if (!caps) return st;
    if (c->n_tokens == 0) return ok();
    Product a{c->codes, c->codes_row_stride, c->scales, {c->weight, nullptr}, {c->weight_scales, nullptr}, c->n_tokens,
              c->k, c->n, c->out, c->out_row_stride, c->out_dtype, 0, c->bias, c->bias_dtype, c->flags, nullptr, 0};
    st = launch_product<false>(a, true, *caps, as_stream(stream));
    return st != VY_OK ? st : check_launch("vy_int8_linear");
}

extern "C" size_t vy_int8_gated_ffn_workspace_size(const vy_int8_ffn_call* c) {
    if (!c || c->n_tokens <= 0 || c->hidden <= 0 || c->inter <= 0) return 0;
    return ffn_layout(c, nullptr).bytes;
}

extern "C" int vy_int8_gated_ffn(const vy_int8_ffn_call* c, void* stream) {
    int st;
    if ((st = check_ffn(c)) != VY_OK) return st;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    const ClusterCaps* caps = cluster_caps(&st);
    if (!caps) return st;
    if (c->n_tokens == 0) return ok();
    cudaStream_t s = as_stream(stream);
    const FfnLayout L = ffn_layout(
        c, reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(c->workspace) + 255) & ~uintptr_t(255)));
    const int t = static_cast<int>(c->n_tokens);
    EpiParams d{};
    d.out = c->out;
    d.ldo = c->out_row_stride;
    d.out_dtype = c->act_dtype;
    d.col_scale[0] = c->down_scales;
    if (c->n_tokens <= kSourceTokens) {
        const int nk = (c->hidden + 127) / 128;
        const int ctas = stream_ctas(2, t, 1, c->inter, nk, *caps);
        EpiParams g{};
        g.out = L.h;
        g.ldo = c->inter;
        g.act = c->activation;
        g.col_scale[0] = c->gate_scales;
        g.col_scale[1] = c->up_scales;
        // the rows' maxima taken in every CTA: worth a launch while a row set is small (32 KB)
        const bool rows = c->n_tokens * c->hidden <= 16384 && aligned16(c->x) && (t == 1 || c->x_row_stride % 8 == 0);
        if (rows) {
            const StreamCall gate{c->w_gate, c->w_up, c->x, c->x_row_stride, t, 1, c->inter, c->hidden, false, L.maxima, ctas, nullptr};
            VY_TRY(c->act_dtype == VY_BF16 ? (stream_launch<EPI_I8GATE, VY_BF16, SRC_ROWS>(gate, g, c->flags, *caps, s))
                                           : (stream_launch<EPI_I8GATE, VY_F16, SRC_ROWS>(gate, g, c->flags, *caps, s)));
        } else {
            VY_TRY(launch_quantize(c->x, c->act_dtype, c->x_row_stride, c->n_tokens, c->hidden, L.x_codes, L.x_scales,
                                   dev->sm_count, s));
            g.row_scale = L.x_scales;
            const StreamCall gate{c->w_gate, c->w_up, L.x_codes, c->hidden, t, 1, c->inter, c->hidden, true, L.maxima, ctas, nullptr};
            VY_TRY((stream_launch<EPI_I8GATE, VY_BF16>(gate, g, c->flags, *caps, s)));
        }
        const StreamCall down{c->w_down, nullptr, L.h, c->inter, t, 1, c->hidden, c->inter, true, L.maxima, ctas, nullptr};
        VY_TRY((stream_launch<EPI_I8, VY_BF16, SRC_HIDDEN>(down, d, c->flags, *caps, s)));
        return check_launch("vy_int8_gated_ffn");
    }
    VY_TRY(launch_quantize(c->x, c->act_dtype, c->x_row_stride, c->n_tokens, c->hidden, L.x_codes, L.x_scales, dev->sm_count, s));
    Product gu{L.x_codes, c->hidden, L.x_scales, {c->w_gate, c->w_up}, {c->gate_scales, c->up_scales}, c->n_tokens,
               c->hidden, c->inter, L.h, c->inter, VY_F32, c->activation, nullptr, 0, c->flags, nullptr, 0};
    VY_TRY(launch_product<true>(gu, false, *caps, s));
    VY_TRY(launch_quantize(L.h, VY_F32, c->inter, c->n_tokens, c->inter, L.h_codes, L.h_scales, dev->sm_count, s));
    Product down{L.h_codes, c->inter, L.h_scales, {c->w_down, nullptr}, {c->down_scales, nullptr}, c->n_tokens, c->inter,
                 c->hidden, c->out, c->out_row_stride, c->act_dtype, 0, nullptr, 0, c->flags, nullptr, 0};
    VY_TRY(launch_product<false>(down, false, *caps, s));
    return check_launch("vy_int8_gated_ffn");
}
