// vy_int8.cu -- 8-bit integer linears: per-token quantisation, the scaled int8 product, and the
// gated feed-forward block on int8 weights.
//
// Bounds.  Quantisation: HBM (each value read once, kept in registers between the row maximum and
// the rounding).  The products: the weights' bytes for few tokens, the tensor cores' int8 rate
// (twice the bf16 rate) for many.
#include "vy_stream.cuh"
#include "vy_tile.cuh"

namespace vy {
namespace {

constexpr int kMaxK = 131072;      // 128 * 128 * k stays below 2^31
constexpr int kQuantThreads = 256;
constexpr int kQuantVecs = 4;      // 16-value pieces of a row a thread holds in registers

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

// ── quantisation ────────────────────────────────────────────────────────────────────────────

struct QuantParams {
    const void* x;
    int64_t x_stride, rows, cols;
    int8_t* codes;
    float* scales;
    bool vec;      // rows and codes take 16-byte accesses
};

// Nearest integer of the exact quotient x / s, ties to even.  t = x * (1/s) is within 2.3e-5 of
// x / s (two roundings of a value up to 127.5), so it decides every value that is not that near a
// tie; the rest (about one in 10^4) are divided in fp64, which separates any quotient of two fp32
// numbers from a tie.  `tiny`: 1 / s is out of range, fp64 for all.
__device__ __forceinline__ int quant_code(float x, float s, float inv, bool tiny) {
    float t = x * inv;
    float r = rintf(t);
    if (tiny || fabsf(fabsf(t - r) - 0.5f) < 1e-4f) r = static_cast<float>(rint(double(x) / double(s)));
    return static_cast<int>(fminf(fmaxf(r, -127.f), 127.f));
}

template <int DT>
__device__ __forceinline__ void load16(const void* x, int64_t at, float (&v)[16]) {
    if constexpr (DT == VY_F32) {
        const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(x) + at);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 f = p[q];
            v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
        }
    } else {
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(x) + at);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint4 u = p[q];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[8 * q + 2 * j] = act_from_bits<DT>(w[j] & 0xFFFFu);
                v[8 * q + 2 * j + 1] = act_from_bits<DT>(w[j] >> 16);
            }
        }
    }
}

// One block per row.
template <int DT>
__global__ void __launch_bounds__(kQuantThreads) quantize_kernel(QuantParams p) {
    __shared__ uint32_t part[kQuantThreads / 32];
    grid_dependency_wait();
    grid_dependents_launch();
    const int64_t row = blockIdx.x;
    const int64_t base = row * p.x_stride;
    const int tid = threadIdx.x;
    // magnitudes order like their bit patterns, NaN above infinity: one integer maximum
    uint32_t top = 0;
    float keep[kQuantVecs][16];
    const int64_t pieces = p.vec ? p.cols / 16 : 0;
    const bool fits = pieces <= int64_t(kQuantVecs) * kQuantThreads;
    if (fits) {
#pragma unroll
        for (int i = 0; i < kQuantVecs; ++i) {
            const int64_t at = tid + int64_t(i) * kQuantThreads;
            if (at < pieces) {
                load16<DT>(p.x, base + at * 16, keep[i]);
#pragma unroll
                for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(keep[i][j]) & 0x7FFFFFFFu);
            }
        }
    } else {
        for (int64_t at = tid; at < pieces; at += kQuantThreads) {
            float v[16];
            load16<DT>(p.x, base + at * 16, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        }
    }
    for (int64_t k = pieces * 16 + tid; k < p.cols; k += kQuantThreads)
        top = max(top, __float_as_uint(load_as_float(p.x, DT, base + k)) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((tid & 31) == 0) part[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQuantThreads / 32; ++w) top = max(top, part[w]);

    const bool finite = top < 0x7F800000u;
    const float scale = finite ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7FC00000u);
    if (tid == 0) p.scales[row] = scale;
    const bool zero = !(scale > 0.f);          // a zero row, or NaN
    const bool tiny = scale < 1e-30f;
    const float inv = zero || tiny ? 0.f : __fdiv_rn(1.f, scale);
    int8_t* out = p.codes + row * p.cols;
    auto put16 = [&](int64_t at, const float (&v)[16]) {
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            w[q] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[q] |= (zero ? 0u : uint32_t(quant_code(v[4 * q + j], scale, inv, tiny)) & 0xFFu) << (8 * j);
        }
        *reinterpret_cast<uint4*>(out + at * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    };
    if (fits) {
#pragma unroll
        for (int i = 0; i < kQuantVecs; ++i) {
            const int64_t at = tid + int64_t(i) * kQuantThreads;
            if (at < pieces) put16(at, keep[i]);
        }
    } else {
        for (int64_t at = tid; at < pieces; at += kQuantThreads) {
            float v[16];
            load16<DT>(p.x, base + at * 16, v);
            put16(at, v);
        }
    }
    for (int64_t k = pieces * 16 + tid; k < p.cols; k += kQuantThreads)
        out[k] = static_cast<int8_t>(zero ? 0 : quant_code(load_as_float(p.x, DT, base + k), scale, inv, tiny));
}

int launch_quantize(const void* x, int dtype, int64_t stride, int64_t rows, int64_t cols, int8_t* codes, float* scales,
                    cudaStream_t s) {
    QuantParams p{x, stride, rows, cols, codes, scales, false};
    const int64_t size = dtype == VY_F32 ? 4 : 2;
    p.vec = aligned16(x) && (rows == 1 || (stride * size) % 16 == 0) && aligned16(codes) && (rows == 1 || cols % 16 == 0);
    auto kern = dtype == VY_F32 ? quantize_kernel<VY_F32> : dtype == VY_F16 ? quantize_kernel<VY_F16> : quantize_kernel<VY_BF16>;
    const cudaError_t e = launch_chained(kern, dim3(static_cast<unsigned>(rows)), dim3(kQuantThreads), 0, s, p);
    if (e != cudaSuccess) return fail(VY_ERR_CUDA, "int8 quantise launch: %s", cudaGetErrorString(e));
    return VY_OK;
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
};

template <bool GATE>
int launch_product(const Product& a, bool first, const DeviceInfo* dev, cudaStream_t s) {
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
    if (a.tokens <= kStreamMaxTokens)
        return stream_launch<EPI, VY_BF16>(a.w[0], a.w[1], a.codes, a.codes_ld, static_cast<int>(a.tokens), a.n, a.k,
                                           !first, e, a.flags, dev, s);
    TileParams p{};
    TileProblem& q = p.prob[0];
    q.m = static_cast<int>(a.tokens);
    q.n = a.n;
    q.bn = tile_columns(a.tokens, GATE ? 2 * int64_t(a.n) : a.n, dev->sm_count / 2);
    q.nk[0] = (a.k + 127) / 128;
    VY_TRY(tile_operand(&q.a[0], VY_E4M3, a.codes, a.tokens, a.k, a.codes_ld, false, 128));
    VY_TRY(tile_operand(&q.b[0], VY_E4M3, a.w[0], a.n, a.k, a.k, false, q.bn / 2));
    if (GATE) VY_TRY(tile_operand(&q.b[1], VY_E4M3, a.w[1], a.n, a.k, a.k, false, q.bn / 2));
    q.epi = e;
    p.flags = a.flags;
    tile_place(&p, 0, GATE);
    return tile_launch<EPI, VY_BF16>(p, dev, s);
}

bool float_dtype(int d) { return d == VY_BF16 || d == VY_F16 || d == VY_F32; }

int check_linear(const vy_int8_linear_call* c) {
    if (!c) return fail(VY_ERR_INVALID, "null call");
    if (c->n_tokens < 0 || c->k <= 0 || c->n <= 0)
        return fail(VY_ERR_INVALID, "n_tokens %lld, k %d, n %d", (long long)c->n_tokens, c->k, c->n);
    if (c->n_tokens > (int64_t(1) << 30)) return fail(VY_ERR_UNSUPPORTED, "n_tokens %lld", (long long)c->n_tokens);
    if (c->k % 16 || c->k >= kMaxK) return fail(VY_ERR_UNSUPPORTED, "k %d must be a multiple of 16 below %d", c->k, kMaxK);
    if (!float_dtype(c->out_dtype) || (c->bias && !float_dtype(c->bias_dtype)))
        return fail(VY_ERR_UNSUPPORTED, "out / bias dtype code %d / %d", c->out_dtype, c->bias_dtype);
    if (c->n_tokens == 0) return VY_OK;
    if (!c->codes || !c->scales || !c->weight || !c->weight_scales || !c->out) return fail(VY_ERR_INVALID, "null operand");
    if (!aligned16(c->codes) || !aligned16(c->weight) || c->codes_row_stride % 16 || c->codes_row_stride < c->k)
        return fail(VY_ERR_ALIGNMENT, "codes and weight must have 16-byte aligned rows (row stride %lld)",
                    (long long)c->codes_row_stride);
    if (c->out_row_stride < c->n) return fail(VY_ERR_INVALID, "out row stride %lld", (long long)c->out_row_stride);
    const size_t bytes = vy_int8_linear_workspace_size(c);
    if (bytes && (!c->workspace || c->workspace_bytes < bytes))
        return fail(VY_ERR_WORKSPACE, "workspace %zu bytes, %zu needed", c->workspace_bytes, bytes);
    return VY_OK;
}

// Buffers of the int8 block inside its workspace.
struct FfnLayout {
    int8_t *x_codes, *h_codes;
    float *x_scales, *h_scales, *h;
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
    if (!device_info(&st)) return st;
    st = launch_quantize(x, x_dtype, x_row_stride, rows, cols, codes, scales, as_stream(stream));
    return st != VY_OK ? st : check_launch("vy_int8_quantize");
}

extern "C" size_t vy_int8_linear_workspace_size(const vy_int8_linear_call*) { return 0; }

extern "C" int vy_int8_linear(const vy_int8_linear_call* c, void* stream) {
    int st;
    if ((st = check_linear(c)) != VY_OK) return st;
    const DeviceInfo* dev = device_info(&st);
    if (!dev) return st;
    if (c->n_tokens == 0) return ok();
    Product a{c->codes, c->codes_row_stride, c->scales, {c->weight, nullptr}, {c->weight_scales, nullptr}, c->n_tokens,
              c->k, c->n, c->out, c->out_row_stride, c->out_dtype, 0, c->bias, c->bias_dtype, c->flags};
    st = launch_product<false>(a, true, dev, as_stream(stream));
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
    if (c->n_tokens == 0) return ok();
    cudaStream_t s = as_stream(stream);
    const FfnLayout L = ffn_layout(
        c, reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(c->workspace) + 255) & ~uintptr_t(255)));
    VY_TRY(launch_quantize(c->x, c->act_dtype, c->x_row_stride, c->n_tokens, c->hidden, L.x_codes, L.x_scales, s));
    Product gu{L.x_codes, c->hidden, L.x_scales, {c->w_gate, c->w_up}, {c->gate_scales, c->up_scales}, c->n_tokens,
               c->hidden, c->inter, L.h, c->inter, VY_F32, c->activation, nullptr, 0, c->flags};
    VY_TRY(launch_product<true>(gu, false, dev, s));
    VY_TRY(launch_quantize(L.h, VY_F32, c->inter, c->n_tokens, c->inter, L.h_codes, L.h_scales, s));
    Product down{L.h_codes, c->inter, L.h_scales, {c->w_down, nullptr}, {c->down_scales, nullptr}, c->n_tokens, c->inter,
                 c->hidden, c->out, c->out_row_stride, c->act_dtype, 0, nullptr, 0, c->flags};
    VY_TRY(launch_product<false>(down, false, dev, s));
    return check_launch("vy_int8_gated_ffn");
}
