// vy_dense.cuh -- what the dense 16-bit and int8 operators share: activations, epilogue
// parameters, vector stores.
#pragma once

#include "vy_umma.cuh"

namespace vy {

// ── activations of a gated block and their derivatives (fp32) ───────────────────────────────

// Both are g times a sigmoid: silu(g) = g s(g), and since (1 + tanh v) / 2 = s(2v), gelu_tanh(g) =
// g s(2 sqrt(2/pi) (g + 0.044715 g^3)).  One exponential and one approximate division (2 ulp): no
// branch, so the loads of a tile's other columns are not held up behind it.  (The two ulp are far below
// the 16-bit roundings; in the int8 block they move the codes of h that lie that near to a tie.)
constexpr double kGeluCubic = 0.044715, kGeluScale = 1.5957691216057308;      // 2 sqrt(2/pi)
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + expf(-z)); }
__device__ __forceinline__ float gate_arg(float g, int act) {
    return act == VY_ACT_SILU ? g : float(kGeluScale) * (g + float(kGeluCubic) * g * g * g);
}
__device__ __forceinline__ float gate_act(float g, int act) { return g * sigmoid(gate_arg(g, act)); }
// (value, derivative): d(g s(z)) = s + g s (1 - s) z'
__device__ __forceinline__ float2 gate_act_grad(float g, int act) {
    const float s = sigmoid(gate_arg(g, act));
    // beyond +-16 gelu's s (1 - s) is zero; the clamp keeps z' finite there
    const float c = fminf(fmaxf(g, -16.f), 16.f);
    const float dz = act == VY_ACT_SILU ? 1.f : float(kGeluScale) + float(3 * kGeluScale * kGeluCubic) * c * c;
    const float gs = g * s;
    return make_float2(gs, s + gs * (1.f - s) * dz);
}

template <int ACT>
__device__ __forceinline__ uint32_t pack_act(float lo, float hi) {
    if constexpr (ACT == VY_BF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    } else {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t*>(&v);
    }
}

// 16 consecutive values of a row as 16-bit floats; `valid` of them (a multiple of 8) are stored.
template <int ACT>
__device__ __forceinline__ void store16(uint16_t* dst, const float (&v)[16], int valid) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (valid >= 8 * (h + 1)) {
            uint4 o;
            o.x = pack_act<ACT>(v[8 * h + 0], v[8 * h + 1]);
            o.y = pack_act<ACT>(v[8 * h + 2], v[8 * h + 3]);
            o.z = pack_act<ACT>(v[8 * h + 4], v[8 * h + 5]);
            o.w = pack_act<ACT>(v[8 * h + 6], v[8 * h + 7]);
            *reinterpret_cast<uint4*>(dst + 8 * h) = o;
        }
    }
}

__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float v) {
    switch (dtype) {
        case VY_BF16: reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v); break;
        case VY_F16: reinterpret_cast<__half*>(p)[i] = __float2half_rn(v); break;
        default: reinterpret_cast<float*>(p)[i] = v;
    }
}

// Up to 16 consecutive values at element `at` of a row in `dtype`; vec: 16-byte stores are aligned
// and `valid` is 16.
__device__ __forceinline__ void store16_dyn(void* p, int dtype, int64_t at, const float (&v)[16], int valid, bool vec) {
    if (vec && valid == 16) {
        if (dtype == VY_BF16) {
            store16<VY_BF16>(reinterpret_cast<uint16_t*>(p) + at, v, 16);
        } else if (dtype == VY_F16) {
            store16<VY_F16>(reinterpret_cast<uint16_t*>(p) + at, v, 16);
        } else {
            float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at);
#pragma unroll
            for (int q = 0; q < 4; ++q) d[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (j < valid) store_as(p, dtype, at + j, v[j]);
}

// g and u in fp32 between the passes, in the order the tile epilogues move them: blocks of 32 tokens x
// 16 channels, g before u, each [4 channels][32 tokens][4 channels], so that a warp (a token per lane)
// reads and writes its chunk of 16 columns as eight whole 512-byte lines.  (One column after another
// over all tokens, 32 separate 128-byte lines a chunk, took dh at 2048 x 4096 x 14336 235 us beside
// 214 this way.)
constexpr int kSavedBlock = 2 * 16 * 32;
__host__ __device__ constexpr int64_t saved_bands(int64_t tokens) { return (tokens + 31) / 32; }
__device__ __forceinline__ int64_t saved_at(int64_t bands, int64_t token, int channel) {
    return ((channel >> 4) * bands + (token >> 5)) * kSavedBlock + ((channel >> 2) & 3) * 128 + (token & 31) * 4 +
           (channel & 3);
}

// Calls of up to this many tokens keep the hidden row h (and dg, du) as two 16-bit parts, high and low,
// and run both through the next product: rounding it to one part adds as much error as rounding the
// result does, and with few tokens the few roundings do not average out.  The products there cost
// their weights' bytes, so the second part is free.  (Both parts have the type's range: an fp16 h beyond
// 65504 is infinite.)  With more tokens a second part would double the next products' operations.
constexpr int kPartTokens = 32;
template <int ACT>
__device__ __forceinline__ float low_part(float v) {
    const float rest = v - round_act<ACT>(v);
    return fabsf(rest) < INFINITY ? rest : 0.f;      // an overflowed or NaN high part says it all
}

// What a GEMM's epilogue does with its sums.
enum Epilogue {
    EPI_STORE = 0,   // out = sum, in the activation type
    EPI_GATE = 1,    // h = act(g) * u in the activation type; g and u kept in fp32 when `saved`
    EPI_DGATE = 2,   // from dh, g, u: dg, du and h in the activation type
    EPI_I8 = 3,      // out = (int32 sum * row scale) * column scale (+ bias)
    EPI_I8GATE = 4   // h = act(g) * u in fp32, g and u scaled like EPI_I8
};
__host__ __device__ constexpr bool epi_is_gate(int e) { return e == EPI_GATE || e == EPI_I8GATE; }
__host__ __device__ constexpr bool epi_is_i8(int e) { return e == EPI_I8 || e == EPI_I8GATE; }

struct EpiParams {
    void* out;               // rows = tokens (or weight rows of a weight gradient)
    int64_t ldo;
    int out_dtype;
    int vec;                 // out rows take 16-byte stores
    int act;                 // vy_activation
    float* saved;            // g and u, see saved_at
    int64_t saved_bands;     // groups of 32 tokens in it
    uint16_t *dg, *du, *h;   // EPI_DGATE, rows `ldo` apart
    // When not 0, a hidden row (h, dg, du) is kept as a sum of two 16-bit parts, the second this many
    // elements behind the first: see kPartTokens.
    int64_t part;
    const float* row_scale;
    const float* col_scale[2];
    const void* bias;
    int bias_dtype;
};

// ── host: clusters the device runs at once ──────────────────────────────────────────────────

constexpr int kSmemMost = 225 * 1024, kSmemHalf = 111 * 1024;   // dynamic bytes of one CTA, of two on an SM

// How many clusters of 1, 2, 4 and 8 CTAs are resident together with one or two CTAs an SM.  A cluster
// sits in one GPC, so the larger ones leave SMs over: 148, 74, 33 and 15 at one CTA an SM.
struct ClusterCaps {
    int one[4], two[4];
};
static __global__ void __launch_bounds__(384, 1) cluster_probe_kernel() {}
inline const ClusterCaps* cluster_caps(int* status) {
    static ClusterCaps caps[kMaxDevices];
    *status = once_per_device(reinterpret_cast<const void*>(caps), [](int device, void* c) {
        cudaError_t e = cudaFuncSetAttribute(cluster_probe_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
        for (int i = 0; i < 8 && e == cudaSuccess; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1024);
            cfg.blockDim = dim3(384);
            cfg.dynamicSmemBytes = i < 4 ? kSmemMost : kSmemHalf;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1u << (i & 3);
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, cluster_probe_kernel, &cfg);
            ClusterCaps& to = static_cast<ClusterCaps*>(c)[device];
            (i < 4 ? to.one : to.two)[i & 3] = n > 0 ? n : 1;
        }
        return e == cudaSuccess ? VY_OK : fail(VY_ERR_CUDA, "cluster occupancy: %s", cudaGetErrorString(e));
    }, caps);
    if (*status != VY_OK) return nullptr;
    const int dev = current_device();
    if (dev < 0) {
        *status = VY_ERR_CUDA;
        return nullptr;
    }
    return &caps[dev];
}

}  // namespace vy
