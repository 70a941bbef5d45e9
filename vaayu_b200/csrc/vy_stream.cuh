// vy_stream.cuh -- dense GEMM for few rows: out[T, N] = x[T, K] W[N, K]^T with T <= 128.
//
// The weights' bytes are the cost, so the kernel is a weight stream that happens to use the tensor
// core: 128 weight rows are the MMA's M (a gated product holds 128 gate and 128 up rows), the tokens
// its N, rounded up to 16.  Weight tiles arrive by TMA in a ring deep enough to keep about 100 KB in
// flight per CTA, two CTAs on an SM; HBM needs about 45 KB an SM in flight at its latency.
//
// K is split over the CTAs of a cluster: each accumulates its share in TMEM and writes the sums of
// every slice of the rows into the shared memory of the CTA that owns the slice; after one cluster
// barrier each CTA adds its slice over all shares, in rank order.  No workspace, no atomics, one
// order of summation, and no remote read to wait for.
//
// A kernel that is not the first of its call starts loading weights before the kernel in front of it
// has finished (they do not depend on it); its token tiles wait for it.
#pragma once

#include "vy_dense.cuh"

namespace vy {

constexpr int kStreamRows = 128;        // weight rows of a unit (of each matrix)
constexpr int kStreamMaxTokens = 128;
constexpr int kStreamThreads = 192;     // warps 0-3 read the sums, 4 loads, 5 issues the MMAs
constexpr int kStreamMaxStages = 12;
constexpr int kSmemMost = 226 * 1024, kSmemHalf = 112 * 1024;   // dynamic bytes of one CTA, of two on an SM

struct StreamParams {
    CUtensorMap w[2], x;
    int tokens, n, nk;      // rows of x; nk: K blocks of 128 bytes
    int cols;               // MMA N: tokens rounded up to 16
    int stages, tmem_cols;
    int sums_at;            // offset of the received sums in dynamic shared memory
    int early;              // weights may be loaded before the previous kernel has finished
    int parts;              // 2: x holds high parts, then low parts; an output is the sum of both
    EpiParams epi;
    int32_t* flags;
};

struct StreamBars {
    uint64_t full[kStreamMaxStages], empty[kStreamMaxStages], done;
    float token_scale[kStreamMaxTokens];
    uint32_t tmem_base;
    int abort_flag;
};

// One output value (weight row `row`, token `t`) from its sums.
// What an output needs besides its sums, fetched while they are still being formed.
struct ColumnScale {
    float a, b;      // int8: scale of the weight row, and of its up row or its bias
};
template <int EPI>
__device__ __forceinline__ ColumnScale column_scale(const StreamParams& p, int row) {
    ColumnScale c{0.f, 0.f};
    if constexpr (epi_is_i8(EPI)) {
        const EpiParams& e = p.epi;
        if (row < p.n) {
            c.a = e.col_scale[0][row];
            if constexpr (EPI == EPI_I8GATE)
                c.b = e.col_scale[1][row];
            else if (e.bias)
                c.b = load_as_float(e.bias, e.bias_dtype, row);
        }
    }
    return c;
}
template <int EPI, int ACT>
__device__ __forceinline__ void stream_put(const StreamParams& p, int row, int t, uint32_t s0, uint32_t s1,
                                           const ColumnScale& cs, const float* token_scale) {
    const EpiParams& e = p.epi;
    const int64_t at = int64_t(t) * e.ldo + row;
    if constexpr (EPI == EPI_GATE) {
        const float g = __uint_as_float(s0), u = __uint_as_float(s1);
        const float h = gate_act(g, e.act) * u;
        reinterpret_cast<uint16_t*>(e.out)[at] = static_cast<uint16_t>(act_bits<ACT>(h));
        if (e.part) reinterpret_cast<uint16_t*>(e.out)[at + e.part] = static_cast<uint16_t>(act_bits<ACT>(low_part<ACT>(h)));
        if (e.saved) {
            float* s = e.saved + saved_at(e.saved_bands, t, row);
            s[0] = g;
            s[kSavedBlock / 2] = u;
        }
    } else if constexpr (EPI == EPI_STORE) {
        reinterpret_cast<uint16_t*>(e.out)[at] = static_cast<uint16_t>(act_bits<ACT>(__uint_as_float(s0)));
    } else if constexpr (EPI == EPI_I8GATE) {
        const float g = __fmul_rn(__fmul_rn(float(int(s0)), token_scale[t]), cs.a);
        const float u = __fmul_rn(__fmul_rn(float(int(s1)), token_scale[t]), cs.b);
        reinterpret_cast<float*>(e.out)[at] = gate_act(g, e.act) * u;
    } else {
        float v = __fmul_rn(__fmul_rn(float(int(s0)), token_scale[t]), cs.a);
        if (e.bias) v = __fadd_rn(v, cs.b);
        store_as(e.out, e.out_dtype, at, v);
    }
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <int EPI, int ACT>
__global__ void __launch_bounds__(kStreamThreads) stream_kernel(const __grid_constant__ StreamParams p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    __shared__ StreamBars S;
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr bool I8 = epi_is_i8(EPI);
    constexpr int NW = epi_is_gate(EPI) ? 2 : 1;
    constexpr int kBlockK = I8 ? 128 : 64;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t splits;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(splits));
    const uint32_t rank = cluster_rank();
    const int unit = blockIdx.x / splits;
    const int row0 = unit * kStreamRows;
    const uint32_t x_bytes = uint32_t(p.cols) * 128u;
    const uint32_t stage_bytes = NW * 16384u + x_bytes;
    const int k_first = int(int64_t(p.nk) * rank / splits), k_last = int(int64_t(p.nk) * (rank + 1) / splits);
    const int nk = k_last - k_first;

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(&S.full[i], 1);
            mbar_init(&S.empty[i], 1);
        }
        mbar_init(&S.done, 1);
        S.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4 && lane == 0) {
        prefetch_map(&p.w[0]);
        if (NW == 2) prefetch_map(&p.w[1]);
        prefetch_map(&p.x);
    }
    if (warp == 0) tmem_alloc_n<0>(&S.tmem_base, p.tmem_cols);
    tc_fence_before();
    __syncthreads();
    // waited for before the first write into another CTA's shared memory: it has started by then
    if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    tc_fence_after();
    const uint32_t tmem = S.tmem_base;
    volatile int* abort_flag = &S.abort_flag;
    if (warp != 4) {
        grid_dependency_wait();
        grid_dependents_launch();
    }

    if (warp == 4) {
        auto load_w = [&](int i, uint32_t s) {
            const int k = (k_first + i) * kBlockK;
            unsigned char* at = ring + s * stage_bytes;
            mbar_expect_tx(&S.full[s], stage_bytes);
            tma_load_2d(at, &p.w[0], k, row0, &S.full[s]);
            if (NW == 2) tma_load_2d(at + 16384, &p.w[1], k, row0, &S.full[s]);
        };
        auto load_x = [&](int i, uint32_t s) {
            tma_load_2d(ring + s * stage_bytes + NW * 16384, &p.x, (k_first + i) * kBlockK, 0, &S.full[s]);
        };
        const int ahead = p.early ? min(p.stages, nk) : 0;
        if (elect_one())
            for (int i = 0; i < ahead; ++i) load_w(i, i);
        __syncwarp();
        grid_dependency_wait();
        grid_dependents_launch();
        if (elect_one())
            for (int i = 0; i < ahead; ++i) load_x(i, i);
        __syncwarp();
        int i = ahead, stage = ahead == p.stages ? 0 : ahead;
        uint32_t phase = ahead == p.stages ? 0 : 1;      // parity the ring's next pass waits for
        for (; i < nk; ++i) {
            if (!mbar_wait_warp(&S.empty[stage], phase, abort_flag, p.flags)) break;
            if (elect_one()) {
                load_w(i, stage);
                load_x(i, stage);
            }
            __syncwarp();
            if (++stage == p.stages) stage = 0, phase ^= 1;
        }
        // all loads have landed and been read before the ring is used again or the CTA leaves
        if (lane == 0)
            for (int j = max(0, i - p.stages); j < i; ++j) mbar_drain(&S.empty[j % p.stages], (j / p.stages) & 1, p.flags);
    } else if (warp == 5) {
        const uint32_t idesc = umma_idesc(I8, ACT == VY_BF16, 0, 0, kStreamRows, p.cols);
        const uint64_t first = umma_desc(smem_u32(ring), 16, 1024);
        uint32_t stage = 0, phase = 0;
        for (int i = 0; i < nk; ++i) {
            if (!mbar_wait_warp(&S.full[stage], phase, abort_flag, p.flags)) break;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t dw = first + (stage * stage_bytes >> 4), dx = dw + NW * 1024;
#pragma unroll
                for (int m = 0; m < NW; ++m)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_ss<I8, 0>(tmem + m * p.cols, dw + m * 1024 + 2 * k, dx + 2 * k, idesc, i != 0 || k != 0);
                mma_commit_one(&S.empty[stage]);
                if (i == nk - 1) mma_commit_one(&S.done);
            }
            __syncwarp();
            if (++stage == uint32_t(p.stages)) stage = 0, phase ^= 1;
        }
    }
    __syncwarp();

    // received sums [share][matrix][token][row of my slice], rows fastest
    const int rows = kStreamRows / splits;      // 1, 2, 4 or 8 shares
    uint32_t* sums = reinterpret_cast<uint32_t*>(ring + p.sums_at);
    // the weight row of this thread: its lane's when it reads all sums itself, else of my slice
    // (whole multiples of a slice's rows take part, so every output a thread adds has the same row)
    const int step = kStreamThreads / rows * rows;
    const bool direct = splits == 1 && p.parts == 1;      // nothing to join: outputs straight from TMEM
    const int my_row = row0 + (direct ? tid & (kStreamRows - 1) : int(rank) * rows + tid % rows);
    const ColumnScale cs = column_scale<EPI>(p, my_row);
    if constexpr (epi_is_i8(EPI)) {
        for (int t = tid; t < p.tokens; t += kStreamThreads) S.token_scale[t] = p.epi.row_scale[t];
        __syncthreads();
    }
    if (splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp < 4) {
        const bool ready = __all_sync(0xffffffffu, mbar_wait(&S.done, 0, abort_flag, p.flags));
        tc_fence_after();
        const uint32_t lanes = uint32_t(warp * 32) << 16;
        const int row = warp * 32 + lane;
        const uint32_t owner = map_to_rank(smem_u32(sums), row / rows) +
                               4u * (rank * NW * p.tokens * rows + row % rows);
        if (ready) {
            for (int c = 0; c < p.cols; c += 16) {
                uint32_t v[NW][16];
#pragma unroll
                for (int m = 0; m < NW; ++m) tmem_ld16(tmem + lanes + m * p.cols + c, v[m]);
#pragma unroll
                for (int m = 0; m < NW; ++m) tmem_wait16(v[m]);
                if (direct) {
                    if (row0 + row < p.n) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (c + j < p.tokens) stream_put<EPI, ACT>(p, row0 + row, c + j, v[0][j], v[NW - 1][j], cs,
                                                     S.token_scale);
                    }
                } else {
#pragma unroll
                    for (int m = 0; m < NW; ++m)
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (c + j < p.tokens) st_cluster(owner + 4u * ((m * p.tokens + c + j) * rows), v[m][j]);
                }
            }
        }
        tc_fence_before();
    }
    __syncwarp();
    if (!direct) {
        cluster_sync();
        const int share = NW * p.tokens * rows;
        for (int q = tid < step ? tid : rows * p.tokens; q < rows * (p.tokens / p.parts); q += step) {
            const int t = q / rows;
            if (my_row >= p.n) continue;
            uint32_t sum[NW];
#pragma unroll
            for (int m = 0; m < NW; ++m) {
                const uint32_t* at = sums + (m * p.tokens + t) * rows + q % rows;
                uint32_t acc = at[0];
                for (uint32_t r = 1; r < splits; ++r) {
                    const uint32_t v = at[r * share];
                    acc = I8 ? acc + v : __float_as_uint(__fadd_rn(__uint_as_float(acc), __uint_as_float(v)));
                }
                if (EPI == EPI_STORE && p.parts == 2) {
                    at += p.tokens / 2 * rows;
                    float low = __uint_as_float(at[0]);
                    for (uint32_t r = 1; r < splits; ++r) low = __fadd_rn(low, __uint_as_float(at[r * share]));
                    acc = __float_as_uint(__fadd_rn(__uint_as_float(acc), low));
                }
                sum[m] = acc;
            }
            stream_put<EPI, ACT>(p, my_row, t, sum[0], sum[NW - 1], cs, S.token_scale);
        }
    } else {
        __syncthreads();
    }
    tc_fence_after();
    if (warp == 0) tmem_free_n<0>(tmem, p.tmem_cols);
}

// ── host ────────────────────────────────────────────────────────────────────────────────────

// How a call is laid out on the machine: CTAs that share a unit's K, ring stages, shared memory.
struct StreamPlan {
    int splits, stages, sums, stage;
};
// The most shares (up to 8) whose CTAs are all resident at once: a second round would leave the
// memory system idle while its CTAs start and join.  Two CTAs run on an SM (and the next kernel's
// first ones start under this kernel's last) while ring and received sums take half its shared
// memory.  Up to 32 tokens two stages a CTA are enough for that (16 x 7168 x 2048, bf16: 27.5 us
// against 32.3 with one deep ring an SM); with more, the token tiles crowd the ring, and one CTA with
// five stages is faster than two with two (64 x 4096 x 14336: 82 us against 99).
inline StreamPlan stream_plan(int nw, int tokens, int parts, int n, int nk, int sm_count) {
    const int units = (n + kStreamRows - 1) / kStreamRows;
    StreamPlan p{};
    p.stage = nw * 16384 + (tokens + 15) / 16 * 16 * 128;
    for (p.splits = 8; p.splits >= 1; p.splits /= 2) {
        p.sums = p.splits > 1 || parts > 1 ? (nw * tokens * kStreamRows * 4 + 1023) / 1024 * 1024 : 0;
        const int half = (kSmemHalf - 1024 - p.sums) / p.stage, whole = (kSmemMost - 1024 - p.sums) / p.stage;
        const bool two = half >= (tokens <= 32 ? 2 : 3);
        p.stages = two ? half : whole;
        if (p.splits == 1) break;
        if (p.stages >= 2 && nk >= 2 * p.splits && units * p.splits <= (two ? 2 : 1) * sm_count) break;
    }
    if (p.stages > kStreamMaxStages) p.stages = kStreamMaxStages;
    return p;
}

// w: NW weight matrices [n, k], contiguous; x: [tokens, k] (parts == 2: high parts, then low parts).
template <int EPI, int ACT>
int stream_launch(const void* w0, const void* w1, const void* x, int64_t x_ld, int tokens, int parts, int n, int k,
                  bool early, const EpiParams& epi, int32_t* flags, const DeviceInfo* dev, cudaStream_t s) {
    constexpr bool I8 = epi_is_i8(EPI);
    constexpr int NW = epi_is_gate(EPI) ? 2 : 1;
    constexpr int block = I8 ? 128 : 64;
    const int dtype = I8 ? VY_E4M3 : ACT;
    StreamParams p{};
    p.tokens = tokens;
    p.n = n;
    p.nk = (k + block - 1) / block;
    p.cols = (tokens + 15) / 16 * 16;
    p.early = early;
    p.parts = parts;
    p.epi = epi;
    p.flags = flags;
    p.tmem_cols = 32;
    while (p.tmem_cols < NW * p.cols) p.tmem_cols *= 2;
    int st;
    if ((st = make_map_2d(&p.w[0], dtype, w0, n, k, k, block, kStreamRows)) != VY_OK) return st;
    if (NW == 2 && (st = make_map_2d(&p.w[1], dtype, w1, n, k, k, block, kStreamRows)) != VY_OK) return st;
    if ((st = make_map_2d(&p.x, dtype, x, tokens, k, x_ld, block, p.cols)) != VY_OK) return st;
    const StreamPlan plan = stream_plan(NW, tokens, parts, n, p.nk, dev->sm_count);
    if (plan.stages < 2) return fail(VY_ERR_UNSUPPORTED, "dense stream: %d tokens", tokens);
    p.stages = plan.stages;
    p.sums_at = plan.stages * plan.stage;
    const int bytes = p.sums_at + plan.sums + 1024;
    auto kern = stream_kernel<EPI, ACT>;
    st = once_per_device(reinterpret_cast<const void*>(kern), [](int, void* f) {
        const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
        return e == cudaSuccess ? VY_OK : fail(VY_ERR_CUDA, "dense stream shared memory: %s", cudaGetErrorString(e));
    }, reinterpret_cast<void*>(kern));
    if (st != VY_OK) return st;
    const unsigned units = (n + kStreamRows - 1) / kStreamRows;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(units * plan.splits);
    cfg.blockDim = dim3(kStreamThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = plan.splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return fail(VY_ERR_CUDA, "dense stream launch: %s", cudaGetErrorString(e));
    return VY_OK;
}

}  // namespace vy
