// vy_stream.cuh -- dense GEMM for few rows: out[T, N] = x[T, K] W[N, K]^T.
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
// The backward products read the same weights across their rows: there the weight tile is MN-major
// ([K, N] in memory), and d_x takes its K from two tensor pairs (dg with Wg, du with Wu).
//
// With up to 16 tokens the int8 block needs no quantisation kernels (Source): the four warps that read
// the sums at the end are idle until then and write the token tile's codes themselves, a 16-value
// piece of a token each per K block, from rows that are still floats.  The rows' largest magnitudes
// come from the kernel in front, whose every CTA leaves the maximum of the columns it wrote (no
// global atomics, nothing to clear), or, while all rows together are at most 16384 values (one or two
// tokens of a wide layer, 16 of a small one), are taken over the whole rows in every CTA.
//
// A kernel that is not the first of its call starts loading weights before the kernel in front of it
// has finished (they do not depend on it); its token tiles wait for it.
#pragma once

#include "vy_dense.cuh"
#include "vy_quant.cuh"

namespace vy {

constexpr int kStreamRows = 128;        // weight rows of a unit (of each matrix)
// Up to here a product streams its weights; above, the pairs of vy_tile.cuh take it.  Device time in a
// captured chain, us, stream : pairs.
//   plain, int8            96 tokens    128        160
//     4096 -> 4096         10 : 15      12 : 15    14 : 15   (192 tokens: 15 : 15)
//     14336 -> 4096                     19 : 27    22 : 27
//     4096 -> 14336        22 : 18      24 : 19    27 : 19   (112 units leave no K shares: no rule yet)
//   whole bf16 block       64 tokens    96         128 (in brackets what runs: gate on pairs, down streamed)
//     2048 x 2048          17 : 28      23 : 28    27 : 29 (25)
//     7168 x 2048          31 : 43      46 : 43    51 : 44 (46)
//     4096 x 14336         72 : 96      78 : 96    86 : 97 (81)
constexpr int kStreamMaxGate = 96, kStreamMaxPlain = 160;
constexpr int kStreamThreads = 192;     // warps 0-3 read the sums, 4 loads, 5 issues the MMAs
constexpr int kStreamMaxStages = 12;
// Weight bytes a CTA asks for in L2 before it waits for the kernel in front, behind what its ring holds
// (37 x 7168 -> 2048, int8: 7.4 -> 6.9 us; more of it takes bandwidth from the kernel in front).
constexpr int kStreamFetch = 64 * 1024;

// Where the token tile comes from.
enum Source {
    SRC_TMA = 0,      // [tokens, K] in the weights' type
    SRC_ROWS = 1,     // int8 codes made here from 16-bit rows, whose maxima are taken here
    SRC_HIDDEN = 2    // int8 codes made here from fp32 rows, whose maxima the previous kernel left
};
constexpr int kSourceTokens = 16;      // 8 pieces of a K block each, one per thread of four warps

struct StreamParams {
    CUtensorMap w[2], x[2]; // of a gated product gate and up, else of the K segments
    int tokens, n, nk;      // rows of x; nk: K blocks of 128 bytes
    int segment;            // K blocks of the first segment (nk when there is one)
    int cols;               // MMA N: tokens rounded up to 16
    int stages, tmem_cols;
    int sums_at;            // offset of the received sums in dynamic shared memory
    int early;              // weights may be loaded before the previous kernel has finished
    int parts;              // 2: x holds high parts, then low parts; an output is the sum of both
    EpiParams epi;
    int32_t* flags;
    const void* rows;       // SRC_ROWS, SRC_HIDDEN: [tokens, k], row stride, K in elements
    int64_t rows_ld;
    int k;
    uint32_t* maxima;       // EPI_I8GATE: this kernel's, [CTA][token]; SRC_HIDDEN: the previous one's
    int n_maxima;           // CTAs in it (0: none wanted)
};

struct StreamBars {
    uint64_t full[kStreamMaxStages], empty[kStreamMaxStages], done;
    float token_scale[kStreamMaxPlain];
    uint32_t token_top[kSourceTokens], part_top[4][kSourceTokens];
    uint32_t tmem_base;
    int abort_flag;
};

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
// One output value (weight row `row`, token `t`) from its sums.
template <int EPI, int ACT>
__device__ __forceinline__ void stream_put(const StreamParams& p, int row, int t, uint32_t s0, uint32_t s1,
                                           const ColumnScale& cs, const float* token_scale, uint32_t* token_top) {
    const EpiParams& e = p.epi;
    const int64_t at = int64_t(t) * e.ldo + row;
    if constexpr (EPI == EPI_DGATE) {
        const float dh = __uint_as_float(s0);
        const float* s = e.saved + saved_at(e.saved_bands, t, row);
        const float g = s[0], u = s[kSavedBlock / 2];
        const float2 a = gate_act_grad(g, e.act);
        const float v[3] = {dh * u * a.y, dh * a.x, a.x * u};
        uint16_t* const to[3] = {e.dg, e.du, e.h};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            to[i][at] = static_cast<uint16_t>(act_bits<ACT>(v[i]));
            if (e.part) to[i][at + e.part] = static_cast<uint16_t>(act_bits<ACT>(low_part<ACT>(v[i])));
        }
    } else if constexpr (EPI == EPI_GATE) {
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
        const float h = gate_act(g, e.act) * u;
        reinterpret_cast<float*>(e.out)[at] = h;
        if (p.n_maxima) atomicMax(token_top + t, __float_as_uint(h) & 0x7FFFFFFFu);
    } else {
        float v = __fmul_rn(__fmul_rn(float(int(s0)), token_scale[t]), cs.a);
        if (e.bias) v = __fadd_rn(v, cs.b);
        store_as(e.out, e.out_dtype, at, v);
    }
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// A piece of 16 values of a row that starts on a 16-byte boundary.
template <int SRC, int ACT>
struct RowPiece {
    static constexpr int DT = SRC == SRC_HIDDEN ? VY_F32 : ACT;
    static constexpr int V = DT == VY_F32 ? 4 : 2;      // 16-byte loads
    uint4 u[V];
    __device__ __forceinline__ void load(const void* rows, int64_t at, bool in) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(rows) + at * (DT == VY_F32 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = in ? ld_piece(p + i) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ uint4 codes(const RowScale& r) const {
        using P = Piece<DT>;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float v[P::N];
            uint32_t o[P::N / 4];
            P::values(u[i], v);
            quant_words<P::N>(v, r, o);
#pragma unroll
            for (int j = 0; j < P::N / 4; ++j) w[i * (P::N / 4) + j] = o[j];
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <int EPI, int ACT, int SRC, bool MN>
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
    constexpr bool kOwnCodes = SRC != SRC_TMA;
    const int k_first = int(int64_t(p.nk) * rank / splits), k_last = int(int64_t(p.nk) * (rank + 1) / splits);
    const int nk = k_last - k_first;

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(&S.full[i], kOwnCodes ? 5 : 1);      // the loads, and the four code-writing warps
            mbar_init(&S.empty[i], 1);
        }
        mbar_init(&S.done, 1);
        S.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4 && lane == 0) {
        prefetch_map(&p.w[0]);
        if (NW == 2 || p.segment < p.nk) prefetch_map(&p.w[1]);
        if (!kOwnCodes) prefetch_map(&p.x[0]);
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

    if (kOwnCodes && warp < 4) {
        // thread: token tid / 8, piece tid % 8 of each K block
        const int t = tid >> 3, c = tid & 7;
        uint32_t top = 0;
        if constexpr (SRC == SRC_HIDDEN) {
            if (t < p.tokens)
                for (int i = c; i < p.n_maxima; i += 8) top = max(top, p.maxima[i * p.tokens + t]);
#pragma unroll
            for (int d = 1; d < 8; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
        } else if constexpr (SRC == SRC_ROWS) {
            using P = Piece<ACT>;
            for (int r = 0; r < p.tokens; ++r) {
                const uint4* row = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.rows) + r * p.rows_ld);
                uint32_t m = 0;
#pragma unroll 4
                for (int i = tid; i < p.k / 8; i += 128) m = P::top(m, ld_piece(row + i));
                m = __reduce_max_sync(0xffffffffu, P::wide(m));
                if (lane == 0) S.part_top[warp][r] = m;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (t < p.tokens)
                for (int w = 0; w < 4; ++w) top = max(top, S.part_top[w][t]);
        }
        const RowScale scale = row_scale(top);
        if (c == 0 && t < p.tokens) S.token_scale[t] = scale.s;
        RowPiece<SRC, ACT> piece;
        const int64_t at = t * p.rows_ld + int64_t(k_first) * kBlockK + c * 16;
        const int left = p.k - k_first * kBlockK - c * 16;      // values from my first piece to the row's end
        piece.load(p.rows, at, t < p.tokens && left > 0);
        int stage = 0;
        uint32_t phase = 1;
        for (int i = 0; i < nk; ++i) {
            const uint4 codes = piece.codes(scale);
            if (i + 1 < nk) piece.load(p.rows, at + (i + 1) * kBlockK, t < p.tokens && left > (i + 1) * kBlockK);
            if (!mbar_wait_warp(&S.empty[stage], phase, abort_flag, p.flags)) break;
            // rows of padding tokens keep what the ring holds: their sums are not used
            if (t < p.tokens)
                *reinterpret_cast<uint4*>(ring + stage * stage_bytes + NW * 16384 + t * 128 + ((c ^ (t & 7)) << 4)) = codes;
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&S.full[stage]);
            if (++stage == p.stages) stage = 0, phase ^= 1;
        }
    }
    if (warp == 4) {
        auto load_w = [&](int i, uint32_t s) {
            unsigned char* at = ring + s * stage_bytes;
            mbar_expect_tx(&S.full[s], kOwnCodes ? NW * 16384u : stage_bytes);
            if constexpr (MN) {
                const int kb = k_first + i, seg = kb >= p.segment, k = (kb - (seg ? p.segment : 0)) * kBlockK;
                tma_load_2d(at, &p.w[seg], row0, k, &S.full[s]);
                tma_load_2d(at + 8192, &p.w[seg], row0 + 64, k, &S.full[s]);
            } else {
                const int k = (k_first + i) * kBlockK;
                tma_load_2d(at, &p.w[0], k, row0, &S.full[s]);
                if (NW == 2) tma_load_2d(at + 16384, &p.w[1], k, row0, &S.full[s]);
            }
        };
        auto load_x = [&](int i, uint32_t s) {
            const int kb = k_first + i, seg = MN && kb >= p.segment;
            if (!kOwnCodes)
                tma_load_2d(ring + s * stage_bytes + NW * 16384, &p.x[seg], (kb - (seg ? p.segment : 0)) * kBlockK, 0,
                            &S.full[s]);
        };
        const int ahead = p.early ? min(p.stages, nk) : 0;
        if (elect_one()) {
            for (int i = 0; i < ahead; ++i) load_w(i, i);
            const int fetch = min(nk, ahead + kStreamFetch / (NW * 16384));
            for (int i = ahead; i < fetch && !MN; ++i)
                for (int m = 0; m < NW; ++m) tma_prefetch_2d(&p.w[m], (k_first + i) * kBlockK, row0);
        }
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
        const uint32_t idesc = umma_idesc(I8, ACT == VY_BF16, MN, 0, kStreamRows, p.cols);
        const uint64_t first = umma_desc(smem_u32(ring), MN ? 8192 : 16, 1024);
        const uint64_t first_x = umma_desc(smem_u32(ring), 16, 1024) + NW * 1024;
        constexpr uint32_t w_step = MN ? 128 : 2;      // one MMA's K: 16 rows of 128 bytes, or 32 bytes of a row
        uint32_t stage = 0, phase = 0;
        for (int i = 0; i < nk; ++i) {
            if (!mbar_wait_warp(&S.full[stage], phase, abort_flag, p.flags)) break;
            tc_fence_after();
            if (elect_one()) {
                const uint64_t dw = first + (stage * stage_bytes >> 4), dx = first_x + (stage * stage_bytes >> 4);
#pragma unroll
                for (int m = 0; m < NW; ++m)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_ss<I8, 0>(tmem + m * p.cols, dw + m * 1024 + w_step * k, dx + 2 * k, idesc, i != 0 || k != 0);
                mma_commit_one(&S.empty[stage]);
                if (i == nk - 1) mma_commit_one(&S.done);
            }
            __syncwarp();
            if (++stage == uint32_t(p.stages)) stage = 0, phase ^= 1;
        }
    }
    __syncwarp();

    // received sums [share][matrix][token][row of my slice], rows fastest
    const int row_bits = 7 - (31 - __clz(splits)), rows = 1 << row_bits;      // 1, 2, 4 or 8 shares of 128 rows
    uint32_t* sums = reinterpret_cast<uint32_t*>(ring + p.sums_at);
    // the weight row of this thread: its lane's when it reads all sums itself, else of my slice
    // (whole multiples of a slice's rows take part, so every output a thread adds has the same row)
    const int step = rows == kStreamRows ? kStreamRows : kStreamThreads;
    const bool direct = splits == 1 && p.parts == 1;      // nothing to join: outputs straight from TMEM
    const int my_row = row0 + (direct ? tid & (kStreamRows - 1) : int(rank) * rows + (tid & (rows - 1)));
    const ColumnScale cs = column_scale<EPI>(p, my_row);
    if constexpr (epi_is_i8(EPI)) {
        if (!kOwnCodes)
            for (int t = tid; t < p.tokens; t += kStreamThreads) S.token_scale[t] = p.epi.row_scale[t];
        if (tid < kSourceTokens) S.token_top[tid] = 0;
        __syncthreads();
    }
    if (splits > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (warp < 4) {
        const bool ready = __all_sync(0xffffffffu, mbar_wait(&S.done, 0, abort_flag, p.flags));
        tc_fence_after();
        const uint32_t lanes = uint32_t(warp * 32) << 16;
        const int row = warp * 32 + lane;
        const uint32_t owner = map_to_rank(smem_u32(sums), row >> row_bits) +
                               4u * (rank * NW * p.tokens * rows + (row & (rows - 1)));
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
                                                     S.token_scale, S.token_top);
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
        const int share = NW * p.tokens * rows, count = p.parts == 2 ? p.tokens / 2 * rows : p.tokens * rows;
        // all shares of a sum are fetched before the first is added
        auto joined = [&](const uint32_t* at) {
            uint32_t v[8];
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r)
                if (r < splits) v[r] = at[r * share];
            uint32_t acc = v[0];
#pragma unroll
            for (uint32_t r = 1; r < 8; ++r)
                if (r < splits)
                    acc = I8 ? acc + v[r] : __float_as_uint(__fadd_rn(__uint_as_float(acc), __uint_as_float(v[r])));
            return acc;
        };
        for (int q = tid; q < count && tid < step && my_row < p.n; q += step) {
            const int t = q >> row_bits;
            const uint32_t* at = sums + q;
            uint32_t sum[NW];
            sum[0] = joined(at);
            if (NW == 2) sum[NW - 1] = joined(at + p.tokens * rows);
            if (EPI == EPI_STORE && p.parts == 2)
                sum[0] = __float_as_uint(__fadd_rn(__uint_as_float(sum[0]), __uint_as_float(joined(at + count))));
            stream_put<EPI, ACT>(p, my_row, t, sum[0], sum[NW - 1], cs, S.token_scale, S.token_top);
        }
    } else {
        __syncthreads();
    }
    if constexpr (EPI == EPI_I8GATE) {
        if (p.n_maxima) {
            __syncthreads();
            if (tid < p.tokens) p.maxima[int64_t(blockIdx.x) * p.tokens + tid] = S.token_top[tid];
        }
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
// memory.  Up to 32 tokens two stages a CTA are enough for that; with more, the token tiles crowd the
// ring, and one CTA with five stages is faster than two with two.  Half ring against whole, us (the
// whole one may also leave fewer K shares, since fewer clusters are resident):
//   bf16 block  1 x 4096 x 14336 57.8 : 61.5   16 x 7168 x 2048 25.2 : 26.6   64 x 4096 x 14336 85.0 : 71.9
//   int8 block  16 x 7168 x 2048 20.5 : 22.9   8 x 4096 x 14336 42.8 : 48.2
//   int8        37 x 7168 -> 2048 7.1 : 8.3    64 x 4096 -> 14336 18.4 : 16.4   128 x 4096 -> 14336 23.7 : 20.2
// (The last two have 112 CTAs for 148 SMs, where the half ring with its three stages is not the better
// one; the rule does not tell them apart yet.)
inline StreamPlan stream_plan(int nw, int tokens, int parts, int n, int nk, const ClusterCaps& caps) {
    const int units = (n + kStreamRows - 1) / kStreamRows;
    StreamPlan p{};
    p.stage = nw * 16384 + (tokens + 15) / 16 * 16 * 128;
    for (int i = 3; i >= 0; --i) {
        p.splits = 1 << i;
        p.sums = p.splits > 1 || parts > 1 ? (nw * tokens * kStreamRows * 4 + 1023) / 1024 * 1024 : 0;
        const int half = (kSmemHalf - 1024 - p.sums) / p.stage, whole = (kSmemMost - 1024 - p.sums) / p.stage;
        const bool two = half >= (tokens <= 32 ? 2 : 3);
        p.stages = two ? half : whole;
        if (p.splits == 1) break;
        if (p.stages >= 2 && nk >= 2 * p.splits && units <= (two ? caps.two : caps.one)[i]) break;
    }
    if (p.stages > kStreamMaxStages) p.stages = kStreamMaxStages;
    return p;
}

// One product: its weight matrices [n, k] (contiguous) and its token rows.
struct StreamCall {
    const void *w0, *w1;      // w1: the up matrix of a gated product, or (MN) the second K segment's, or null
    const void* x;            // [tokens, k]; parts == 2: high parts, then low parts of tokens / 2 rows
    int64_t x_ld;
    int tokens, parts, n, k;
    bool early;               // a kernel of the same call runs in front of this one
    uint32_t* maxima;         // see StreamParams
    int n_maxima;
    const void* x1;           // (MN) the second K segment's tokens
};

// CTAs of a product's launch.
inline int stream_ctas(int nw, int tokens, int parts, int n, int nk, const ClusterCaps& caps) {
    return (n + kStreamRows - 1) / kStreamRows * stream_plan(nw, tokens, parts, n, nk, caps).splits;
}

// MN: the weights are [k, n] in memory; k is that of one segment.
template <int EPI, int ACT, int SRC = SRC_TMA, bool MN = false>
int stream_launch(const StreamCall& a, const EpiParams& epi, int32_t* flags, const ClusterCaps& caps, cudaStream_t s) {
    constexpr bool I8 = epi_is_i8(EPI);
    constexpr int NW = epi_is_gate(EPI) ? 2 : 1;
    constexpr int block = I8 ? 128 : 64;
    const int dtype = I8 ? VY_E4M3 : ACT;
    StreamParams p{};
    p.tokens = a.tokens;
    p.n = a.n;
    p.segment = (a.k + block - 1) / block;
    p.nk = MN && a.w1 ? 2 * p.segment : p.segment;
    p.cols = (a.tokens + 15) / 16 * 16;
    p.early = a.early;
    p.parts = a.parts;
    p.epi = epi;
    p.flags = flags;
    p.maxima = a.maxima;
    p.n_maxima = a.n_maxima;
    p.tmem_cols = 32;
    while (p.tmem_cols < NW * p.cols) p.tmem_cols *= 2;
    int st;
    const void* const w[2] = {a.w0, a.w1};
    for (int i = 0; i < 2 && w[i]; ++i) {
        st = MN ? make_map_2d(&p.w[i], dtype, w[i], a.k, a.n, a.n, 64, 64)
                : make_map_2d(&p.w[i], dtype, w[i], a.n, a.k, a.k, block, kStreamRows);
        if (st != VY_OK) return st;
    }
    if (SRC == SRC_TMA) {
        if ((st = make_map_2d(&p.x[0], dtype, a.x, a.tokens, a.k, a.x_ld, block, p.cols)) != VY_OK) return st;
        if (a.x1 && (st = make_map_2d(&p.x[1], dtype, a.x1, a.tokens, a.k, a.x_ld, block, p.cols)) != VY_OK) return st;
    } else {
        p.rows = a.x;
        p.rows_ld = a.x_ld;
        p.k = a.k;
    }
    const StreamPlan plan = stream_plan(NW, a.tokens, a.parts, a.n, p.nk, caps);
    if (plan.stages < 2) return fail(VY_ERR_UNSUPPORTED, "dense stream: %d tokens", a.tokens);
    p.stages = plan.stages;
    p.sums_at = plan.stages * plan.stage;
    const int bytes = p.sums_at + plan.sums + 1024;
    auto kern = stream_kernel<EPI, ACT, SRC, MN>;
    st = once_per_device(reinterpret_cast<const void*>(kern), [](int, void* f) {
        const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
        return e == cudaSuccess ? VY_OK : fail(VY_ERR_CUDA, "dense stream shared memory: %s", cudaGetErrorString(e));
    }, reinterpret_cast<void*>(kern));
    if (st != VY_OK) return st;
    const unsigned units = (a.n + kStreamRows - 1) / kStreamRows;
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
