// vy_tile.cuh -- dense GEMM on CTA pairs: out[M, N] = A[M, K] B[N, K]^T for many rows.
//
// A pair of CTAs computes a 256 x bn tile (bn = 256 or 128) with tcgen05.mma.cta_group::2: each
// CTA holds 128 rows of A and half of B's rows in shared memory, so an operand byte is read from
// L2 once for twice the work of one CTA's tile (a 128 x 256 tile on its own would ask L2 for about
// 96 bytes a clock and SM, the pair for 64).  K advances in blocks of 128 bytes (64 16-bit
// elements or 128 int8) through a ring of TMA-filled stages; accumulators are double-buffered in
// TMEM, so the epilogue of one tile runs under the MMAs of the next.  Both operands may be K-major
// or MN-major (the weight gradients contract over tokens, the activations' slow axis), and K may
// come in segments from several tensors (dx = dg Wg + du Wu).  One launch takes up to four
// GEMMs, whose tiles fill the machine together.
//
// Few tiles.  Pairs are persistent, one for two SMs, and take tiles in turn.  A launch whose tiles can
// each have a resident cluster of 2 or 4 pairs (33 and 15 such clusters), and whose K leaves a pair
// kShareLeast blocks or more, instead gives each tile such a cluster, which splits its K: every
// pair sends each other pair the sums of the columns that one owns, into shared memory, and adds its
// own columns over all shares in K order.  (Joining through global memory, the last of the pairs adding
// all shares, measured 59 us where this takes 21 and no split 27: 1003 x 2048 x 768 forward.)
//
// Roles of a CTA (12 warps): warp 0 loads, warp 1 of the pair's first CTA issues the MMAs, warp 2
// owns TMEM, warps 4-11 run the epilogue.  Every wait is bounded: on a timeout the CTA records the
// error, leaves its loop, and the pair still meets at its final barrier.
#pragma once

#include "vy_dense.cuh"

namespace vy {

constexpr int kTileThreads = 384;
constexpr int kTileProblems = 4;
constexpr int kHalfBytes = 128 * 128;          // one operand's share of a stage: 128 rows x 128 bytes
constexpr uint32_t kTileTmemCols = 512;

struct TileProblem {
    CUtensorMap out;             // EPI_STORE: the output in 32 x 64 tiles
    CUtensorMap a[2], b[2];      // operands of the K segments (a gated product: b is gate, up)
    int m, n;                    // rows, output columns
    int nk[2];                   // K blocks of each segment
    uint8_t a_of[2], b_of[2];    // each segment's operands
    int a_mn, b_mn;              // 1: that operand is MN-major (memory [K, M] / [K, N])
    int bn;                      // tile columns, 256 or 128
    int m_tiles, n_tiles, first; // tiles [first, first + m_tiles * n_tiles)
    EpiParams epi;
};

struct TileParams {
    TileProblem prob[kTileProblems];
    int n_problems, n_tiles;
    int splits;              // pairs of a cluster, which share a tile's K: 1, 2 or 4
    int n_long, extra;       // see TileTurn
    int32_t* flags;
};

// A plain product's epilogue needs 32 KB to lay its rows out for TMA stores; the others store directly.
template <int EPI>
struct __align__(1024) TileSmem {
    static constexpr int kTileStages = EPI == EPI_STORE ? 5 : 6;
    unsigned char a[kTileStages][kHalfBytes];
    unsigned char b[kTileStages][kHalfBytes];
    unsigned char rows[EPI == EPI_STORE ? 8 : 1][EPI == EPI_STORE ? 4096 : 16];
    uint64_t full[kTileStages], empty[kTileStages];
    uint64_t acc_full[2], acc_empty[2];
    float cols[8][2][128];       // int8: an epilogue warp's column scales (gate, up) or scale and bias
    uint32_t tmem_base;
    int abort_flag;
};

__host__ __device__ __forceinline__ int k_total(const TileProblem& q) { return q.nk[0] + q.nk[1]; }

// A pair's tiles: first, first + pairs, ...  When the first problem's tiles are long ones (dx: its K is
// both halves' channels), they come first, n_long of them, and the pairs that get one fewer of them
// take `extra` of the others each before all go on in turn.
__device__ __forceinline__ int tile_of_turn(const TileParams& p, int turn, int pair, int pairs) {
    if (p.extra == 0) return pair + turn * pairs;
    const int odd = p.n_long % pairs, rounds = p.n_long / pairs + (pair < odd);      // my long tiles
    if (turn < rounds) return pair + turn * pairs;
    turn -= rounds;
    const int light = pairs - odd;
    if (pair >= odd) {
        if (turn < p.extra) return p.n_long + turn * light + pair - odd;
        turn -= p.extra;
    }
    return p.n_long + p.extra * light + turn * pairs + pair;
}
struct TileAt {
    int prob, m, n;   // tile's problem, row tile, column tile
};
// Bands of 8 row tiles, row tiles fastest inside a band: the tiles in flight share few operand rows.
__device__ __forceinline__ TileAt tile_at(const TileParams& p, int tile) {
    TileAt t;
    t.prob = 0;
    while (t.prob + 1 < p.n_problems && tile >= p.prob[t.prob + 1].first) ++t.prob;
    const TileProblem& q = p.prob[t.prob];
    const int r = tile - q.first, band = r / (8 * q.n_tiles);
    const int rows = min(8, q.m_tiles - band * 8), in = r - band * 8 * q.n_tiles;
    t.m = band * 8 + in % rows;
    t.n = in / rows;
    return t;
}

// Sums of 16 columns of a tile: from TMEM, or (splits > 1) all shares of my columns, received in
// shared memory as [share][4 columns][row][4], added in K order.
struct TileSums {
    uint32_t tmem;
    const float4* recv;      // at my row
    int splits, first, own;  // my columns [first, first + own) of each matrix
    int mats, width;         // matrices of a tile (2: gate and up) and columns of each
    template <bool I8>
    __device__ __forceinline__ void get(int mat, int c, uint32_t (&r)[16]) const {
        if (splits == 1) {
            tmem_ld16(tmem + mat * width + c, r);
            tmem_wait16(r);
            return;
        }
        const float4* s = recv + (mat * own + c - first) / 4 * 128;
        for (int i = 0; i < splits; ++i, s += mats * own / 4 * 128) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 f = s[q * 128];
                const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t& d = r[4 * q + j];
                    const uint32_t u = __float_as_uint(v[j]);
                    d = i == 0 ? u : I8 ? d + u : __float_as_uint(__fadd_rn(__uint_as_float(d), __uint_as_float(u)));
                }
            }
        }
    }
    // Sends my share of the tile (half of its columns a warp) to the pairs that own the columns.
    __device__ __forceinline__ void send(uint32_t recv_base, uint32_t rank, int share, int half) const {
        const int cols = mats * width;
        for (int c = half * (cols / 2); c < (half + 1) * (cols / 2); c += 16) {
            uint32_t r[16];
            tmem_ld16(tmem + c, r);
            tmem_wait16(r);
            const int mat = c / width, in = c % width, owner = in / own;
            const int local = (share * mats + mat) * own + in % own;
            const uint32_t to = map_to_rank(recv_base, owner * 2 + rank) + local / 4 * 2048;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + q * 2048), "r"(r[4 * q]),
                             "r"(r[4 * q + 1]), "r"(r[4 * q + 2]), "r"(r[4 * q + 3])
                             : "memory");
        }
    }
};

// The scales (and bias) of a warp's columns [c0, c1) of a tile, fetched while the sums are still being
// formed; a column at a time beside its sums costs a memory latency per 16 columns (1.1 us each).
template <int EPI>
__device__ __forceinline__ void load_cols(float (&cols)[2][128], const TileProblem& q, int n_tile, int c0, int c1) {
    if constexpr (epi_is_i8(EPI)) {
        const EpiParams& e = q.epi;
        const int width = epi_is_gate(EPI) ? q.bn / 2 : q.bn, first = n_tile * width + c0;
        __syncwarp();
        for (int i = threadIdx.x & 31; i < c1 - c0; i += 32) {
            const int c = min(first + i, q.n - 1);
            cols[0][i] = e.col_scale[0][c];
            if constexpr (EPI == EPI_I8GATE)
                cols[1][i] = e.col_scale[1][c];
            else if (e.bias)
                cols[1][i] = load_as_float(e.bias, e.bias_dtype, c);
        }
        __syncwarp();
    }
}

template <int EPI, int ACT>
__device__ __forceinline__ void tile_epilogue(const TileProblem& q, int row, int n_tile, const TileSums& sums, int c0,
                                              int c1, float rs, const float (&cols)[2][128]) {
    const EpiParams& e = q.epi;
    const bool live = row < q.m;
    if constexpr (epi_is_gate(EPI)) {
        const int width = q.bn / 2;                  // output columns of the tile
        for (int c = c0; c < c1; c += 16) {
            uint32_t g[16], u[16];
            sums.get<epi_is_i8(EPI)>(0, c, g);
            sums.get<epi_is_i8(EPI)>(1, c, u);
            const int col = n_tile * width + c;
            const int valid = min(16, q.n - col);
            if (!live || valid <= 0) continue;
            float h[16];
            if constexpr (EPI == EPI_I8GATE) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float gf = __fmul_rn(__fmul_rn(float(int(g[j])), rs), cols[0][c - c0 + j]);
                    const float uf = __fmul_rn(__fmul_rn(float(int(u[j])), rs), cols[1][c - c0 + j]);
                    h[j] = gate_act(gf, e.act) * uf;
                }
                store16_dyn(e.out, VY_F32, int64_t(row) * e.ldo + col, h, valid, true);
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) h[j] = gate_act(__uint_as_float(g[j]), e.act) * __uint_as_float(u[j]);
                if (e.saved) {
                    float4* s = reinterpret_cast<float4*>(e.saved + saved_at(e.saved_bands, row, col));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[j * 32] = make_float4(__uint_as_float(g[4 * j]), __uint_as_float(g[4 * j + 1]),
                                                __uint_as_float(g[4 * j + 2]), __uint_as_float(g[4 * j + 3]));
                        s[128 + j * 32] = make_float4(__uint_as_float(u[4 * j]), __uint_as_float(u[4 * j + 1]),
                                                      __uint_as_float(u[4 * j + 2]), __uint_as_float(u[4 * j + 3]));
                    }
                }
                store16<ACT>(reinterpret_cast<uint16_t*>(e.out) + int64_t(row) * e.ldo + col, h, valid);
            }
        }
    } else {
        for (int c = c0; c < c1; c += 16) {
            uint32_t r[16];
            sums.get<epi_is_i8(EPI)>(0, c, r);
            const int col = n_tile * q.bn + c;
            const int valid = min(16, q.n - col);
            if (!live || valid <= 0) continue;
            float v[16];
            if constexpr (EPI == EPI_I8) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    v[j] = __fmul_rn(__fmul_rn(float(int(r[j])), rs), cols[0][c - c0 + j]);
                    if (e.bias) v[j] = __fadd_rn(v[j], cols[1][c - c0 + j]);
                }
                store16_dyn(e.out, e.out_dtype, int64_t(row) * e.ldo + col, v, valid, e.vec != 0);
            } else if constexpr (EPI == EPI_STORE) {
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                store16<ACT>(reinterpret_cast<uint16_t*>(e.out) + int64_t(row) * e.ldo + col, v, valid);
            }
        }
    }
}

// dg, du and h of a tile from its dh and the saved g and u.  The tile's g and u are read a chunk of 16
// columns ahead, the first one before the tile's sums are awaited: their latency is paid under the
// MMAs and the previous chunk's arithmetic.
struct GateChunk {
    float4 g[4], u[4];
};
__device__ __forceinline__ void load_gate(GateChunk& k, const EpiParams& e, int row, int col, bool live, int n) {
    // blocks are whole: columns behind n are padding of the buffer
    const bool in = live && col < n;
    const float4* s = reinterpret_cast<const float4*>(e.saved + (in ? saved_at(e.saved_bands, row, col) : 0));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        k.g[j] = s[j * 32];
        k.u[j] = s[128 + j * 32];
    }
}
template <int ACT>
__device__ __forceinline__ void dgate_epilogue(const TileProblem& q, GateChunk& next, int row, int n_tile,
                                               const TileSums& sums, int c0, int c1) {
    const EpiParams& e = q.epi;
    const bool live = row < q.m;
    for (int c = c0; c < c1; c += 16) {
        const GateChunk k = next;
        const int col = n_tile * q.bn + c;
        if (c + 16 < c1) load_gate(next, e, row, col + 16, live, q.n);
        uint32_t r[16];
        sums.get<false>(0, c, r);
        const int valid = min(16, q.n - col);
        if (!live || valid <= 0) continue;
        float dg[16], du[16], h[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float4 g4 = k.g[j / 4], u4 = k.u[j / 4];
            const float g = j % 4 == 0 ? g4.x : j % 4 == 1 ? g4.y : j % 4 == 2 ? g4.z : g4.w;
            const float u = j % 4 == 0 ? u4.x : j % 4 == 1 ? u4.y : j % 4 == 2 ? u4.z : u4.w;
            const float dh = __uint_as_float(r[j]);
            const float2 a = gate_act_grad(g, e.act);
            dg[j] = dh * u * a.y;
            du[j] = dh * a.x;
            h[j] = a.x * u;
        }
        const int64_t at = int64_t(row) * e.ldo + col;
        store16<ACT>(e.dg + at, dg, valid);
        store16<ACT>(e.du + at, du, valid);
        store16<ACT>(e.h + at, h, valid);
    }
}

// A warp's 32 rows x columns [c0, c1) of a tile, 64 columns at a time: packed into shared memory in the
// 128-byte swizzle and written by TMA, whole 128-byte lines.  (Storing 32 bytes of each row directly
// takes the load/store unit 32 lines an instruction, 5 us a tile, which the MMAs of a weight gradient
// over few tokens do not hide: 190 us for three of 4096 x 14336 over 16 tokens, 103 this way.)
template <int ACT>
__device__ __forceinline__ void store_rows(const TileProblem& q, unsigned char* rows, int row0, int col0, uint32_t tmem,
                                           int c0, int c1) {
    const int lane = threadIdx.x & 31;
    for (int c = c0; c < c1; c += 64) {
        if (lane == 0) tma_store_wait_read();
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            uint32_t r[2][16];
            tmem_ld16(tmem + c + 16 * k, r[0]);
            tmem_ld16(tmem + c + 16 * k + 16, r[1]);
            tmem_wait16(r[0]);
            tmem_wait16(r[1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t* v = &r[i / 2][8 * (i & 1)];
                uint4 o;
                o.x = pack_act<ACT>(__uint_as_float(v[0]), __uint_as_float(v[1]));
                o.y = pack_act<ACT>(__uint_as_float(v[2]), __uint_as_float(v[3]));
                o.z = pack_act<ACT>(__uint_as_float(v[4]), __uint_as_float(v[5]));
                o.w = pack_act<ACT>(__uint_as_float(v[6]), __uint_as_float(v[7]));
                *reinterpret_cast<uint4*>(rows + lane * 128 + (((2 * k + i) ^ (lane & 7)) << 4)) = o;
            }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0 && row0 < q.m && col0 + c < q.n) tma_store_2d(&q.out, col0 + c, row0, rows);
    }
}

template <int EPI, int ACT>
__global__ void __launch_bounds__(kTileThreads, 1) tile_kernel(const __grid_constant__ TileParams p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    using Smem = TileSmem<EPI>;
    constexpr int kTileStages = Smem::kTileStages;
    Smem& S = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr bool I8 = epi_is_i8(EPI);
    constexpr int kBlockK = I8 ? 128 : 64;      // elements of a 128-byte K block
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t place = cluster_rank(), rank = place & 1, leader = place & ~1u;
    const int splits = p.splits, share = int(place >> 1);
    const int cluster = blockIdx.x / (2 * splits), n_clusters = gridDim.x / (2 * splits);

    if (tid == 0) {
        for (int i = 0; i < kTileStages; ++i) {
            mbar_init(&S.full[i], 1);     // the first CTA's loader; bytes of both CTAs
            mbar_init(&S.empty[i], 1);    // the pair's commit
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&S.acc_full[i], 1);
            mbar_init(&S.acc_empty[i], 16);   // 8 epilogue warps of each CTA
        }
        S.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) tmem_alloc_n<1>(&S.tmem_base, kTileTmemCols);
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = S.tmem_base;
    volatile int* abort_flag = &S.abort_flag;
    grid_dependency_wait();
    grid_dependents_launch();

    if (warp == 0) {
        uint32_t it = 0, stage = 0, phase = 1;      // phase: parity the ring's next pass waits for
        bool go = true;
        for (int turn = 0, tile; go && (tile = tile_of_turn(p, turn, cluster, n_clusters)) < p.n_tiles; ++turn) {
            const TileAt t = tile_at(p, tile);
            const TileProblem& q = p.prob[t.prob];
            const int m0 = t.m * 256 + int(rank) * 128;
            // a gated product's pair holds the same columns of gate (first CTA) and up
            const int n0 = epi_is_gate(EPI) ? t.n * (q.bn / 2) : t.n * q.bn + int(rank) * (q.bn / 2);
            const uint32_t bytes = 2u * (kHalfBytes + uint32_t(q.bn) * 64u);
            const int nk = k_total(q), k_first = nk * share / splits, k_last = nk * (share + 1) / splits;
            for (int seg = 0, before = 0; go && seg < 2; before += q.nk[seg++]) {
                const CUtensorMap* ma = &q.a[q.a_of[seg]];
                const CUtensorMap* mb = &q.b[epi_is_gate(EPI) ? rank : q.b_of[seg]];
                const int last = min(q.nk[seg], k_last - before);
                for (int kb = max(0, k_first - before); kb < last; ++kb, ++it) {
                    if (!mbar_wait_warp(&S.empty[stage], phase, abort_flag, p.flags)) {
                        go = false;
                        break;
                    }
                    if (elect_one()) {
                        const uint32_t bar = map_to_rank(smem_u32(&S.full[stage]), leader);
                        if (rank == 0) mbar_expect_tx(&S.full[stage], bytes);
                        const int k0 = kb * kBlockK;
                        const uint32_t da = smem_u32(S.a[stage]), db = smem_u32(S.b[stage]);
                        if (!I8 && q.a_mn) {
                            tma_load_2d_pair(da, ma, m0, k0, bar);
                            tma_load_2d_pair(da + 8192, ma, m0 + 64, k0, bar);
                        } else {
                            tma_load_2d_pair(da, ma, k0, m0, bar);
                        }
                        if (!I8 && q.b_mn) {
                            tma_load_2d_pair(db, mb, n0, k0, bar);
                            if (q.bn == 256) tma_load_2d_pair(db + 8192, mb, n0 + 64, k0, bar);
                        } else {
                            tma_load_2d_pair(db, mb, k0, n0, bar);
                        }
                    }
                    __syncwarp();
                    if (++stage == kTileStages) stage = 0, phase ^= 1;
                }
            }
        }
        // every stage this loader filled is read before the CTA may leave (bounded)
        if (lane == 0) {
            for (uint32_t i = 0; i < kTileStages && i < it; ++i) {
                const uint32_t last = it - 1 - i;
                mbar_drain(&S.empty[last % kTileStages], (last / kTileStages) & 1, p.flags);
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            uint32_t n = 0, stage = 0, phase = 0;
            bool go = true;
            for (int tile; go && (tile = tile_of_turn(p, n, cluster, n_clusters)) < p.n_tiles; ++n) {
                const TileProblem& q = p.prob[tile_at(p, tile).prob];
                const uint32_t idesc = umma_idesc(I8, ACT == VY_BF16, q.a_mn, q.b_mn, 256, q.bn);
                // one MMA's K (32 bytes): along the swizzled row, or 16 rows of 128 bytes
                const uint32_t a_step = q.a_mn ? 128 : 2, b_step = q.b_mn ? 128 : 2;
                const uint64_t a_desc = umma_desc(smem_u32(S.a[0]), q.a_mn ? 8192 : 16, 1024);
                const uint64_t b_desc = umma_desc(smem_u32(S.b[0]), q.b_mn ? 8192 : 16, 1024);
                const uint32_t buf = n & 1, d = tmem + buf * 256;
                const int nk = k_total(q), blocks = nk * (share + 1) / splits - nk * share / splits;
                if (!mbar_wait_warp(&S.acc_empty[buf], ((n >> 1) & 1) ^ 1, abort_flag, p.flags)) break;
                tc_fence_after();
                for (int kb = 0; kb < blocks; ++kb) {
                    if (!mbar_wait_warp(&S.full[stage], phase, abort_flag, p.flags)) {
                        go = false;
                        break;
                    }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t da = a_desc + stage * (kHalfBytes >> 4), db = b_desc + stage * (kHalfBytes >> 4);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ss<I8, 1>(d, da + k * a_step, db + k * b_step, idesc, kb != 0 || k != 0);
                        mma_commit_pair(&S.empty[stage], leader);
                        if (kb == blocks - 1) mma_commit_pair(&S.acc_full[buf], leader);
                    }
                    __syncwarp();
                    if (++stage == kTileStages) stage = 0, phase ^= 1;
                }
            }
        }
    } else if (warp >= 4 && splits == 1) {
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        uint32_t n = 0;
        for (int tile; (tile = tile_of_turn(p, n, cluster, n_clusters)) < p.n_tiles; ++n) {
            const TileAt t = tile_at(p, tile);
            const uint32_t buf = n & 1;
            const TileProblem& q = p.prob[t.prob];
            const int row = t.m * 256 + int(rank) * 128 + quarter * 32 + lane;
            const int width = epi_is_gate(EPI) ? q.bn / 2 : q.bn, c0 = half * (width / 2), c1 = c0 + width / 2;
            const TileSums sums{tmem + buf * 256 + (uint32_t(quarter * 32) << 16), nullptr, 1, 0, width,
                                epi_is_gate(EPI) ? 2 : 1, width};
            GateChunk first;
            if constexpr (EPI == EPI_DGATE) load_gate(first, q.epi, row, t.n * q.bn + c0, row < q.m, q.n);
            load_cols<EPI>(S.cols[warp & 7], q, t.n, c0, c1);
            const float rs = epi_is_i8(EPI) && row < q.m ? q.epi.row_scale[row] : 0.f;
            const bool ready = mbar_wait(&S.acc_full[buf], (n >> 1) & 1, abort_flag, p.flags);
            if (!__all_sync(0xffffffffu, ready)) break;
            tc_fence_after();
            if constexpr (EPI == EPI_DGATE)
                dgate_epilogue<ACT>(q, first, row, t.n, sums, c0, c1);
            else if constexpr (EPI == EPI_STORE)
                store_rows<ACT>(q, S.rows[warp & 7], row - lane, t.n * q.bn, sums.tmem, c0, c1);
            else
                tile_epilogue<EPI, ACT>(q, row, t.n, sums, c0, c1, rs, S.cols[warp & 7]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(map_to_rank(smem_u32(&S.acc_empty[buf]), leader));
        }
        if (EPI == EPI_STORE && lane == 0) tma_store_wait();
    }
    if (splits > 1) {
        // one tile a cluster: send, meet, add my columns
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const TileAt t = tile_at(p, cluster);
        const TileProblem& q = p.prob[t.prob];
        const int row = t.m * 256 + int(rank) * 128 + quarter * 32 + lane;
        const int width = epi_is_gate(EPI) ? q.bn / 2 : q.bn, own = width / splits;
        const int c0 = share * own + half * (own / 2), c1 = c0 + own / 2;
        const TileSums sums{tmem + (uint32_t(quarter * 32) << 16),
                            reinterpret_cast<const float4*>(S.a) + quarter * 32 + lane, splits, share * own, own,
                            epi_is_gate(EPI) ? 2 : 1, width};
        GateChunk first;
        bool ready = false;
        const float rs = epi_is_i8(EPI) && row < q.m ? q.epi.row_scale[row] : 0.f;
        __syncwarp();
        if (warp >= 4) {
            load_cols<EPI>(S.cols[warp & 7], q, t.n, c0, c1);
            if constexpr (EPI == EPI_DGATE) load_gate(first, q.epi, row, t.n * q.bn + c0, row < q.m, q.n);
            ready = __all_sync(0xffffffffu, mbar_wait(&S.acc_full[0], 0, abort_flag, p.flags));
            tc_fence_after();
        }
        cluster_sync();      // every pair's MMAs are done: the rings may be written over
        if (ready) sums.send(smem_u32(S.a) + (quarter * 32 + lane) * 16, rank, share, half);
        __syncwarp();
        cluster_sync();
        if (ready) {
            if constexpr (EPI == EPI_DGATE)
                dgate_epilogue<ACT>(q, first, row, t.n, sums, c0, c1);
            else
                tile_epilogue<EPI, ACT>(q, row, t.n, sums, c0, c1, rs, S.cols[warp & 7]);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();      // neither CTA leaves while the other may still signal or read it
    tc_fence_after();
    if (warp == 2) tmem_free_n<1>(tmem, kTileTmemCols);
}

// ── host ────────────────────────────────────────────────────────────────────────────────────

// The operands of one K segment: `rows` x K matrices, K-major or (mn) stored [K, rows].
inline int tile_operand(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t k, int64_t ld, bool mn,
                        int box_rows) {
    const int block = dtype == VY_BF16 || dtype == VY_F16 ? 64 : 128;
    return mn ? make_map_2d(map, dtype, base, k, rows, ld, 64, 64)
              : make_map_2d(map, dtype, base, rows, k, ld, block, box_rows);
}

// Lays a launch's problems out (sizes and K blocks set): tile columns, tiles, K shares.  A gated
// product's tile has bn / 2 output columns.
// K blocks a pair's share is worth joining for.  With 16 : 8 : 4, us: forward 512 x 1024 x 1024 17 : 24 : 24,
// 200 x 2048 x 768 22 : 21 : 24, 200 x 2048 x 2048 29 : 28 : 28, 1003 x 2048 x 768 24 : 24 : 28; int8
// 300 x 2048 -> 2048 8.7 : 12.2 : 12.3; with gradients 200 x 2048 x 768 58 : 52 : 56, 1003 x 2048 x 768
// 64 : 61 : 65.  (8 gains little where it gains and loses 40 % where 16 blocks become two shares.)
constexpr int kShareLeast = 16;
inline void tile_layout(TileParams* p, bool gate, const ClusterCaps& caps) {
    const int pairs = caps.one[1];
    int least = 1 << 30, wide = 0;
    for (int i = 0; i < p->n_problems; ++i) {
        const TileProblem& q = p->prob[i];
        const int n = gate ? 2 * q.n : q.n;
        if (k_total(q) < least) least = k_total(q);
        wide += (q.m + 255) / 256 * ((n + 255) / 256);
    }
    p->splits = 1;
    // every tile's cluster is resident at once, and every share long enough
    for (int i = 2; i < 4 && wide <= caps.one[i] && least >= kShareLeast << (i - 1); ++i) p->splits = 1 << (i - 1);
    const bool narrow = p->splits == 1 && wide * 2 <= pairs;
    p->n_tiles = 0;
    for (int i = 0; i < p->n_problems; ++i) {
        TileProblem& q = p->prob[i];
        q.bn = narrow || (gate ? 2 * q.n : q.n) <= 128 ? 128 : 256;
        if (q.bn == 128 && p->splits > 2) p->splits = 2;      // an epilogue warp takes 16 columns at least
        const int width = gate ? q.bn / 2 : q.bn;
        q.m_tiles = (q.m + 255) / 256;
        q.n_tiles = (q.n + width - 1) / width;
        q.first = p->n_tiles;
        p->n_tiles += q.m_tiles * q.n_tiles;
    }
    p->n_long = p->extra = 0;
    const TileProblem& q = p->prob[0];
    if (p->n_problems > 1 && k_total(q) >= 2 * least && p->n_tiles > pairs) {
        const int n = q.m_tiles * q.n_tiles, odd = n % pairs;
        const int extra = (k_total(q) + least / 2) / least;
        if (odd && extra * (pairs - odd) <= p->n_tiles - n) p->n_long = n, p->extra = extra;
    }
}

// Adds a problem to a launch: m x n, `segments` K segments of nk blocks.
inline TileProblem& tile_add(TileParams* p, int64_t m, int64_t n, int nk, int segments = 1) {
    TileProblem& q = p->prob[p->n_problems++];
    q.m = static_cast<int>(m);
    q.n = static_cast<int>(n);
    for (int i = 0; i < segments; ++i) q.nk[i] = nk;
    return q;
}

template <int EPI, int ACT>
int tile_launch(const TileParams& p, const ClusterCaps& caps, cudaStream_t s) {
    const int pairs = caps.one[1];
    auto kern = tile_kernel<EPI, ACT>;
    constexpr int smem = sizeof(TileSmem<EPI>) + 1024;
    int st = once_per_device(reinterpret_cast<const void*>(kern), [](int, void* k) {
        const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        return e == cudaSuccess ? VY_OK : fail(VY_ERR_CUDA, "dense GEMM shared memory: %s", cudaGetErrorString(e));
    }, reinterpret_cast<void*>(kern));
    if (st != VY_OK) return st;
    const int clusters = p.n_tiles < pairs ? p.n_tiles : pairs;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * p.splits * clusters);
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2 * p.splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return fail(VY_ERR_CUDA, "dense GEMM launch: %s", cudaGetErrorString(e));
    return VY_OK;
}

}  // namespace vy
