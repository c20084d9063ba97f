// Products grouped by expert for few rows an expert (ragged.cu holds the forms for many): the operands' roles exchanged,
//     out_e^T = act(w[e] x_e^T + bias[e]) (+ residual_e^T),        dx_e^T = w[e]^T dy_e^T
// so that the 128-row side of the tensor-core tile is 128 output columns, always full, and its free side a few of the
// expert's rows (ROWS = 16 to 64).  The layer is bound by streaming the weights of the experts that have rows, each once;
// 256-row tiles of the pair kernel would be mostly padding and too few to have all SMs load.
//
// A CTA walks units (expert, up to ROWS of its rows, 128 columns) round robin; two CTAs share an SM.  192 threads: warp 0
// fills a ring of {weights 128 x 64, rows ROWS x 64} by TMA (128-byte swizzle), warp 1 issues the MMAs into one of two
// accumulators in tensor memory, warps 2 to 5 read the other (lane = output column, TMEM column = row), add bias, activation and
// residual and turn sixteen rows at a time in shared memory, so that four lanes write the 64 bytes that a warp has of a
// row.  For the row gradients the weights are contracted over their rows: boxes of 64 x 64, the MN-major form of the operand.
//
// Where the units are fewer than the SMs can take and the contraction is long, SPLIT CTAs of a cluster take a part of it each
// and the partial sums, left in shared memory, are added in the order of the ranks, every rank some of the rows.
//
// Measured at 24 rows on 16 experts, 512 -> 2048 (31.7 MB): 8.8 us, 19.1 with the pair kernel.  What decides between the two stands
// in ragged.cu.  The second kernel makes weight gradients in tiles of the same size.
// Every wait is bounded; one that gives up raises the status word and the roles drain through the barriers.
#include "ragged.cuh"

namespace tb200 {
void count_launch();

namespace {

constexpr int kThreads = 192;
constexpr int kTile = 128;                      // output columns of a unit
constexpr int kBlock = 64;
constexpr uint32_t kWBytes = kTile * 128;
constexpr uint32_t kRingBytes = 96 * 1024;      // two CTAs fit an SM
constexpr int kMaxStages = 8;

template <typename T, int ROWS, bool GRADS, int SPLIT>
__global__ void __launch_bounds__(kThreads, 2)
ragged_few_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const RaggedArgs g) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int s_abort;
    __shared__ __align__(16) T turn[4][16][32];                 // a warp's sixteen rows
    constexpr int kPartStride = kTile + 4;                      // floats between the rows of a partial sum
    constexpr uint32_t kXBytes = ROWS * 128, kStage = kWBytes + kXBytes;
    constexpr int kStages = kRingBytes / kStage < kMaxStages ? kRingBytes / kStage : kMaxStages;
    constexpr uint32_t kAccCols = ROWS < 16 ? 16 : ROWS, kTmemCols = 2 * kAccCols < 32 ? 32 : 2 * kAccCols;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int32_t* begin = reinterpret_cast<int32_t*>(ring + kStages * kStage);
    int32_t* pre = begin + g.experts + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 4);
        }
        s_abort = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmap_x);
        tma_prefetch_desc(&tmap_w);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_slot, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    chain_release();   // not before every CTA holds its tensor memory (see launch_chained)
    chain_wait();
    if (warp == 2) {
        first_rows(g, begin, lane);
        prefix(pre, g.experts, lane, [&](int e) { return (begin[e + 1] - begin[e] + ROWS - 1) / ROWS; });
    }
    __syncthreads();

    // unit -> expert, first row, first column
    const int col_tiles = (g.cols + kTile - 1) / kTile;
    const int64_t units = static_cast<int64_t>(pre[g.experts]) * col_tiles;
    const int all_blocks = (g.depth + kBlock - 1) / kBlock;
    const int rank = SPLIT > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int block0 = all_blocks * rank / SPLIT, block1 = all_blocks * (rank + 1) / SPLIT;
    const int64_t first_unit = blockIdx.x / SPLIT, unit_step = gridDim.x / SPLIT;      // with a split a cluster has one unit at most
    auto decode = [&](int64_t u, int& e, int& row, int& col) {
        const int64_t piece = u / col_tiles;
        e = expert_of(pre, g.experts, piece);
        row = begin[e] + static_cast<int>(piece - pre[e]) * ROWS;
        col = static_cast<int>(u % col_tiles) * kTile;
    };
    int e, row, col;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (int64_t u = first_unit; u < units && ok; u += unit_step) {
                decode(u, e, row, col);
                for (int b = block0; b < block1; ++b) {
                    if (!mbar_wait_sleep(&empty_bar[s], ph ^ 1) || *reinterpret_cast<volatile int*>(&s_abort)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = ring + s * kStage;
                    mbar_expect_tx(&full_bar[s], kStage);
                    if (GRADS) {
                        tma_load_3d(dst, &tmap_w, col * 2, b * kBlock, e, &full_bar[s]);
                        tma_load_3d(dst + kChunkBytes, &tmap_w, col * 2 + 128, b * kBlock, e, &full_bar[s]);
                    } else {
                        tma_load_3d(dst, &tmap_w, b * 128, col, e, &full_bar[s]);
                    }
                    tma_load_2d(dst + kWBytes, &tmap_x, b * 128, row, &full_bar[s]);
                    if (++s == kStages) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
        }
    } else if (warp == 1) {    // all lanes walk the loop, an elected one issues (see mbar_wait_warp)
        const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
        const uint32_t idesc = umma_idesc(fmt, fmt, GRADS ? 1 : 0, 0, kTile, ROWS);
        const uint64_t desc_w = GRADS ? umma_desc_sw128(0, 1024, kChunkBytes) : umma_desc_sw128(0, 1024, 16), desc_x = umma_desc_sw128(0, 1024, 16);
        constexpr int step_w = GRADS ? 128 : 2;
        const uint32_t ring_lo = (smem_u32(ring) & 0x3FFFFu) >> 4;
        uint32_t s = 0, ph = 0, buf = 0, aph = 0;
        for (int64_t u = first_unit; u < units && ok; u += unit_step) {
            if (!mbar_wait_warp(&acc_empty[buf], aph ^ 1)) { ok = false; break; }
            tc_fence_after_sync();
            for (int b = block0; b < block1; ++b) {
                if (!mbar_wait_warp(&full_bar[s], ph)) { ok = false; break; }
                tc_fence_after_sync();
                const uint64_t dw = desc_w + ring_lo + s * (kStage >> 4), dx = desc_x + ring_lo + s * (kStage >> 4) + (kWBytes >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kBlock / 16; ++k) mma_f16_ss(tmem + buf * kAccCols, dw + step_w * k, dx + 2 * k, idesc, b > block0 || k > 0 ? 1u : 0u);
                    tc_commit(&empty_bar[s]);
                }
                __syncwarp();
                if (++s == kStages) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (!ok) break;
            if (elect_one()) tc_commit(&acc_full[buf]);
            __syncwarp();
            aph ^= buf;
            buf ^= 1;
        }
    } else {
        const int quarter = warp & 3;
        const int mine = quarter * 32 + lane;                   // output column inside the unit = TMEM lane
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        if (g.clear) rows_of_none(g, begin, static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x - 64, static_cast<int64_t>(gridDim.x) * 128);
        float* part = reinterpret_cast<float*>(ring);
        uint32_t buf = 0, aph = 0;
        for (int64_t u = first_unit; u < units; u += unit_step) {
            decode(u, e, row, col);
            const int c = col + mine;
            const int rows = min(begin[e + 1] - row, ROWS);
            const float bias = g.bias != nullptr && c < g.cols ? __ldg(g.bias + static_cast<int64_t>(e) * g.cols + c) : 0.f;
            if (ok) {
                int passed = 1;
                if (lane == 0) passed = mbar_wait_sleep(&acc_full[buf], aph) ? 1 : 0;
                if (__shfl_sync(0xffffffffu, passed, 0) == 0) ok = false;
            }
            tc_fence_after_sync();
            for (int m = 0; m < ROWS; m += 16) {
                uint32_t acc[16];
                if (m < rows) {
                    tmem_ld_x16(tmem_base + buf * kAccCols + lane_addr + m, acc);
                    tc_wait_ld(acc);
                }
                if (m + 16 >= ROWS) {
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_empty[buf]);
                }
                if (m >= rows) continue;
                if (SPLIT > 1) {                                // every load has been consumed: the ring is free
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(m + i) * kPartStride + mine] = __uint_as_float(acc[i]);
                    continue;
                }
                // a lane's piece of the result: row m + lane / 4 (and eight further), columns 8 (lane % 4) of the warp's 32
                const int pc = col + quarter * 32 + (lane & 3) * 8;
                uint4 res[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = m + (lane >> 2) + 8 * h;
                    res[h] = make_uint4(0u, 0u, 0u, 0u);
                    if (g.residual != nullptr && r < rows && pc < g.cols)
                        res[h] = *reinterpret_cast<const uint4*>(static_cast<const T*>(g.residual) + (static_cast<int64_t>(row) + r) * g.cols + pc);
                }
                // the residual is added in fp32 on this side of the turn, from the lane that has loaded it
                if (g.residual != nullptr) {
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < 2; ++h) *reinterpret_cast<uint4*>(&turn[quarter][(lane >> 2) + 8 * h][(lane & 3) * 8]) = res[h];
                }
                __syncwarp();
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    v[i] = __uint_as_float(acc[i]) + bias;
                    if (g.silu) v[i] = silu(v[i]);
                    if (g.residual != nullptr) v[i] += to_float<T>(turn[quarter][i][lane]);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) turn[quarter][i][lane] = from_float<T>(v[i]);      // a lane's own column
                __syncwarp();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = m + (lane >> 2) + 8 * h;
                    if (r < rows && pc < g.cols)
                        *reinterpret_cast<uint4*>(static_cast<T*>(g.out) + (static_cast<int64_t>(row) + r) * g.cols + pc) =
                            *reinterpret_cast<const uint4*>(&turn[quarter][(lane >> 2) + 8 * h][(lane & 3) * 8]);
                }
                __syncwarp();
            }
            aph ^= buf;
            buf ^= 1;
        }
    }
    if (SPLIT > 1) {
        __syncwarp();
        cluster_sync_all();                                     // every rank's partial sum is in place
        if (warp >= 2 && first_unit < units) {
            decode(first_unit, e, row, col);
            const int mine = (warp & 3) * 32 + lane, c = col + mine;
            const int rows = min(begin[e + 1] - row, ROWS);
            const uint32_t at = smem_u32(ring) + mine * 4;
            const float bias = g.bias != nullptr && c < g.cols ? __ldg(g.bias + static_cast<int64_t>(e) * g.cols + c) : 0.f;
            for (int m0 = rank; m0 < rows; m0 += 8 * SPLIT) {      // eight of this rank's rows at a time, all loads ahead of the sums
                float v[8][SPLIT];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int m = min(m0 + i * SPLIT, ROWS - 1);
#pragma unroll
                    for (int r = 0; r < SPLIT; ++r) v[i][r] = ld_peer(at + m * kPartStride * 4, r);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int m = m0 + i * SPLIT;
                    if (m >= rows || c >= g.cols) break;
                    float sum = bias;
#pragma unroll
                    for (int r = 0; r < SPLIT; ++r) sum += v[i][r];
                    if (g.silu) sum = silu(sum);
                    const int64_t o = (static_cast<int64_t>(row) + m) * g.cols + c;
                    if (g.residual != nullptr) sum += to_float<T>(static_cast<const T*>(g.residual)[o]);
                    static_cast<T*>(g.out)[o] = from_float<T>(sum);
                }
            }
        }
        __syncwarp();
        cluster_sync_all();                                     // nobody leaves while its partial sum is being read
    }
    if (!ok) {
        s_abort = 1;
        if (g.status != nullptr) atomicExch(g.status, 1);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// Weight gradients dw[e] = dy_e^T x_e in 128 x 128 tiles, a CTA each and round robin, two CTAs an SM: four times the tiles of the pair
// kernel, each with a shorter start and a quarter of the epilogue, for layers whose experts have few rows or which have few tiles.
// Both operands are MN-major, contracted over the expert's rows, the rows of the next expert in a last block cleared by the warp
// that issues the MMAs; warps 2 to 5 turn the accumulator in shared memory, 32 columns at a time, so that four lanes write 64 bytes
// of a row; warps 6 to 9 add the rows of dy for the bias gradient.
//
// The layers of a model with many rows and narrow weights have few tiles, each a long contraction that a CTA's ring bounds (0.5 to 0.65 us a
// block, three stages in flight).  SPLIT CTAs of a cluster then take a part of the blocks each and leave partial tiles in their shared memory,
// of which every rank adds some rows, in the order of the ranks.  One expert of 8000 rows, 512 -> 512, in eight: 17.5 us, 39 without.
// The sums over the cluster take 2 us in two parts and 3.5 in eight; read by octets, two loads of 16 bytes 32 apart, they took 9.
constexpr int kSumWarps = 4;
constexpr uint32_t kWeightStage = 4 * kChunkBytes;
static_assert(kTile * (kTile + 4) * 4 <= kRingBytes, "a partial tile fits the ring");

template <typename T, bool CHUNKED, int SPLIT>
__global__ void __launch_bounds__(kThreads + kSumWarps * 32, 2)
ragged_few_weights_kernel(const __grid_constant__ CUtensorMap tmap_dy, const __grid_constant__ CUtensorMap tmap_x, const RaggedArgs g) {
    extern __shared__ uint8_t smem_raw[];
    constexpr int kStages = kRingBytes / kWeightStage;
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int s_abort;
    __shared__ __align__(16) uint4 turn[SPLIT > 1 ? 1 : 4][32 * 4];             // a warp's 32 rows x 64 bytes
    __shared__ __align__(16) float db_part[SPLIT > 1 ? kTile : 4];
    constexpr int kPartStride = kTile + 4;                      // floats between the rows of a partial tile
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int32_t* begin = reinterpret_cast<int32_t*>(ring + kStages * kWeightStage);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], g.db != nullptr ? 1 + kSumWarps : 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&acc_full[b], 1);
            mbar_init(&acc_empty[b], 4);
        }
        s_abort = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmap_dy);
        tma_prefetch_desc(&tmap_x);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_slot, 2 * kTile);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    chain_release();   // not before every CTA holds its tensor memory (see launch_chained)
    chain_wait();
    if (warp == 2) first_rows(g, begin, lane);
    __syncthreads();

    const int b_tiles = (g.cols + kTile - 1) / kTile, tiles = (g.n + kTile - 1) / kTile * b_tiles;
    const int64_t units = static_cast<int64_t>(g.experts) * tiles;
    const int rank = SPLIT > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int64_t first_unit = blockIdx.x / SPLIT, unit_step = gridDim.x / SPLIT;      // with a split a cluster has one unit
    int e, a0, b0, blocks, block0, block1;                      // blocks of the tile; this CTA's
    int64_t first, rows;
    auto decode = [&](int64_t u) {
        e = static_cast<int>(u / tiles);
        const int tile = static_cast<int>(u % tiles);
        a0 = tile / b_tiles * kTile;
        b0 = tile % b_tiles * kTile;
        first = begin[e];
        rows = begin[e + 1] - first;
        blocks = static_cast<int>((rows + kBlock - 1) / kBlock);
        block0 = static_cast<int>(static_cast<int64_t>(blocks) * rank / SPLIT);
        block1 = static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / SPLIT);
    };
    uint32_t s = 0, ph = 0, buf = 0, aph = 0;
    auto next_stage = [&]() {
        if (++s == kStages) {
            s = 0;
            ph ^= 1;
        }
    };
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            for (int64_t u = first_unit; u < units && ok; u += unit_step) {
                decode(u);
                for (int b = block0; b < block1; ++b) {
                    if (!mbar_wait_sleep(&empty_bar[s], ph ^ 1) || *reinterpret_cast<volatile int*>(&s_abort)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = ring + s * kWeightStage;
                    const int32_t y = static_cast<int32_t>(first) + b * kBlock;
                    mbar_expect_tx(&full_bar[s], kWeightStage);
                    load_rows<CHUNKED>(&tmap_dy, dst, a0, y, &full_bar[s]);
                    load_rows<CHUNKED>(&tmap_x, dst + 2 * kChunkBytes, b0, y, &full_bar[s]);
                    next_stage();
                }
            }
        }
    } else if (warp == 1) {    // all lanes walk the loop, an elected one issues (see mbar_wait_warp)
        const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
        constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
        const uint32_t idesc = umma_idesc(fmt, fmt, 1, 1, kTile, kTile);
        const uint64_t desc = umma_desc_sw128(0, 1024, kChunkBytes);
        const uint32_t ring_lo = (smem_u32(ring) & 0x3FFFFu) >> 4;
        for (int64_t u = first_unit; u < units && ok; u += unit_step) {
            decode(u);
            if (block0 == block1) continue;
            if (!mbar_wait_warp(&acc_empty[buf], aph ^ 1)) { ok = false; break; }
            tc_fence_after_sync();
            for (int b = block0; b < block1; ++b) {
                if (!mbar_wait_warp(&full_bar[s], ph)) { ok = false; break; }
                const int64_t valid = rows - static_cast<int64_t>(b) * kBlock;
                int depth = kBlock;
                if (valid < kBlock) {
                    depth = tail_depth(static_cast<int>(valid));
                    clear_tail(ring + s * kWeightStage, static_cast<int>(valid), lane);
                }
                tc_fence_after_sync();
                const uint64_t da = desc + ring_lo + s * (kWeightStage >> 4), db = da + (2 * kChunkBytes >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kBlock / 16; ++k)
                        if (k * 16 < depth) mma_f16_ss(tmem + buf * kTile, da + 128 * k, db + 128 * k, idesc, b > block0 || k > 0 ? 1u : 0u);
                    tc_commit(&empty_bar[s]);
                }
                __syncwarp();
                next_stage();
            }
            if (!ok) break;
            if (elect_one()) tc_commit(&acc_full[buf]);
            __syncwarp();
            aph ^= buf;
            buf ^= 1;
        }
    } else if (warp >= 6) {
        RowSum<T> sum(warp - 6, lane);
        for (int64_t u = first_unit; u < units && ok; u += unit_step) {
            decode(u);
            sum.clear();
            for (int b = block0; b < block1; ++b) {
                if (!mbar_wait_warp(&full_bar[s], ph)) { ok = false; break; }
                if (b0 == 0) sum.add(ring + s * kWeightStage, rows - static_cast<int64_t>(b) * kBlock);
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[s]);
                next_stage();
            }
            if (b0 != 0) continue;
            sum.join();
            const int c = a0 + (warp - 6) * 32 + (lane & 3) * 8;
            if (SPLIT > 1 && lane < 4) sum.store(db_part + (warp - 6) * 32 + (lane & 3) * 8);
            else if (lane < 4 && c < g.n) sum.store(g.db + static_cast<int64_t>(e) * g.n + c);
        }
        if (SPLIT > 1) {                                            // done with the ring
            __syncwarp();
            asm volatile("bar.arrive 1, 256;" ::: "memory");
        }
    } else {
        const int quarter = warp & 3;
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        uint4* box = turn[quarter];
        for (int64_t u = first_unit; u < units; u += unit_step) {
            decode(u);
            if (ok && block0 < block1) {
                int passed = 1;
                if (lane == 0) passed = mbar_wait_sleep(&acc_full[buf], aph) ? 1 : 0;
                if (__shfl_sync(0xffffffffu, passed, 0) == 0) ok = false;
            }
            tc_fence_after_sync();
            if (SPLIT > 1) {                                        // the partial tile, into the ring: the MMAs have read it, the bias warps too
                if (g.db != nullptr) asm volatile("bar.sync 1, 256;" ::: "memory");
                float* part = reinterpret_cast<float*>(ring) + (quarter * 32 + lane) * kPartStride;
                for (int c = 0; c < kTile && block0 < block1; c += 32) {
                    uint32_t acc[32];
                    tmem_ld_2x16(tmem_base + buf * kTile + lane_addr + c, acc);
                    tc_wait_ld(acc);
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        *reinterpret_cast<uint4*>(part + c + 4 * q) = make_uint4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
                }
                continue;
            }
            T* out = static_cast<T*>(g.out) + static_cast<int64_t>(e) * g.n * g.cols;
            for (int c = 0; c < kTile; c += 32) {
                uint32_t acc[32];
                if (blocks > 0) {
                    tmem_ld_2x16(tmem_base + buf * kTile + lane_addr + c, acc);
                    tc_wait_ld(acc);
                    if (c + 32 == kTile) {
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_empty[buf]);
                    }
                } else {      // no rows: zeros, without the tensor cores
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[i] = 0u;
                }
                if (b0 + c >= g.cols) continue;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(acc[8 * q + i]);
                    box[lane * 4 + (q ^ ((lane >> 1) & 3))] = Vec16<T>::pack(v);      // a phase's lanes in different banks
                }
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = q * 8 + (lane >> 2), p = lane & 3;
                    const int row = a0 + quarter * 32 + r, col = b0 + c + p * 8;
                    if (row < g.n && col < g.cols) *reinterpret_cast<uint4*>(out + static_cast<int64_t>(row) * g.cols + col) = box[r * 4 + (p ^ ((r >> 1) & 3))];
                }
                __syncwarp();
            }
            if (blocks > 0) {
                aph ^= buf;
                buf ^= 1;
            }
        }
    }
    if (SPLIT > 1) {
        __syncwarp();
        cluster_sync_all();                                     // every rank's partial tile is in place
        if (warp >= 2) {
            decode(first_unit);
            const uint32_t at = smem_u32(ring);
            const int t = threadIdx.x - 64, threads = blockDim.x - 64;
            constexpr int kItems = kTile / SPLIT * (kTile / 4), kBatch = SPLIT < 8 ? 8 / SPLIT : 1;      // four columns of one of this rank's rows
            for (int i0 = t; i0 < kItems; i0 += kBatch * threads) {
                float4 v[kBatch][SPLIT];
                int r[kBatch], c[kBatch];
                bool live[kBatch];
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    const int i = i0 + b * threads;
                    r[b] = rank * (kTile / SPLIT) + i / (kTile / 4);
                    c[b] = i % (kTile / 4) * 4;
                    live[b] = i < kItems && a0 + r[b] < g.n && b0 + c[b] < g.cols;
#pragma unroll
                    for (int k = 0; k < SPLIT; ++k) {
                        const bool there = live[b] && static_cast<int64_t>(blocks) * k / SPLIT < static_cast<int64_t>(blocks) * (k + 1) / SPLIT;
                        v[b][k] = there ? ld_peer4(at + (r[b] * kPartStride + c[b]) * 4, k) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    float4 sum = v[b][0];
#pragma unroll
                    for (int k = 1; k < SPLIT; ++k) sum = make_float4(sum.x + v[b][k].x, sum.y + v[b][k].y, sum.z + v[b][k].z, sum.w + v[b][k].w);
                    __align__(8) const T four[4] = {from_float<T>(sum.x), from_float<T>(sum.y), from_float<T>(sum.z), from_float<T>(sum.w)};
                    T* dst = static_cast<T*>(g.out) + (static_cast<int64_t>(e) * g.n + a0 + r[b]) * g.cols + b0 + c[b];
                    if (live[b]) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(four);
                }
            }
            if (g.db != nullptr && rank == 0 && b0 == 0 && t < kTile && a0 + t < g.n) {
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < SPLIT; ++k) sum += ld_peer(smem_u32(db_part) + t * 4, k);
                g.db[static_cast<int64_t>(e) * g.n + a0 + t] = sum;
            }
        }
        __syncwarp();
        cluster_sync_all();                                     // nobody leaves while its partial tile is being read
    }
    if (!ok) {
        s_abort = 1;
        if (g.status != nullptr) atomicExch(g.status, 1);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 2 * kTile);
    }
}

// `ctas` of `threads` in clusters of `split`, which may start while the kernel in front still runs
template <typename K, typename... Args>
int launch_clusters(K kernel, int split, int64_t ctas, int threads, size_t smem, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = static_cast<unsigned>(ctas);
    cfg.blockDim = static_cast<unsigned>(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(split);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = split > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);
    count_launch();
    return launch_status();
}

template <typename T, bool CHUNKED, int SPLIT>
int launch_weights(const CUtensorMap& tdy, const CUtensorMap& tx, const RaggedArgs& g, int64_t ctas, cudaStream_t st) {
    static bool attr_set[64] = {};
    const DeviceInfo& dev = device_info();
    if (!attr_set[dev.index]) {
        cudaFuncSetAttribute(ragged_few_weights_kernel<T, CHUNKED, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kRingBytes + 1024 + (kMaxExperts + 1) * 4));
        attr_set[dev.index] = true;
    }
    return launch_clusters(ragged_few_weights_kernel<T, CHUNKED, SPLIT>, SPLIT, ctas, kThreads + (g.db != nullptr ? kSumWarps * 32 : 0),
                           kRingBytes + 1024 + (static_cast<size_t>(g.experts) + 1) * 4, st, tdy, tx, g);
}

template <typename T, bool CHUNKED>
int split_weights(const void* x, const void* dy, const RaggedArgs& g, cudaStream_t st) {
    CUtensorMap tdy, tx;
    const uint64_t rows = static_cast<uint64_t>(g.T);
    if (!(CHUNKED ? make_chunk_map(&tdy, dy, g.n, rows, 0) && make_chunk_map(&tx, x, g.cols, rows, 0)
                  : make_map(&tdy, dy, g.n, rows, 0, 64) && make_map(&tx, x, g.cols, rows, 0, 64)))
        return TB200_ERR_DRIVER;
    const int64_t units = static_cast<int64_t>(g.experts) * ((g.n + kTile - 1) / kTile) * ((g.cols + kTile - 1) / kTile);
    const int64_t here = 2 * static_cast<int64_t>(device_info().sm_count);
    switch (weights_split(units, (g.T / g.experts + kBlock - 1) / kBlock, here)) {
        case 8: return launch_weights<T, CHUNKED, 8>(tdy, tx, g, 8 * units, st);
        case 4: return launch_weights<T, CHUNKED, 4>(tdy, tx, g, 4 * units, st);
        case 2: return launch_weights<T, CHUNKED, 2>(tdy, tx, g, 2 * units, st);
        default: return launch_weights<T, CHUNKED, 1>(tdy, tx, g, units < here ? units : here, st);
    }
}

template <typename T, int ROWS, bool GRADS, int SPLIT>
int launch(const CUtensorMap& tx, const CUtensorMap& tw, const RaggedArgs& g, int64_t ctas, cudaStream_t st) {
    static bool attr_set[64] = {};
    const DeviceInfo& dev = device_info();
    if (!attr_set[dev.index]) {
        cudaFuncSetAttribute(ragged_few_kernel<T, ROWS, GRADS, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kRingBytes + 1024 + (kMaxExperts + 1) * 8));
        attr_set[dev.index] = true;
    }
    return launch_clusters(ragged_few_kernel<T, ROWS, GRADS, SPLIT>, SPLIT, ctas, kThreads,
                           kRingBytes + 1024 + (static_cast<size_t>(g.experts) + 1) * 8, st, tx, tw, g);
}

template <typename T, int ROWS, bool GRADS>
int sized(const void* rows, const void* w, const RaggedArgs& g, int32_t N, int32_t K, cudaStream_t st) {
    CUtensorMap tx, tw;
    if (!make_map(&tx, rows, g.depth, static_cast<uint64_t>(g.T), 0, ROWS) || !make_map(&tw, w, K, N, g.experts, GRADS ? 64 : 128)) return TB200_ERR_DRIVER;
    // units at most, and about how many there will be; a split while those fit the chip at once and every CTA has four blocks of the
    // contraction at least.  Measured, split / not: 16 experts of 16 rows, 2048 deep, 512 columns (64 units) 11.4 / 14.7 us in
    // four; 24 rows on 16 experts, 512 deep, 2048 columns (240 units) 14.8 / 8.8 in two.
    const int64_t columns = (g.cols + kTile - 1) / kTile, some = g.experts < g.T ? g.experts : g.T, full = g.T / ROWS;
    const int64_t most = (full + some) * columns, likely = (full > some / 2 ? full + some / 2 : some) * columns;
    const int64_t here = 2 * static_cast<int64_t>(device_info().sm_count);
    const int blocks = (g.depth + kBlock - 1) / kBlock;
    if (4 * likely <= here && blocks >= 16) return launch<T, ROWS, GRADS, 4>(tx, tw, g, 4 * most, st);
    if (2 * likely <= here && blocks >= 8) return launch<T, ROWS, GRADS, 2>(tx, tw, g, 2 * most, st);
    return launch<T, ROWS, GRADS, 1>(tx, tw, g, most < here ? most : here, st);
}

template <typename T, bool GRADS>
int serve(const void* rows, const void* w, const RaggedArgs& g, int32_t N, int32_t K, cudaStream_t st) {
    // rows of a unit: twice an expert's mean, so that few experts need two
    const int64_t want = 2 * g.T / g.experts;
    if (want <= 16) return sized<T, 16, GRADS>(rows, w, g, N, K, st);
    if (want <= 32) return sized<T, 32, GRADS>(rows, w, g, N, K, st);
    return sized<T, 64, GRADS>(rows, w, g, N, K, st);
}

}  // namespace

// g.cols and g.depth: of the result and contracted
int ragged_few(const void* rows, const void* w, const RaggedArgs& g, int32_t N, int32_t K, bool grads, bool bf16, cudaStream_t st) {
    if (grads) return bf16 ? serve<__nv_bfloat16, true>(rows, w, g, N, K, st) : serve<__half, true>(rows, w, g, N, K, st);
    return bf16 ? serve<__nv_bfloat16, false>(rows, w, g, N, K, st) : serve<__half, false>(rows, w, g, N, K, st);
}

// g.n and g.cols: of a weight gradient
int ragged_few_weights(const void* x, const void* dy, const RaggedArgs& g, bool bf16, cudaStream_t st) {
    const bool chunked = g.n % 64 == 0 && g.cols % 64 == 0;
    if (bf16) return chunked ? split_weights<__nv_bfloat16, true>(x, dy, g, st) : split_weights<__nv_bfloat16, false>(x, dy, g, st);
    return chunked ? split_weights<__half, true>(x, dy, g, st) : split_weights<__half, false>(x, dy, g, st);
}

}  // namespace tb200
