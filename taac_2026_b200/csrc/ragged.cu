// Matrix products grouped by expert with ragged sizes, and their gradients, for sm_100a.  The rows of x [T, K] lie expert by
// expert: expert e owns the rows offsets[e] .. offsets[e + 1] and has weights w[e] [N, K] of its own.
//
//   rows       out[r] = act(x[r] w[e]^T + bias[e]) (+ residual[r])                 r a row of e
//   row grads  dx[r]  = dy[r] w[e]
//   weights    dw[e]  = sum over the rows r of e of dy[r]^T x[r],     db[e] = sum of dy[r]
//
// The offsets are read on the device, so that a router's result needs no copy to the host.  They are clamped to [0, T] and
// to what came before them: whatever they hold, nothing outside the tensors is touched and no row is computed twice.
//
// `ragged_pair_kernel` serves all three on clusters of two CTAs with 256 x 256 tiles, tcgen05 cta_group::2 and fp32 accumulation
// in tensor memory: warp 0 of each CTA feeds a ring of TMA stages, warp 1 of the leader issues the MMAs, eight epilogue warps
// work a tile behind on the other half of the accumulator.  What differs is which dimension is contracted:
//   rows       both operands have the contraction innermost (K-major), as they lie in memory;
//   row grads  w[e] is contracted over its rows: boxes of 64 contraction rows x 64 columns, the MN-major form of the operand;
//   weights    both operands are contracted over the expert's rows, both MN-major.  The last block of an expert reaches into
//              the next one's rows: these are set to zero in shared memory, in both operands (0 x NaN is NaN), before
//              the MMAs see them.
// A row tile that crosses its expert's end computes rows of the next expert for nothing and does not store them.
//
// Distribution.  Row tiles go round robin over the pairs.  The tiles of the weight gradients of uneven experts differ in
// length: they go round robin as well, the long ones first, unless that would leave pairs idle for long; then the rest is cut into
// shares that even the pairs out (see Line), and a tile that two or more pairs share leaves fp32 partial tiles in a workspace, which
// `ragged_join_kernel` adds in the order of the pairs.  The bias gradient comes with the weight gradient: four more warps add the
// rows of dy that lie in shared memory.
//
// Layers with few rows an expert or few tiles go to the kernels of ragged_few.cu (see few_rows and few_weights).
//
// Every wait on an mbarrier is bounded; a wait that gives up raises the status word and all roles drain through the final barrier.
#include "ragged.cuh"
#include "tc_pair.cuh"

namespace tb200 {
void count_launch();
int ragged_few(const void* rows, const void* w, const RaggedArgs& g, int32_t N, int32_t K, bool grads, bool bf16, cudaStream_t st);
int ragged_few_weights(const void* x, const void* dy, const RaggedArgs& g, bool bf16, cudaStream_t st);

namespace {

enum Mode : int { kRows = 0, kRowGrads = 1, kWeights = 2 };

constexpr int kTile = 256;                                // of a pair, both ways; a CTA holds 128 of its rows
constexpr int kBlock = 64;                                // contracted per stage: 128 bytes of a 16-bit type, or 64 rows
constexpr uint32_t kOperandBytes = 128 * 128;             // one CTA's half of an operand in a stage
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
constexpr int kMaxStages = 6;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + kEpiWarps * 32;
constexpr int kSumWarps = 4;                              // weights with a bias gradient: warps that add the rows of dy
constexpr uint32_t kBoxBytes = 32 * 128;                  // an epilogue warp's staging box: 32 rows x 64 columns
constexpr uint32_t kTmemCols = 512;
constexpr int kSnap = 4;
constexpr int64_t kPartFloats = int64_t(kTile) * kTile;   // of a partial tile
constexpr size_t kSmemLimit = 227 * 1024 - 512;           // less the static part

__device__ __forceinline__ int row_tiles(const int32_t* begin, int e) { return (begin[e + 1] - begin[e] + kTile - 1) / kTile; }
// 64-row blocks of an expert's weight gradient, as its tiles' length in the line: at least what writing a tile costs (an expert without
// rows has its zeros written), which is below 2 kSnap, so that such tiles are not shared
constexpr int kLeast = 6;
__device__ __forceinline__ int row_blocks(const int32_t* begin, int e) {
    const int n = (begin[e + 1] - begin[e] + kBlock - 1) / kBlock;
    return n < kLeast ? kLeast : n;
}

// How the tiles of the weight gradients are shared out.  All experts have `tiles` tiles, each as long as its expert has blocks.  The
// experts stand in a line, the long ones in front (but those whose tiles are longer than a pair's equal share at the end), and
// their tiles one after the other.  The first `wave_tiles` of the line, mostly all, go round robin, so that the pairs are on the
// same few experts at a time and read the same rows while these are in the L2.  What lies behind is cut so that all pairs end
// up with equal shares: what few long tiles need.  Measured at 16 experts of 2048 rows, 2048 x 2048: 359 us with one contiguous
// share for every pair (rows of all experts are in use all the time), 218 round robin.
struct Line {
    int32_t* begin;       // [experts + 1] first rows
    int32_t* pre;         // [experts + 1] blocks of one column of tiles before the i-th expert of the line
    int32_t* order;       // [experts] expert numbers in the order of the line
    int64_t* wave_tiles;  // [1]
    int64_t* cut;         // [2] begin and end of this pair's share of the rest
    int32_t* place;       // [kClasses + 1] while the line is made
};
constexpr int kClasses = 32;
__host__ __device__ __forceinline__ size_t line_bytes(int experts) { return 24 + 4 * (3 * static_cast<size_t>(experts) + 2 + kClasses + 1); }
__device__ __forceinline__ Line line_at(void* smem, int experts) {
    int64_t* w = static_cast<int64_t*>(smem);
    int32_t* p = reinterpret_cast<int32_t*>(w + 3);
    return Line{p, p + experts + 1, p + 2 * (experts + 1), w, w + 1, p + 3 * experts + 2};
}
// `p` moved to an edge of its tile where it lies near one: a partial tile costs about as much as kSnap blocks
__device__ __forceinline__ int64_t snapped(const Line& line, int experts, int tiles, int64_t p) {
    if (p >= static_cast<int64_t>(line.pre[experts]) * tiles) return p;
    const int i = expert_of(line.pre, experts, p / tiles);
    const int64_t nb = line.pre[i + 1] - line.pre[i], o = (p - static_cast<int64_t>(line.pre[i]) * tiles) % nb;
    return o < kSnap ? p - o : (nb - o < kSnap ? p - o + nb : p);
}
// By one warp, for one of the pairs.
__device__ void make_line(const RaggedArgs& g, const Line& line, int tiles, int pairs, int pair, int lane) {
    first_rows(g, line.begin, lane);
    if (g.partial == nullptr) {      // no tile is ever shared: all of them go round robin
        prefix(line.pre, g.experts, lane, [&](int e) { return row_blocks(line.begin, e); });
        for (int e = lane; e < g.experts; e += 32) line.order[e] = e;
        if (lane == 0) {
            *line.wave_tiles = static_cast<int64_t>(g.experts) * tiles;
            line.cut[0] = line.cut[1] = 0;
        }
        __syncwarp();
        return;
    }
    int32_t sum = 0;
    for (int e = lane; e < g.experts; e += 32) sum += row_blocks(line.begin, e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int64_t total = static_cast<int64_t>(sum) * tiles, share = total / pairs;
    // the line: a counting sort by length, kClasses steps up to a pair's share, the longest first and those beyond it last
    const int width = static_cast<int>((share < INT32_MAX ? share : INT32_MAX) / kClasses) + 1;
    auto class_of = [&](int e) {
        const int nb = row_blocks(line.begin, e);
        return nb > share ? kClasses : kClasses - 1 - (nb - 1) / width;
    };
    for (int c = lane; c <= kClasses; c += 32) line.place[c] = 0;
    __syncwarp();
    for (int e = lane; e < g.experts; e += 32) atomicAdd(&line.place[class_of(e)], 1);
    __syncwarp();
    if (lane == 0) {
        int at = 0;
        for (int c = 0; c <= kClasses; ++c) {
            const int n = line.place[c];
            line.place[c] = at;
            at += n;
        }
    }
    __syncwarp();
    const int shorter = line.place[kClasses];
    for (int base = 0; base < g.experts; base += 32) {
        const int e = base + lane;
        const int c = e < g.experts ? class_of(e) : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, c);
        const int before = __popc(same & ((1u << lane) - 1));
        const int at = c < 0 ? 0 : line.place[c];
        __syncwarp();
        if (c >= 0) {
            line.order[at + before] = e;
            if (before == 0) line.place[c] = at + __popc(same);
        }
        __syncwarp();
    }
    prefix(line.pre, g.experts, lane, [&](int i) { return row_blocks(line.begin, line.order[i]); });
    // The line as whole tiles, round after round of the pairs, each as long as its first tile: good enough unless it takes half as long
    // again as equal shares would, and some.  Pairs that are done early leave the others their bandwidth, and a cut costs
    // its partial tiles: 16 experts of 2048 rows, 512 -> 2048 (4 rounds for 3.5) take 63 us in whole tiles and 72 cut, 9 of 7282 rows
    // 115 and 134; one expert of 8192 rows (16 tiles) 56 and 35.
    const int64_t rounds = (static_cast<int64_t>(g.experts) * tiles + pairs - 1) / pairs;
    int64_t span = 0;
    for (int64_t w = lane; w < rounds; w += 32) {
        const int i = static_cast<int>(w * pairs / tiles);
        span += line.pre[i + 1] - line.pre[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) span += __shfl_xor_sync(0xffffffffu, span, o);
    if (shorter == g.experts && 2 * span <= 3 * share + 12 * kSnap) {
        if (lane == 0) {
            *line.wave_tiles = static_cast<int64_t>(g.experts) * tiles;
            line.cut[0] = line.cut[1] = 0;
        }
        __syncwarp();
        return;
    }
    // else as many rounds as leave every pair within its share: none of a round's tiles is longer than its first one and a class
    const int64_t fit = static_cast<int64_t>(shorter) * tiles / pairs;
    int64_t waves = 0, reached = 0;
    for (bool more = fit > 0; more;) {
        int64_t length = INT32_MAX;
        if (waves + lane < fit) {
            const int i = static_cast<int>((waves + lane) * pairs / tiles);
            length = line.pre[i + 1] - line.pre[i] + width;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, length, o);
            if (lane >= o) length += u;
        }
        const int n = __popc(__ballot_sync(0xffffffffu, reached + length <= share));      // lengths are positive: the first n lanes
        if (n > 0) reached += __shfl_sync(0xffffffffu, length, n - 1);
        waves += n;
        more = n == 32;
    }
    if (lane == 0) *line.wave_tiles = waves * pairs;
    int64_t before = 0;      // blocks of the waves that go to the pairs in front
    const int64_t rest = waves * pairs / tiles;      // the expert that the line's rest begins in
    const int64_t start = waves * pairs >= static_cast<int64_t>(g.experts) * tiles
                              ? total : static_cast<int64_t>(line.pre[rest]) * tiles + waves * pairs % tiles * (line.pre[rest + 1] - line.pre[rest]);
    for (int base = 0; base <= pairs; base += 32) {
        const int q = base + lane;
        int64_t load = 0;
        if (q < pairs) {
            for (int64_t w = 0; w < waves; ++w) {
                const int i = static_cast<int>((w * pairs + q) / tiles);
                load += line.pre[i + 1] - line.pre[i];
            }
        }
        int64_t upto = load;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        if (q == pair || q == pair + 1) {
            const int64_t p = q == pairs ? total : start + total / pairs * q + total % pairs * q / pairs - (before + upto - load);
            line.cut[q - pair] = snapped(line, g.experts, tiles, p);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    __syncwarp();
}

// One piece of a pair's work
struct Job {
    int e;
    int64_t begin, end;        // the expert's rows
    int64_t m0;                // rows: first row of the tile; weights: first row of the expert that is contracted
    int32_t a0, b0;            // weights: first dw row and column; rows: b0 = first column of the tile
    int blocks;                // stages of this piece
    int slot;                  // weights: partial tile that receives it (0: the tile's begin is another pair's), -1: the whole tile
    bool last;                 // weights: the piece reaches the tile's end
};

// The pieces of a pair's work, in the order in which every role of the pair walks them
template <int MODE>
struct Walk {
    const RaggedArgs& g;
    const Line& line;
    int n_tiles, b_tiles;
    int64_t at, stop, step, wave_stop;
    int i = -1;                    // place of the expert in the line (rows: its number)

    __device__ Walk(const RaggedArgs& args, const Line& l, int pair, int pairs) : g(args), line(l) {
        b_tiles = (g.cols + kTile - 1) / kTile;
        n_tiles = MODE == kWeights ? (g.n + kTile - 1) / kTile : 1;
        at = pair;
        step = pairs;
        if (MODE == kWeights) {
            wave_stop = *line.wave_tiles;
            stop = line.cut[1];
            if (at >= wave_stop) rest();
        } else {
            stop = static_cast<int64_t>(line.pre[g.experts]) * b_tiles;
        }
    }
    __device__ void rest() {       // behind the tiles that go round robin
        at = line.cut[0];
        step = 0;
    }
    __device__ bool next(Job& j) {
        if (MODE == kWeights) {
            if (step == 0 && at >= stop) return false;
            const int tiles = n_tiles * b_tiles;
            int tile, first = 0, nb, take;
            if (step != 0) {
                i = static_cast<int>(at / tiles);
                tile = static_cast<int>(at % tiles);
                nb = take = line.pre[i + 1] - line.pre[i];
                at += step;
                if (at >= wave_stop) rest();
            } else {
                i = expert_of(line.pre, g.experts, at / tiles);
                nb = line.pre[i + 1] - line.pre[i];
                const int64_t local = at - static_cast<int64_t>(line.pre[i]) * tiles;
                tile = static_cast<int>(local / nb);
                first = static_cast<int>(local % nb);
                take = stop - at < nb - first ? static_cast<int>(stop - at) : nb - first;
                at += take;
            }
            j.e = line.order[i];
            j.begin = line.begin[j.e];
            j.end = line.begin[j.e + 1];
            j.a0 = tile / b_tiles * kTile;
            j.b0 = tile % b_tiles * kTile;
            j.m0 = j.begin + static_cast<int64_t>(first) * kBlock;
            const int blocks = static_cast<int>((j.end - j.begin + kBlock - 1) / kBlock);
            j.blocks = blocks < take ? blocks : take;
            j.slot = take == nb ? -1 : (first > 0 ? 0 : 1);
            j.last = first + take == nb;
        } else {
            if (at >= stop) return false;
            const int64_t unit = at / b_tiles;
            if (i < 0) i = expert_of(line.pre, g.experts, unit);
            while (unit >= line.pre[i + 1]) ++i;
            j.e = i;
            j.begin = line.begin[i];
            j.end = line.begin[i + 1];
            j.b0 = static_cast<int>(at % b_tiles) * kTile;
            j.a0 = 0;
            j.m0 = j.begin + (unit - line.pre[i]) * kTile;
            j.blocks = (g.depth + kBlock - 1) / kBlock;
            j.slot = -1;
            at += step;
        }
        return true;
    }
};


// CHUNKED: the maps of MN-major operands have chunks of 64 columns (see make_chunk_map)
template <typename T, int MODE, bool RES, bool CHUNKED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads + (MODE == kWeights ? kSumWarps * 32 : 0), 1)
ragged_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                   const __grid_constant__ CUtensorMap tmap_o, const RaggedArgs g) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full_bar[kMaxStages];     // used in the leader only
    __shared__ uint64_t empty_bar[kMaxStages];
    __shared__ uint64_t own_bar[kMaxStages];      // weights, the other CTA: its own loads
    __shared__ uint64_t tmem_full[2];
    __shared__ uint64_t tmem_empty[2];            // used in the leader only
    __shared__ uint32_t tmem_base_slot;
    __shared__ int s_abort;

    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* out_s = ring + static_cast<size_t>(g.stages) * kStageBytes;
    const Line line = line_at(out_s + kEpiWarps * kBoxBytes, g.experts);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();         // 0 = leader
    const int pair = blockIdx.x >> 1;
    const int pairs = gridDim.x >> 1;
    constexpr bool kFmtBf16 = std::is_same<T, __nv_bfloat16>::value;

    if (threadIdx.x == 0) {
        for (int s = 0; s < g.stages; ++s) {
            mbar_init(&full_bar[s], MODE == kWeights ? 2 : 1);
            mbar_init(&empty_bar[s], MODE == kWeights && g.db != nullptr ? 1 + kSumWarps : 1);
            mbar_init(&own_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], 2 * kEpiWarps);
        }
        s_abort = 0;
        fence_mbar_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmap_a);
        tma_prefetch_desc(&tmap_b);
    }
    if (warp == 1) tmem_alloc_pair(&tmem_base_slot, kTmemCols);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();                           // both CTAs' barriers exist before anything is signalled remotely
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    chain_release();                              // not before every CTA holds its tensor memory (see launch_chained)
    chain_wait();
    if (warp == 0) {
        if (MODE == kWeights) {
            make_line(g, line, (g.n + kTile - 1) / kTile * ((g.cols + kTile - 1) / kTile), pairs, pair, lane);
        } else {
            first_rows(g, line.begin, lane);
            prefix(line.pre, g.experts, lane, [&](int e) { return row_tiles(line.begin, e); });
        }
    }
    __syncthreads();

    Walk<MODE> walk(g, line, pair, pairs);
    Job j;
    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer (both CTAs)
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            bool ok = true;
            while (ok && walk.next(j)) {
                for (int b = 0; b < j.blocks; ++b) {
                    if (!mbar_wait_sleep(&empty_bar[s], ph ^ 1) || *reinterpret_cast<volatile int*>(&s_abort)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = ring + static_cast<size_t>(s) * kStageBytes;
                    if (MODE == kWeights) {
                        const int64_t row = j.m0 + static_cast<int64_t>(b) * kBlock;
                        const int32_t y = static_cast<int32_t>(row);
                        const int32_t a0 = j.a0 + static_cast<int>(rank) * 128, b0 = j.b0 + static_cast<int>(rank) * 128;
                        // each CTA's loads count in a barrier of its own, for the warps that add rows; the other CTA's warp 1 tells
                        // the leader when its half is there
                        uint64_t* bar = rank == 0 ? &full_bar[s] : &own_bar[s];
                        mbar_expect_tx(bar, kStageBytes);
                        load_rows<CHUNKED>(&tmap_a, dst, a0, y, bar);
                        load_rows<CHUNKED>(&tmap_b, dst + kOperandBytes, b0, y, bar);
                    } else {
                        if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * kStageBytes);   // the bytes of both CTAs
                        tma_load_2d_pair(dst, &tmap_a, b * 128, static_cast<int32_t>(j.m0) + static_cast<int>(rank) * 128, &full_bar[s]);
                        const int32_t col = j.b0 + static_cast<int>(rank) * 128;
                        if (MODE == kRows) {
                            tma_load_3d_pair(dst + kOperandBytes, &tmap_b, b * 128, col, j.e, &full_bar[s]);
                        } else if (CHUNKED) {
                            tma_load_4d_pair(dst + kOperandBytes, &tmap_b, 0, b * kBlock, col / 64, j.e, &full_bar[s]);
                        } else {
                            tma_load_3d_pair(dst + kOperandBytes, &tmap_b, col * 2, b * kBlock, j.e, &full_bar[s]);
                            tma_load_3d_pair(dst + kOperandBytes + kChunkBytes, &tmap_b, col * 2 + 128, b * kBlock, j.e, &full_bar[s]);
                        }
                    }
                    if (++s == static_cast<uint32_t>(g.stages)) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (!ok) {
                s_abort = 1;
                if (g.status != nullptr) atomicExch(g.status, 1);
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            // ------------------------------------------------------------ MMA issuer (leader; an elected lane issues, see mbar_wait_warp)
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            constexpr uint32_t fmt = kFmtBf16 ? 1 : 0;
            const uint32_t idesc = umma_idesc(fmt, fmt, MODE == kWeights ? 1 : 0, MODE == kRows ? 0 : 1, kTile, kTile);
            // K-major: groups of 8 rows are 1024 bytes apart, 16 elements further along K are 32 bytes.  MN-major: groups of 8
            // contraction rows are 1024 bytes apart, the next 64 columns are a chunk further, 16 contraction rows are 2048 bytes.
            const uint64_t desc_k = umma_desc_sw128(0, 1024, 16), desc_mn = umma_desc_sw128(0, 1024, kChunkBytes);
            const uint64_t da0 = MODE == kWeights ? desc_mn : desc_k, db0 = MODE == kRows ? desc_k : desc_mn;
            constexpr int step_a = MODE == kWeights ? 128 : 2, step_b = MODE == kRows ? 2 : 128;
            const uint32_t ring_lo = (smem_u32(ring) & 0x3FFFFu) >> 4;
            uint32_t s = 0, ph = 0, buf = 0, aph = 0;
            bool ok = true;
            while (ok && walk.next(j)) {
                if (MODE == kWeights && j.blocks == 0) continue;
                if (!mbar_wait_warp(&tmem_empty[buf], aph ^ 1)) { ok = false; break; }
                tc_fence_after_sync();
                const uint32_t d_tmem = tmem + buf * kTile;
                for (int b = 0; b < j.blocks; ++b) {
                    if (!mbar_wait_warp(&full_bar[s], ph)) { ok = false; break; }
                    int depth = kBlock;
                    if (MODE == kWeights) {
                        const int64_t valid = j.end - (j.m0 + static_cast<int64_t>(b) * kBlock);
                        if (valid < kBlock) {
                            depth = tail_depth(static_cast<int>(valid));
                            asm volatile("fence.acq_rel.cluster;" ::: "memory");      // the other CTA has cleared its last rows
                            clear_tail(ring + static_cast<size_t>(s) * kStageBytes, static_cast<int>(valid), lane);
                        }
                    }
                    tc_fence_after_sync();
                    const uint64_t da = da0 + ring_lo + s * (kStageBytes >> 4);
                    const uint64_t db = db0 + ring_lo + s * (kStageBytes >> 4) + (kOperandBytes >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < kBlock / 16; ++k)
                            if (MODE != kWeights || k * 16 < depth) mma_f16_ss_pair(d_tmem, da + step_a * k, db + step_b * k, idesc, (b | k) != 0 ? 1u : 0u);
                        tc_commit_pair(&empty_bar[s]);
                    }
                    __syncwarp();
                    if (++s == static_cast<uint32_t>(g.stages)) {
                        s = 0;
                        ph ^= 1;
                    }
                }
                if (!ok) break;
                if (elect_one()) tc_commit_pair(&tmem_full[buf]);
                __syncwarp();
                aph ^= buf;
                buf ^= 1;
            }
            if (!ok) {
                s_abort = 1;
                if (g.status != nullptr) atomicExch(g.status, 1);
            }
        } else if (MODE == kWeights) {
            // ------------------------------------------------------------ the other CTA's half of a stage is there (and its last rows cleared)
            uint32_t s = 0, ph = 0;
            bool ok = true;
            while (ok && walk.next(j)) {
                for (int b = 0; b < j.blocks; ++b) {
                    if (!mbar_wait_warp(&own_bar[s], ph)) { ok = false; break; }
                    const int64_t valid = j.end - (j.m0 + static_cast<int64_t>(b) * kBlock);
                    if (valid < kBlock) {
                        clear_tail(ring + static_cast<size_t>(s) * kStageBytes, static_cast<int>(valid), lane);
                        if (lane == 0) mbar_arrive_leader_release(&full_bar[s]);      // writes of this warp: a release at cluster scope, which takes a microsecond
                    } else if (lane == 0) {
                        mbar_arrive_leader(&full_bar[s]);
                    }
                    __syncwarp();
                    if (++s == static_cast<uint32_t>(g.stages)) {
                        s = 0;
                        ph ^= 1;
                    }
                }
            }
            if (!ok) {
                s_abort = 1;
                if (g.status != nullptr) atomicExch(g.status, 1);
            }
        }
    } else if (MODE == kWeights && warp >= 2 + kEpiWarps) {
        // ---------------------------------------------------------------- bias gradient (both CTAs, own 128 rows of dw)
        // The rows of dy pass through shared memory for the tiles of the first column anyway; for the other tiles the warps only follow.
        const int sw = warp - 2 - kEpiWarps;
        RowSum<T> sum(sw, lane);
        uint64_t* bar = rank == 0 ? full_bar : own_bar;
        uint32_t s = 0, ph = 0;
        bool ok = true;
        while (ok && walk.next(j)) {
            const bool adds = j.b0 == 0;
            sum.clear();
            for (int b = 0; b < j.blocks; ++b) {
                if (!mbar_wait_warp(&bar[s], ph)) { ok = false; break; }
                if (adds) sum.add(ring + static_cast<size_t>(s) * kStageBytes, j.end - (j.m0 + static_cast<int64_t>(b) * kBlock));
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[s]);
                if (++s == static_cast<uint32_t>(g.stages)) {
                    s = 0;
                    ph ^= 1;
                }
            }
            if (!adds) continue;
            sum.join();
            const int c = static_cast<int>(rank) * 128 + sw * 32 + (lane & 3) * 8;      // of the tile's 256
            if (lane < 4 && j.a0 + c < g.n)
                sum.store(j.slot >= 0 ? g.db_partial + (static_cast<int64_t>(pair) * 2 + j.slot) * kTile + c
                                      : g.db + static_cast<int64_t>(j.e) * g.n + j.a0 + c);
        }
        if (!ok) {
            s_abort = 1;
            if (g.status != nullptr) atomicExch(g.status, 1);
        }
    } else {
        // ---------------------------------------------------------------- epilogue (both CTAs, own 128 rows)
        // A warp owns the 32 rows of its TMEM lane quarter and 128 of the tile's 256 columns, in two units of 64: 32 columns at a
        // time from TMEM, bias / activation / residual, rounded into a private 4 KB box (128-byte swizzle), one TMA store a
        // unit.  The tensor map clips columns; rows behind the expert's end must stay as they are, so a box that reaches
        // behind it is written by plain stores instead, each lane its own row.
        const int ew = warp - 2;
        const int half = ew >> 2;
        const int quarter = warp & 3;             // TMEM lanes [32 quarter, +32) are the ones this warp may read
        const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
        uint8_t* box = out_s + ew * kBoxBytes;
        const int swz = lane & 7;
        T* out = static_cast<T*>(g.out);
        if (MODE != kWeights && g.clear)
            rows_of_none(g, line.begin, static_cast<int64_t>(blockIdx.x) * (kEpiWarps * 32) + threadIdx.x - 64, static_cast<int64_t>(gridDim.x) * (kEpiWarps * 32));
        uint32_t buf = 0, aph = 0;
        bool ok = true;
        int4 left0 = make_int4(-1, 0, 0, 0), left1 = left0;
        while (walk.next(j)) {
            const bool none = MODE == kWeights && j.blocks == 0;      // zeros, without the tensor cores
            const int64_t row0 = MODE == kWeights ? j.a0 + static_cast<int>(rank) * 128 + quarter * 32
                                                  : j.m0 + static_cast<int>(rank) * 128 + quarter * 32;
            const int64_t row = row0 + lane;
            const int64_t row_end = MODE == kWeights ? g.n : j.end;
            const bool boxed = MODE == kWeights || row0 + 32 <= row_end;
            const bool live = row < row_end;
            const int col0 = j.b0 + half * 128;
            // the bias of a piece is asked for a piece ahead (behind the tile's last column: of its last columns, not used)
            const bool biased = MODE == kRows && g.bias != nullptr;
            const float* bias_t = biased ? g.bias + static_cast<int64_t>(j.e) * g.cols : nullptr;
            float4 bias[MODE == kRows ? 8 : 1];
            auto fetch_bias = [&](int col) {
                if (biased) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) bias[MODE == kRows ? q : 0] = __ldg(reinterpret_cast<const float4*>(bias_t + min(col + 4 * q, g.cols - 4)));
                }
            };
            fetch_bias(col0);
            const T* res_row = RES ? static_cast<const T*>(g.residual) + row * g.cols : nullptr;
            float* part = nullptr;
            if (MODE == kWeights && j.slot >= 0) {
                (j.slot == 0 ? left0 : left1) = make_int4(j.e, j.a0, j.b0, j.last);
                part = g.partial + (static_cast<int64_t>(pair) * 2 + j.slot) * kPartFloats + static_cast<int64_t>(rank) * (kPartFloats / 2) +
                       (quarter * 32 + lane) * 4;
            }
            // A warp whose wait gives up stops waiting but keeps walking (it still arrives on the accumulator barrier).
            if (ok && !none) {
                int passed = 1;
                if (lane == 0) passed = mbar_wait_sleep(&tmem_full[buf], aph) ? 1 : 0;
                if (__shfl_sync(0xffffffffu, passed, 0) == 0) ok = false;
            }
            tc_fence_after_sync();
#pragma unroll 1
            for (int piece = 0; piece < 4; ++piece) {              // 32 accumulator columns each, two of them a box
                const int sub = piece & 1;
                const int col = col0 + piece * 32;
                uint32_t acc[32];
                uint4 res[RES ? 4 : 1];
                if (RES) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        res[RES ? q : 0] = live && col + q * 8 < g.cols ? *reinterpret_cast<const uint4*>(res_row + col + q * 8) : make_uint4(0u, 0u, 0u, 0u);
                }
                if (!none) {
                    tmem_ld_2x16(tmem_base + buf * kTile + lane_addr + half * 128 + piece * 32, acc);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[i] = 0u;
                }
                if (sub == 0 && lane == 0) bulk_wait_read<0>();    // this warp's previous store has read the box
                if (!none) tc_wait_ld(acc);
                if (piece == 3 && !none) {                         // the warp holds its share in registers: hand the buffer back
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_leader(&tmem_empty[buf]);
                } else {
                    __syncwarp();
                }
                if (MODE == kWeights && part != nullptr) {         // what lies outside dw is not read again
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (live && col + 4 * q < g.cols) *reinterpret_cast<uint4*>(part + static_cast<int64_t>(half * 32 + piece * 8 + q) * 512) =
                            make_uint4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
                    continue;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = col + q * 8;
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(acc[8 * q + e]);
                    if (MODE == kRows) {
                        if (biased) {
                            const float4 b0 = bias[MODE == kRows ? 2 * q : 0], b1 = bias[MODE == kRows ? 2 * q + 1 : 0];
                            v[0] += b0.x; v[1] += b0.y; v[2] += b0.z; v[3] += b0.w;
                            v[4] += b1.x; v[5] += b1.y; v[6] += b1.z; v[7] += b1.w;
                        }
                        if (g.silu) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = silu(v[e]);
                        }
                        if (RES) {
                            float r[8];
                            Vec16<T>::unpack(res[RES ? q : 0], r);
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] += r[e];
                        }
                    }
                    const uint4 w = Vec16<T>::pack(v);
                    if (boxed) *reinterpret_cast<uint4*>(box + lane * 128 + (((sub * 4 + q) ^ swz) << 4)) = w;
                    else if (live && c < g.cols) *reinterpret_cast<uint4*>(out + row * g.cols + c) = w;
                }
                if (piece < 3) fetch_bias(col + 32);
                if (sub == 1 && boxed) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    const int cbox = col0 + (piece >> 1) * 64;
                    if (lane == 0 && cbox < g.cols && row0 < row_end) {
                        if (MODE == kWeights) tma_store_3d(&tmap_o, box, cbox * 2, static_cast<int32_t>(row0), j.e);
                        else tma_store_2d(&tmap_o, box, cbox * 2, static_cast<int32_t>(row0));
                        bulk_commit();
                    }
                }
            }
            if (!none) {
                aph ^= buf;
                buf ^= 1;
            }
        }
        if (MODE == kWeights && g.partial != nullptr && rank == 0 && ew == 0 && lane == 0) {
            g.pieces[2 * pair] = left0;
            g.pieces[2 * pair + 1] = left1;
        }
        if (lane == 0) bulk_wait_read<0>();       // the last store must have left shared memory before the CTA ends
        if (!ok) {
            s_abort = 1;
            if (g.status != nullptr) atomicExch(g.status, 1);
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();                           // the peer may still read this CTA's shared memory or signal its barriers
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// Adds the partial tiles of every shared weight-gradient tile.  CTA (x, y): if pair x left the begin of a tile, what the pairs behind it
// left of the same tile is added to it, in their order, for kJoinCols of the tile's columns (a thread holds one of the 256 rows).  One
// tile may be shared by all pairs, so four partial tiles are loaded at a time.  One expert of 60000 rows, 512 -> 512 (18 pairs a tile),
// with the products: 66.9 us with one at a time and 32 columns a CTA, 53.5 so, 56.5 with 8 columns, 55.7 with CTAs that walk a list of
// the shared tiles (which costs 172.7 for 156.1 where many are shared).
constexpr int kJoinCols = 16;
template <typename T>
__global__ void __launch_bounds__(256) ragged_join_kernel(const RaggedArgs g, int pairs) {
    constexpr int kQuads = kJoinCols / 4, kAhead = 4;
    chain_release();
    chain_wait();
    const int4 mine = __ldcg(g.pieces + 2 * blockIdx.x + 1);
    const int r = threadIdx.x, lane = threadIdx.x & 31;
    const int row = mine.y + r, col = mine.z + blockIdx.y * kJoinCols;
    if (mine.x < 0 || col >= g.cols) return;
    const bool live = row < g.n, biased = blockIdx.y == 0 && g.db != nullptr && mine.z == 0 && live;
    const float* part = g.partial + (r >> 7) * (kPartFloats / 2) + static_cast<int64_t>(blockIdx.y) * (kQuads * 512) + (r & 127) * 4;
    float4 sum[kQuads];
    float db = 0.f;
    if (live) {
#pragma unroll
        for (int q = 0; q < kQuads; ++q) sum[q] = __ldcg(reinterpret_cast<const float4*>(part + (2 * static_cast<int64_t>(blockIdx.x) + 1) * kPartFloats + q * 512));
        if (biased) db = __ldcg(g.db_partial + (2 * static_cast<int64_t>(blockIdx.x) + 1) * kTile + r);
    }
    bool more = true;
    for (int base = blockIdx.x + 1; more && base < pairs; base += 32) {
        // the pairs with a share of the tile, up to the one that has its end
        const int4 piece = base + lane < pairs ? __ldcg(g.pieces + 2 * (base + lane)) : make_int4(-1, 0, 0, 0);
        uint32_t with = __ballot_sync(0xffffffffu, piece.x >= 0);
        const uint32_t end = __ballot_sync(0xffffffffu, piece.x >= 0 && piece.w != 0);
        if (end != 0) {
            with &= end ^ (end - 1);
            more = false;
        }
        while (with != 0) {
            float4 v[kAhead][kQuads];
            float b[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const bool there = with != 0 && live;
                const int64_t slot = 2 * static_cast<int64_t>(base + (with != 0 ? __ffs(with) - 1 : 0));
                with &= with - 1;
                b[k] = there && biased ? __ldcg(g.db_partial + slot * kTile + r) : 0.f;
#pragma unroll
                for (int q = 0; q < kQuads; ++q)
                    v[k][q] = there ? __ldcg(reinterpret_cast<const float4*>(part + slot * kPartFloats + q * 512)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                db += b[k];
#pragma unroll
                for (int q = 0; q < kQuads; ++q)
                    sum[q] = make_float4(sum[q].x + v[k][q].x, sum[q].y + v[k][q].y, sum[q].z + v[k][q].z, sum[q].w + v[k][q].w);
            }
        }
    }
    if (!live) return;
    if (biased) g.db[static_cast<int64_t>(mine.x) * g.n + row] = db;
    T* out = static_cast<T*>(g.out) + (static_cast<int64_t>(mine.x) * g.n + row) * g.cols;
#pragma unroll
    for (int q = 0; q < kQuads; q += 2) {
        if (col + q * 4 >= g.cols) break;
        const float4 a = sum[q], b = sum[q + 1];
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        *reinterpret_cast<uint4*>(out + col + q * 4) = Vec16<T>::pack(v);
    }
}

// db[e] = sum of the expert's rows of dy where no weight gradient is wanted, in two steps of fixed order.  Step one: CTA (x, y) adds the
// rows of chunk x, `chunk` rows of the matrix, for blockDim.x * 8 columns, and leaves a partial sum for every expert that has rows among them; that of
// expert e stands in row x + e of the table, which no other pair of chunk and expert has, for both grow along the matrix.
// Thread (tx, ty) takes eight columns of every blockDim.y-th row, eight loads in flight.  As many chunks as CTAs fit the chip:
// pieces of 32 rows of one expert, a CTA each, took 42 us instead of 24 for 32768 x 2048, start-up and waves of CTAs.
// Step two adds an expert's partial sums, eight threads a column.
template <typename T>
__global__ void __launch_bounds__(256) ragged_bias_part_kernel(const T* __restrict__ dy, const RaggedArgs g, float* __restrict__ part, int64_t chunk) {
    extern __shared__ float sums[];                              // [blockDim.y - 1][blockDim.x * 8], then the first rows
    const int width = blockDim.x * 8;
    int32_t* begin = reinterpret_cast<int32_t*>(sums + (blockDim.y - 1) * width);
    chain_release();
    chain_wait();
    const int tid = threadIdx.y * blockDim.x + threadIdx.x;
    if (tid < 32) first_rows(g, begin, tid);
    __syncthreads();
    const int64_t from = max(blockIdx.x * chunk, static_cast<int64_t>(begin[0]));
    const int64_t to = min((blockIdx.x + 1) * chunk, static_cast<int64_t>(begin[g.experts]));
    const int col = blockIdx.y * width + threadIdx.x * 8;
    const int by = blockDim.y;
    if (from >= to) return;
    for (int e = expert_of(begin, g.experts, from); e < g.experts && begin[e] < to; ++e) {
        const int64_t first = max(from, static_cast<int64_t>(begin[e])), last = min(to, static_cast<int64_t>(begin[e + 1]));
        if (first >= last) continue;
        float acc[8] = {};
        if (col < g.n) {
            for (int64_t r = first + threadIdx.y; r < last; r += 8 * by) {
                uint4 raw[8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    raw[u] = r + u * by < last ? __ldg(reinterpret_cast<const uint4*>(dy + (r + u * by) * g.n + col)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    float v[8];
                    Vec16<T>::unpack(raw[u], v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i] += v[i];
                }
            }
        }
        if (by > 1) {
            if (threadIdx.y > 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[(threadIdx.y - 1) * width + i * blockDim.x + threadIdx.x] = acc[i];
            }
            __syncthreads();
            for (int k = 1; k < by && threadIdx.y == 0; ++k) {
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] += sums[(k - 1) * width + i * blockDim.x + threadIdx.x];
            }
            __syncthreads();
        }
        if (threadIdx.y == 0 && col < g.n) {
            float4* out = reinterpret_cast<float4*>(part + (static_cast<int64_t>(blockIdx.x) + e) * g.n + col);
            out[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            out[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
        }
    }
}

__global__ void __launch_bounds__(256) ragged_bias_sum_kernel(const RaggedArgs g, const float* __restrict__ part, float* __restrict__ db, int64_t chunk) {
    extern __shared__ int32_t begin[];
    __shared__ float sums[7][32];
    chain_release();
    chain_wait();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    if (ty == 0) first_rows(g, begin, tx);
    __syncthreads();
    const int e = blockIdx.x;
    const int c = blockIdx.y * 32 + tx;
    float s = 0.f;
    if (c < g.n && begin[e + 1] > begin[e]) {
        const int last = static_cast<int>((begin[e + 1] - 1) / chunk);
#pragma unroll 4
        for (int x = static_cast<int>(begin[e] / chunk) + ty; x <= last; x += 8) s += part[(static_cast<int64_t>(x) + e) * g.n + c];
    }
    if (ty > 0) sums[ty - 1][tx] = s;
    __syncthreads();
    if (ty > 0 || c >= g.n) return;
#pragma unroll
    for (int k = 0; k < 7; ++k) s += sums[k][tx];
    db[static_cast<int64_t>(e) * g.n + c] = s;
}

// ------------------------------------------------------------------------------------------------ host side
int pairs_here() { return device_info().sm_count / 2; }

size_t smem_of(int stages, int experts) {
    return 1024 + static_cast<size_t>(stages) * kStageBytes + kEpiWarps * kBoxBytes + line_bytes(experts);
}

template <typename T, int MODE, bool RES, bool CHUNKED>
int launch_pairs(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o, RaggedArgs g, int pairs, cudaStream_t st) {
    g.stages = kMaxStages;
    while (smem_of(g.stages, g.experts) > kSmemLimit) --g.stages;
    static bool attr_set[64] = {};
    const DeviceInfo& dev = device_info();
    if (!attr_set[dev.index]) {
        cudaFuncSetAttribute(ragged_pair_kernel<T, MODE, RES, CHUNKED>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemLimit));
        attr_set[dev.index] = true;
    }
    const int threads = kThreads + (MODE == kWeights && g.db != nullptr ? kSumWarps * 32 : 0);
    launch_chained(ragged_pair_kernel<T, MODE, RES, CHUNKED>, 2 * pairs, threads, smem_of(g.stages, g.experts), st, a, b, o, g);
    count_launch();
    return launch_status();
}

// experts, sizes, type, and the offsets' pointer of a call
int checked(int32_t experts, int64_t T, int32_t N, int32_t K, int dtype) {
    if (experts < 0 || T < 0 || N < 8 || K < 8 || N % 8 != 0 || K % 8 != 0) return TB200_ERR_SHAPE;
    if (T > 0x7FFFFE00ll || N > (1 << 28) || K > (1 << 28) || experts > kMaxExperts) return TB200_ERR_SHAPE;
    if (dtype != TB200_BF16 && dtype != TB200_F16) return TB200_ERR_DTYPE;
    return TB200_OK;
}
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Whether rows and row gradients go to the kernel of few rows: where the experts have up to 64 rows (128 with a depth of up to 512), and
// where it is expected to end first.  With the time that an SM takes it for 64 rows x 128 columns x 64 of the depth as the unit, it takes
// units * blocks / SMs; a round of the pairs' tiles takes 1.09 a block and their start 8.1 more (fitted to the figures
// below and others between them).  Measured, it / the pairs, in us: 16 experts, 512 -> 2048, of 32 rows 7.5 / 13.2, of 64 11.1 / 13.5, of 128 14.8 / 14.2, of
// 256 21.9 / 17.8, their row gradients (2048 deep) 11.4 / 15.7, 13.4 / 16.0, 16.0 / 16.8, 26.9 / 17.5; 64 experts of 64 rows 30.4 / 41.5
// and 34.0 / 33.1; 256 of 128 rows, 512 -> 512, 43.5 / 52.1; one of 4000, 512 -> 512, 7.6 / 9.2; 9 of 512 rows 7.9 / 9.8; 3 of 1500 rows,
// 1024 -> 512, 14.9 / 12.4; one of 256 rows, 2048 -> 2048, 10.9 / 16.2.
bool few_rows(const RaggedArgs& g) {
    const int64_t blocks = (g.depth + kBlock - 1) / kBlock, half = (g.experts + 1) / 2;
    if (g.T <= 64ll * g.experts || (g.T <= 128ll * g.experts && blocks <= 8)) return true;
    const int64_t units = (g.T / 64 + half) * ((g.cols + 127) / 128);
    const int64_t rounds = ((g.T / kTile + half) * ((g.cols + kTile - 1) / kTile) + pairs_here() - 1) / pairs_here();
    return 100 * units * blocks < 2 * pairs_here() * (109 * rounds * blocks + 810);   // two SMs a pair
}

template <typename T>
int rows_of(const void* x, const void* w, RaggedArgs g, int32_t N, int32_t K, bool grads, cudaStream_t st) {
    CUtensorMap ta, tb, to;
    const uint64_t rows = static_cast<uint64_t>(g.T);
    const int32_t in = grads ? N : K, out = grads ? K : N;
    g.cols = out;
    g.depth = in;
    if (few_rows(g)) return ragged_few(x, w, g, N, K, grads, std::is_same<T, __nv_bfloat16>::value, st);
    const bool chunked = grads && K % 64 == 0;
    if (!make_map(&ta, x, in, rows, 0, 128) ||
        !(chunked ? make_chunk_map(&tb, w, K, N, g.experts) : make_map(&tb, w, K, N, g.experts, grads ? 64 : 128)) || !make_map(&to, g.out, out, rows, 0, 32))
        return TB200_ERR_DRIVER;
    const int64_t most = (g.T / kTile + g.experts) * ((out + kTile - 1) / kTile);
    const int pairs = static_cast<int>(most < pairs_here() ? most : pairs_here());
    if (chunked) return launch_pairs<T, kRowGrads, false, true>(ta, tb, to, g, pairs, st);
    if (grads) return launch_pairs<T, kRowGrads, false, false>(ta, tb, to, g, pairs, st);
    if (g.residual != nullptr) return launch_pairs<T, kRows, true, false>(ta, tb, to, g, pairs, st);
    return launch_pairs<T, kRows, false, false>(ta, tb, to, g, pairs, st);
}

// rows from which on partial tiles are provided for: with fewer a tile has 2 kSnap blocks at most, which a cut would not shorten
constexpr int64_t kShareRows = 2 * kSnap * kBlock;

// Whether the weight gradients go to the kernel of 128 x 128 tiles: where it is expected to end first, by times (in hundredths of a us) that
// come close to those measured where the experts have similar numbers of rows: the host sees T / experts only.  There a CTA takes 0.65 us a
// block of 64 rows while two busy ones share its SM (0.3 to 0.55 alone) and five blocks' time a tile at least, and clusters add 3 us.  Here a
// pair takes 0.53 us a block and seven blocks' time at least, with whole tiles or in equal shares; the partial tiles of those and their
// sum, of as many as share a tile, come on top.  Measured, 128 x 128 / pairs, with a bias gradient, in us: 16 experts of 128 rows, 512 -> 2048, 15.8 / 20.4, of 512 29.1 / 30.0, of 1024 49.6 / 46.5; 256 of 128 rows, 512 -> 512,
// 48 / 61; one of 1000, 512 -> 512, 10.2 / 21.0, of 8000 17.5 / 27.0, of 60000 75.6 / 54.2; 20 of 1500, 256 -> 256, 17.2 / 25.3; 2 of 3000,
// 512 -> 2048, 24.9 / 33.1; 4 of 10000, 1024 -> 1024, 132.8 / 108.8; one of 100000, 128 -> 128, 102.9 / 58.5.
// Where one expert has most of the rows this rule is wrong: the mean says single CTAs, and its tiles' chains, shared by nobody, decide the
// time.  One of 32768 rows beside 16 of 128, 512 -> 512: 290 us, 25 with even experts; of 16384 beside 16 of 64: 137 and 15; of 131072
// beside 32 of 512, 128 -> 128: 131 and 19.
//
// A CTA of the 128 x 128 kernel may get the whole chain of blocks of an expert that has all the rows (0.54 us a block), and its waits end after
// two seconds: from kMostChained rows on, 0.57 s, the pairs, which share such a tile, serve the call whatever the times are.
constexpr int64_t kMostChained = int64_t(1) << 26;
bool few_weights(int32_t experts, int64_t T, int32_t N, int32_t K) {
    if (T > kMostChained) return false;
    const auto tiles = [&](int tile) { return static_cast<int64_t>(experts) * ((N + tile - 1) / tile) * ((K + tile - 1) / tile); };
    const int64_t blocks = (T / experts + kBlock - 1) / kBlock, small = tiles(128), large = tiles(kTile), pairs = pairs_here(), here = 4 * pairs;
    const int64_t split = weights_split(small, blocks, here), part = (blocks + split - 1) / split;
    const int64_t few = (split > 1 ? 900 : 600) + 65 * ((small * split + here - 1) / here) * (part > 5 ? part : 5);
    const int64_t length = blocks > 7 ? blocks : 7;
    const int64_t whole = 1200 + 53 * ((large + pairs - 1) / pairs) * length;
    const int64_t shared = 1500 + 45 * pairs / large + 53 * large * length / pairs;
    return few < (whole < shared ? whole : shared);
}

template <typename T>
int weights_of(const void* x, const void* dy, RaggedArgs g, cudaStream_t st) {
    if (few_weights(g.experts, g.T, g.n, g.cols)) return ragged_few_weights(x, dy, g, std::is_same<T, __nv_bfloat16>::value, st);
    CUtensorMap ta, tb, to;
    const uint64_t rows = static_cast<uint64_t>(g.T);
    const bool chunked = g.n % 64 == 0 && g.cols % 64 == 0;
    if (!(chunked ? make_chunk_map(&ta, dy, g.n, rows, 0) && make_chunk_map(&tb, x, g.cols, rows, 0)
                  : make_map(&ta, dy, g.n, rows, 0, 64) && make_map(&tb, x, g.cols, rows, 0, 64)) || !make_map(&to, g.out, g.cols, g.n, g.experts, 32))
        return TB200_ERR_DRIVER;
    const int pairs = pairs_here();
    const int code = chunked ? launch_pairs<T, kWeights, false, true>(ta, tb, to, g, pairs, st) : launch_pairs<T, kWeights, false, false>(ta, tb, to, g, pairs, st);
    if (code != TB200_OK || g.partial == nullptr) return code;
    launch_chained(ragged_join_kernel<T>, dim3(pairs, kTile / kJoinCols), 256, 0, st, g, pairs);
    count_launch();
    return launch_status();
}

// floats of the workspace for shared tiles, where the pairs make the weight gradients: their descriptions and the partial tiles
int64_t share_floats(int32_t experts, int64_t T, int32_t N, int32_t K) {
    return T < kShareRows || few_weights(experts, T, N, K) ? 0 : static_cast<int64_t>(pairs_here()) * (8 + 2 * kTile + 2 * kPartFloats);
}

// How the sum of the bias gradient's rows is laid over the chip: as many threads along the columns as there are octets (whole warps, at
// most the CTA), the others along the rows; four CTAs an SM, at least 16 rows each
struct BiasShape {
    int tx, columns;      // threads along the columns, CTAs along them
    int64_t chunk, chunks;
};
BiasShape bias_shape(int64_t T, int32_t N) {
    BiasShape b{32, 0, 16, 0};
    while (b.tx < 256 && b.tx * 8 < N) b.tx *= 2;
    b.columns = (N + b.tx * 8 - 1) / (b.tx * 8);
    const int64_t ctas = static_cast<int64_t>(device_info().sm_count) * 4 / b.columns;
    const int64_t rows = ctas < 1 ? T : (T + ctas - 1) / ctas;
    if (rows > b.chunk) b.chunk = rows;
    b.chunks = (T + b.chunk - 1) / b.chunk;
    return b;
}

}  // namespace
}  // namespace tb200

extern "C" int tb200_ragged_gemm(const void* x, const void* w, const int32_t* offsets, const float* bias, const void* residual, void* out,
                                 int32_t experts, int64_t T, int32_t N, int32_t K, int32_t act, int32_t clear, int dtype, int32_t* status_word,
                                 void* stream) {
    using namespace tb200;
    const int code = checked(experts, T, N, K, dtype);
    if (code != TB200_OK) return code;
    if (act < 0 || act > 1) return TB200_ERR_UNSUPPORTED;
    if (T == 0) return TB200_OK;
    if (x == nullptr || out == nullptr || offsets == nullptr || (experts > 0 && w == nullptr)) return TB200_ERR_NULL;
    if (!aligned16(x) || !aligned16(w) || !aligned16(out) || !aligned16(residual) || !aligned16(bias) || !aligned4(offsets)) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (experts == 0) {
        const size_t bytes = static_cast<size_t>(T) * N * 2;
        if (!clear || residual == out) return TB200_OK;
        return static_cast<int>(residual == nullptr ? cudaMemsetAsync(out, 0, bytes, st) : cudaMemcpyAsync(out, residual, bytes, cudaMemcpyDeviceToDevice, st));
    }
    RaggedArgs g{};
    g.offsets = offsets;
    g.bias = bias;
    g.residual = residual;
    g.out = out;
    g.status = status_word;
    g.experts = experts;
    g.T = T;
    g.silu = act;
    g.clear = clear ? 1 : 0;
    return dtype == TB200_BF16 ? rows_of<__nv_bfloat16>(x, w, g, N, K, false, st) : rows_of<__half>(x, w, g, N, K, false, st);
}

extern "C" int tb200_ragged_gemm_dgrad(const void* dy, const void* w, const int32_t* offsets, void* dx, int32_t experts, int64_t T, int32_t N,
                                       int32_t K, int dtype, int32_t* status_word, void* stream) {
    using namespace tb200;
    const int code = checked(experts, T, N, K, dtype);
    if (code != TB200_OK) return code;
    if (T == 0) return TB200_OK;
    if (dy == nullptr || dx == nullptr || offsets == nullptr || (experts > 0 && w == nullptr)) return TB200_ERR_NULL;
    if (!aligned16(dy) || !aligned16(w) || !aligned16(dx) || !aligned4(offsets)) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (experts == 0) return static_cast<int>(cudaMemsetAsync(dx, 0, static_cast<size_t>(T) * K * 2, st));
    RaggedArgs g{};
    g.offsets = offsets;
    g.out = dx;
    g.status = status_word;
    g.experts = experts;
    g.T = T;
    g.clear = 1;
    return dtype == TB200_BF16 ? rows_of<__nv_bfloat16>(dy, w, g, N, K, true, st) : rows_of<__half>(dy, w, g, N, K, true, st);
}

// Partial tiles where dw is wanted, else the table of the kernel that adds the bias gradient's rows alone
extern "C" int64_t tb200_ragged_wgrad_workspace_of(int32_t experts, int64_t T, int32_t N, int32_t K, int32_t weights) {
    using namespace tb200;
    if (checked(experts, T, N, K, TB200_BF16) != TB200_OK || experts == 0 || !device_info().valid) return 0;
    return 4 * (weights ? share_floats(experts, T, N, K) : (bias_shape(T, N).chunks + experts) * N);
}

extern "C" int64_t tb200_ragged_wgrad_workspace_bytes(int32_t experts, int64_t T, int32_t N, int32_t K) {
    const int64_t with = tb200_ragged_wgrad_workspace_of(experts, T, N, K, 1), without = tb200_ragged_wgrad_workspace_of(experts, T, N, K, 0);
    return with > without ? with : without;
}

extern "C" int tb200_ragged_gemm_wgrad(const void* x, const void* dy, const int32_t* offsets, void* dw, float* db, float* workspace, int32_t experts,
                                       int64_t T, int32_t N, int32_t K, int dtype, int32_t* status_word, void* stream) {
    using namespace tb200;
    int code = checked(experts, T, N, K, dtype);
    if (code != TB200_OK) return code;
    if (experts == 0) return TB200_OK;
    if ((dw == nullptr && db == nullptr) || (T > 0 && (dy == nullptr || offsets == nullptr || workspace == nullptr || (x == nullptr && dw != nullptr))))
        return TB200_ERR_NULL;
    if (!aligned16(x) || !aligned16(dy) || !aligned16(dw) || !aligned16(workspace) || !aligned16(db) || !aligned4(offsets)) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T == 0) {
        cudaError_t err = cudaSuccess;
        if (dw != nullptr) err = cudaMemsetAsync(dw, 0, static_cast<size_t>(experts) * N * K * 2, st);
        if (err == cudaSuccess && db != nullptr) err = cudaMemsetAsync(db, 0, static_cast<size_t>(experts) * N * 4, st);
        return static_cast<int>(err);
    }
    RaggedArgs g{};
    g.offsets = offsets;
    g.out = dw;
    g.status = status_word;
    g.experts = experts;
    g.T = T;
    g.cols = K;
    g.n = N;
    if (dw != nullptr) {
        if (share_floats(experts, T, N, K) > 0) {
            g.pieces = reinterpret_cast<int4*>(workspace);
            g.db_partial = workspace + pairs_here() * 8;
            g.partial = g.db_partial + pairs_here() * 2 * kTile;
        }
        g.db = db;
        return dtype == TB200_BF16 ? weights_of<__nv_bfloat16>(x, dy, g, st) : weights_of<__half>(x, dy, g, st);
    }
    float* part = workspace;
    const BiasShape b = bias_shape(T, N);
    const dim3 grid(static_cast<unsigned>(b.chunks), b.columns), block(b.tx, 256 / b.tx);
    const size_t rows = (static_cast<size_t>(experts) + 1) * 4, smem = static_cast<size_t>(256 / b.tx - 1) * b.tx * 8 * 4 + rows;
    if (dtype == TB200_BF16)
        launch_chained(ragged_bias_part_kernel<__nv_bfloat16>, grid, block, smem, st, static_cast<const __nv_bfloat16*>(dy), g, part, b.chunk);
    else
        launch_chained(ragged_bias_part_kernel<__half>, grid, block, smem, st, static_cast<const __half*>(dy), g, part, b.chunk);
    launch_chained(ragged_bias_sum_kernel, dim3(experts, (N + 31) / 32), 256, rows, st, g, part, db, b.chunk);
    count_launch();
    count_launch();
    return launch_status();
}
