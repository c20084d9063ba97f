// What the kernels of layers grouped by expert share: their arguments, the rows of the experts, tensor maps.
#pragma once
#include "tb200_common.cuh"
#include "tb200_tmap.cuh"
#include "tb200_ptx.cuh"

#include <type_traits>

namespace tb200 {

constexpr int kMaxExperts = 2048;

struct RaggedArgs {
    const int32_t* offsets;     // [experts + 1]
    const float* bias;          // [experts, cols] or NULL (rows)
    const void* residual;       // [T, cols] or NULL (rows)
    void* out;                  // [T, cols], or [experts, n, k] (weights)
    float* db;                  // [experts, n] or NULL (weights)
    float* partial;             // [pairs][2] partial tiles, NULL: tiles are never shared (weights)
    float* db_partial;          // [pairs][2][256] sums of the rows of those pieces
    int4* pieces;               // [pairs][2] what they are part of: expert (-1: nothing), first row and column of the tile, last piece?
    int32_t* status;
    int32_t experts, stages;
    int64_t T;
    int32_t cols;               // of a result row
    int32_t depth;              // contracted length (rows, row grads)
    int32_t n;                  // rows of a weight gradient
    int32_t silu;
    int32_t clear;              // rows of no expert are written too
};

// Where every expert's rows begin, by one warp; the offsets come from the kernel in front.  An offset outside [0, T] is moved to
// the nearer end and one that lies before an earlier one counts as that one, so that no two experts share a row.
__device__ __forceinline__ void first_rows(const RaggedArgs& g, int32_t* begin, int lane) {
    constexpr int kAhead = 4;      // loads in flight
    int32_t top = 0;
    for (int base = 0; base <= g.experts; base += 32 * kAhead) {
        int32_t v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = base + 32 * k + lane <= g.experts ? __ldcg(g.offsets + base + 32 * k + lane) : 0;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int at = base + 32 * k;
            if (at > g.experts) break;
            int32_t m = v[k] < 0 ? 0 : (v[k] > g.T ? static_cast<int32_t>(g.T) : v[k]);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t u = __shfl_up_sync(0xffffffffu, m, o);
                if (lane >= o) m = max(m, u);
            }
            m = max(m, top);
            if (at + lane <= g.experts) begin[at + lane] = m;
            top = __shfl_sync(0xffffffffu, m, 31);
        }
    }
    __syncwarp();
}
// pre[i] = sum of units(0 .. i - 1), by one warp
template <typename F>
__device__ __forceinline__ void prefix(int32_t* pre, int n, int lane, F units) {
    int32_t sum = 0;
    for (int base = 0; base < n; base += 32) {
        int32_t v = base + lane < n ? units(base + lane) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (base + lane < n) pre[base + lane + 1] = sum + v;
        sum += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) pre[0] = 0;
    __syncwarp();
}
// the last i with pre[i] <= unit: the expert whose units hold `unit`
__device__ __forceinline__ int expert_of(const int32_t* pre, int experts, int64_t unit) {
    int lo = 0, hi = experts;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= unit) lo = mid;
        else hi = mid;
    }
    return lo;
}
// The rows in front of the first expert and behind the last hold the residual's, zeros without one: thread i of n
__device__ __forceinline__ void rows_of_none(const RaggedArgs& g, const int32_t* begin, int64_t i, int64_t n) {
    const int64_t head = begin[0], owned = begin[g.experts] - head;
    const int64_t row_pieces = g.cols / 8, pieces = (g.T - owned) * row_pieces;
    for (; i < pieces; i += n) {
        const int64_t at = i < head * row_pieces ? i : i + owned * row_pieces;
        static_cast<uint4*>(g.out)[at] = g.residual == nullptr ? make_uint4(0u, 0u, 0u, 0u) : static_cast<const uint4*>(g.residual)[at];
    }
}
// ---- weight gradients: stages of 64 contraction rows, as chunks of 64 rows x 128 bytes (MN-major operands, 128-byte swizzle)
constexpr uint32_t kChunkBytes = 64 * 128;

// Contraction rows that an expert's last block is taken for: whole steps of 16, the depth of one MMA
__device__ __forceinline__ int tail_depth(int valid) { return (valid + 15) & ~15; }
// Sets the rows [valid, tail_depth(valid)) of a stage's four chunks to zero, by one warp: eight lanes a row
__device__ __forceinline__ void clear_tail(uint8_t* stage, int valid, int lane) {
    const int end = tail_depth(valid);
    for (int r = valid + (lane >> 3); r < end; r += 4) {
#pragma unroll
        for (int chunk = 0; chunk < 4; ++chunk) *reinterpret_cast<uint4*>(stage + chunk * kChunkBytes + r * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    __syncwarp();
}
// 64 rows of 128 columns as an MN-major operand: two chunks of 64 columns, in one copy where the columns are whole chunks (16 experts of
// 2048 rows, 2048 x 2048: 218 us in two copies, 194 in one)
template <bool CHUNKED>
__device__ __forceinline__ void load_rows(const CUtensorMap* map, uint8_t* dst, int32_t col, int32_t row, uint64_t* bar) {
    if (CHUNKED) {
        tma_load_3d(dst, map, 0, row, col / 64, bar);
    } else {
        tma_load_2d(dst, map, col * 2, row, bar);
        tma_load_2d(dst + kChunkBytes, map, col * 2 + 128, row, bar);
    }
}
// The bias gradient from the dy tiles in shared memory: one of four warps adds the rows for 32 of a tile's 128 columns, a lane for
// eight of them and every eighth row (the order of the rows keeps the lanes of a phase in different banks).
template <typename T>
struct RowSum {
    float2 acc[4];
    int sub, piece;              // this lane's row among eight, and its 16-byte piece of the chunk's 128 bytes
    uint32_t chunk;
    __device__ RowSum(int warp, int lane) : sub(((lane >> 2) & 1) << 2 | lane >> 3), piece((warp & 1) * 4 + (lane & 3)), chunk((warp >> 1) * kChunkBytes) {}
    __device__ void clear() {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = make_float2(0.f, 0.f);
    }
    __device__ void add(const uint8_t* stage, int64_t valid) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 8 + sub;
            if (r < valid) {
                float2 v[4];
                Vec16<T>::unpack2(*reinterpret_cast<const uint4*>(stage + chunk + r * 128 + ((piece ^ (r & 7)) << 4)), v);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = __fadd2_rn(acc[e], v[e]);
            }
        }
    }
    // the eight lanes of a column join; lanes 0 .. 3 hold the sums
    __device__ void join() {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                acc[e].x += __shfl_xor_sync(0xffffffffu, acc[e].x, o);
                acc[e].y += __shfl_xor_sync(0xffffffffu, acc[e].y, o);
            }
        }
    }
    __device__ void store(float* dst) const {
        *reinterpret_cast<float4*>(dst) = make_float4(acc[0].x, acc[0].y, acc[1].x, acc[1].y);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[2].x, acc[2].y, acc[3].x, acc[3].y);
    }
};

// CTAs that share the contraction of a 128 x 128 tile of a weight gradient: as many as fit the chip (`here` at once) and have four blocks of 64
// rows each; below twelve blocks none, as the sums over the cluster cost more than they save: one expert of 300 rows, 512 -> 2048
// (64 tiles of 5 blocks), 9.1 us in two and 7.0 alone; of 1000 rows, 512 -> 512 (16 of 16), 9.8 in four, 10.3 in eight, 11.2 alone.
inline int weights_split(int64_t units, int64_t blocks, int64_t here) {
    for (int split = 8; split > 1; split /= 2)
        if (split * units <= here && blocks >= 4 * split && blocks >= 12) return split;
    return 1;
}

// silu(x) = x / (1 + exp(-x))
__device__ __forceinline__ float silu(float x) { return x * __fdividef(1.0f, 1.0f + __expf(-x)); }

// a matrix or a stack of matrices of 16-bit values, boxes of box_rows x 128 bytes
inline bool make_map(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows, uint64_t stack, uint32_t box_rows) {
    const auto fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[3] = {2 * cols, rows, stack};
    const cuuint64_t strides[2] = {2 * cols, 2 * cols * rows};
    const cuuint32_t box[3] = {128, box_rows, 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, stack == 0 ? 2 : 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The same matrices as chunks of 64 columns, for boxes of 64 rows x two chunks, which land chunk after chunk: the 128 columns of an
// MN-major operand in one copy.  Whole chunks only: the last piece of a row would reach into the next.
inline bool make_chunk_map(CUtensorMap* map, const void* base, uint64_t cols, uint64_t rows, uint64_t stack) {
    const auto fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[4] = {128, rows, cols / 64, stack};
    const cuuint64_t strides[3] = {2 * cols, 128, 2 * cols * rows};
    const cuuint32_t box[4] = {128, 64, 2, 1};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, stack == 0 ? 3 : 4, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tb200
