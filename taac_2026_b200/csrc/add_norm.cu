// Residual addition and RMSNorm in one pass, with a 16 / 32-bit or an 8-bit result, and the backward pass.
//
//   t = x + residual,   s = rsqrt(mean(t^2) + eps),   n = t s w
//   total = t rounded;  normed = n rounded;  q = e4m3(n / scale) with one scale per 128 columns of a row
//
// backward, for the upstream gradients dn of n and dt of t:
//   xh = t s,  g = dn w,  d = s (g - xh mean(g xh)) + dt       (the gradient of x and of residual alike)
//   dw = sum over the rows of dn xh
//
// Statistics and sums are held in fp32; t enters them unrounded, and every stored value is rounded once.  The 8-bit form
// never writes n: a block's largest |n| is found among the lanes that hold the block, so the quantised row leaves in the
// same pass (x, residual and total at their own width, one byte for each value and 4 bytes for each 128).
//
// Both directions are bound by HBM.  A lane works on octets (8 consecutive columns: one 16-byte piece of a 16-bit type, two
// of fp32), so that 16 neighbouring lanes hold a block of 128 columns whatever the type.  Rows of up to 1024 columns belong
// to a warp (to half of one at 128 columns): four octets a lane at most, the row's sums are shuffles alone, and the next
// row's pieces are requested before the current row is worked on.  Wider rows belong to a CTA.
#include "quant.cuh"
#include "tb200_common.cuh"

namespace tb200 {
void count_launch();

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxWideThreads = 512;
constexpr int kMaxCols = kMaxWideThreads * 4 * 8;
constexpr int kMaxPartials = 592;      // rows of the backward pass's partial table: four CTAs on each of 148 SMs

enum Scales : int { kNoQuant = 0, kAmax = 1, kMx = 2 };

// Sum over the lanes of a row.  G: lanes of a row inside a warp, 0: the whole CTA (its warps' sums are added in order by
// everyone; `slot` alternates so that a row's sums are not overwritten while a slower warp still reads them).
template <int G>
__device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
    for (int o = (G == 0 ? 16 : G >> 1); o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (G == 0) {
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
        for (int w = 0; w < (blockDim.x >> 5); ++w) v += slot[w];
    }
    return v;
}

template <typename T>
struct FwdArgs {
    const T *x, *residual, *gamma;
    T *total, *normed;       // either may be NULL
    uint32_t* q;             // e4m3, NULL: no 8-bit output
    void* scales;            // fp32 [rows, cols / 128], or scale atoms
    int64_t rows;
    int32_t cols;
    float eps;
};

// OPT: octets of a lane; G: see row_sum; SC: kind of scales
template <typename T, int OPT, int G, int SC>
__global__ void __launch_bounds__(G == 0 ? kMaxWideThreads : kThreads)
add_norm_kernel(const FwdArgs<T> a) {
    __shared__ float slots[2][kMaxWideThreads / 32];
    chain_release();
    chain_wait();
    constexpr int RPW = G == 0 ? 1 : 32 / G;                 // rows of a warp at a time
    constexpr bool AHEAD = G != 0;                           // the next row in flight under the current one
    const int lane = threadIdx.x & 31;
    const int lanes = G == 0 ? static_cast<int>(blockDim.x) : G;
    const int lg = G == 0 ? static_cast<int>(threadIdx.x) : lane % G;
    const int octets = a.cols >> 3;
    const float inv_cols = 1.0f / static_cast<float>(a.cols);
    Octet<T> gm[OPT];
#pragma unroll
    for (int j = 0; j < OPT; ++j) {
        gm[j].clear();
        if (lg + j * lanes < octets) gm[j].load_cached(a.gamma + static_cast<int64_t>(lg + j * lanes) * 8);
    }
    const int64_t first = G == 0 ? blockIdx.x : (static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5)) * RPW;
    const int64_t step = G == 0 ? gridDim.x : static_cast<int64_t>(gridDim.x) * kWarps * RPW;
    const int sub = G == 0 ? 0 : lane / (G == 0 ? 1 : G);
    Octet<T> nx[OPT], nr[OPT];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int c = lg + j * lanes;
            const int64_t at = row * a.cols + static_cast<int64_t>(c) * 8;
            nx[j].clear();
            nr[j].clear();
            if (row < a.rows && c < octets) {
                nx[j].load(a.x + at);
                if (a.residual != nullptr) nr[j].load(a.residual + at);
            }
        }
    };
    int parity = 0;
    if (AHEAD) fetch(first + sub);
    for (int64_t base = first; base < a.rows; base += step, parity ^= 1) {
        const int64_t row = base + sub;
        const bool live = row < a.rows;
        if (!AHEAD) fetch(row);
        float t[OPT][8];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            float r[8];
            nx[j].unpack(t[j]);
            nr[j].unpack(r);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[j][e] += r[e];
                ss = fmaf(t[j][e], t[j][e], ss);
            }
        }
        if (AHEAD) fetch(row + step);
        const float s = rsqrtf(row_sum<G>(ss, slots[parity]) * inv_cols + a.eps);
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int c = lg + j * lanes;
            const bool in = live && c < octets;
            const int64_t at = row * a.cols + static_cast<int64_t>(c) * 8;
            if (in && a.total != nullptr) Octet<T>::store(a.total + at, t[j]);
            float w[8];
            gm[j].unpack(w);
            float amax = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                t[j][e] = t[j][e] * s * w[e];
                if (SC != kNoQuant) amax = fmaxf(amax, fabsf(t[j][e]));
            }
            if (in && a.normed != nullptr) Octet<T>::store(a.normed + at, t[j]);
            if (SC != kNoQuant) {                            // columns are whole blocks: 16 neighbouring lanes hold one
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                float inv, scale = 1.0f;
                uint32_t byte = 0;
                if (SC == kAmax) {                           // the rule of tb200_quant_act_1x128, on the unrounded n
                    scale = amax > 0.f ? amax / 448.0f : 1.0f;
                    inv = 1.0f / scale;
                } else {
                    byte = pow2_scale(amax, &inv);
                }
                if (in) {
                    *reinterpret_cast<uint2*>(a.q + (at >> 2)) =
                        make_uint2(pack_e4m3x4(t[j][0] * inv, t[j][1] * inv, t[j][2] * inv, t[j][3] * inv),
                                   pack_e4m3x4(t[j][4] * inv, t[j][5] * inv, t[j][6] * inv, t[j][7] * inv));
                    if ((c & 15) == 0) {
                        const int blocks = a.cols >> 7, b = c >> 4;
                        if (SC == kAmax) {
                            static_cast<float*>(a.scales)[row * blocks + b] = scale;
                        } else {
                            uint8_t* atom = static_cast<uint8_t*>(a.scales) + ((row >> 7) * blocks + b) * kSfAtom;
                            *reinterpret_cast<uint32_t*>(atom + sf_row_offset(static_cast<int>(row & 127))) = byte * 0x01010101u;
                        }
                    }
                }
            }
        }
    }
}

template <typename T>
struct BwdArgs {
    const T *total, *gamma, *dn, *dt;     // dt may be NULL
    T* d;
    float* partial;                       // [CTAs, cols]
    int64_t rows;
    int32_t cols;
    float eps;
};

template <typename T, int OPT, int G>
__global__ void __launch_bounds__(G == 0 ? kMaxWideThreads : kThreads)
add_norm_bwd_kernel(const BwdArgs<T> a) {
    extern __shared__ float red[];        // [kWarps][cols] where warps own rows
    __shared__ float slots[4][kMaxWideThreads / 32];
    chain_release();
    chain_wait();
    constexpr int RPW = G == 0 ? 1 : 32 / G;
    constexpr bool AHEAD = G != 0;
    const int lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    const int lanes = G == 0 ? static_cast<int>(blockDim.x) : G;
    const int lg = G == 0 ? static_cast<int>(threadIdx.x) : lane % G;
    const int sub = G == 0 ? 0 : lane / (G == 0 ? 1 : G);
    const int octets = a.cols >> 3;
    const float inv_cols = 1.0f / static_cast<float>(a.cols);
    Octet<T> gm[OPT];
    float aw[OPT][8];
#pragma unroll
    for (int j = 0; j < OPT; ++j) {
        gm[j].clear();
        if (lg + j * lanes < octets) gm[j].load_cached(a.gamma + static_cast<int64_t>(lg + j * lanes) * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) aw[j][e] = 0.f;
    }
    const int64_t first = G == 0 ? blockIdx.x : (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * RPW;
    const int64_t step = G == 0 ? gridDim.x : static_cast<int64_t>(gridDim.x) * kWarps * RPW;
    Octet<T> nt[OPT], nn[OPT], nd[OPT];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int c = lg + j * lanes;
            const int64_t at = row * a.cols + static_cast<int64_t>(c) * 8;
            nt[j].clear();
            nn[j].clear();
            nd[j].clear();
            if (row < a.rows && c < octets) {
                nt[j].load(a.total + at);
                nn[j].load(a.dn + at);
                if (a.dt != nullptr) nd[j].load(a.dt + at);
            }
        }
    };
    int parity = 0;
    if (AHEAD) fetch(first + sub);
    for (int64_t base = first; base < a.rows; base += step, parity ^= 1) {
        const int64_t row = base + sub;
        if (!AHEAD) fetch(row);
        float t[OPT][8], g[OPT][8];
        float ss = 0.f;
        Octet<T> cd[OPT];
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            nt[j].unpack(t[j]);
            nn[j].unpack(g[j]);
            cd[j] = nd[j];
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(t[j][e], t[j][e], ss);
        }
        if (AHEAD) fetch(row + step);
        const float s = rsqrtf(row_sum<G>(ss, slots[parity]) * inv_cols + a.eps);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            float w[8];
            gm[j].unpack(w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float xh = t[j][e] * s;
                aw[j][e] = fmaf(g[j][e], xh, aw[j][e]);
                g[j][e] *= w[e];
                dot = fmaf(g[j][e], xh, dot);
                t[j][e] = xh;
            }
        }
        const float m = row_sum<G>(dot, slots[2 + parity]) * inv_cols;
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int c = lg + j * lanes;
            if (row < a.rows && c < octets) {
                float o[8];
                cd[j].unpack(o);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = fmaf(s, fmaf(-t[j][e], m, g[j][e]), o[e]);
                Octet<T>::store(a.d + row * a.cols + static_cast<int64_t>(c) * 8, o);
            }
        }
    }
    // the CTA's partial sums of dw, in a fixed order: lanes of a warp that hold the same columns, then the warps
    float* out = a.partial + static_cast<int64_t>(blockIdx.x) * a.cols;
    if (G == 0) {
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int c = lg + j * lanes;
            if (c < octets) {
                reinterpret_cast<float4*>(out)[2 * c] = make_float4(aw[j][0], aw[j][1], aw[j][2], aw[j][3]);
                reinterpret_cast<float4*>(out)[2 * c + 1] = make_float4(aw[j][4], aw[j][5], aw[j][6], aw[j][7]);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < OPT; ++j) {
        const int c = lg + j * lanes;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (G == 16) aw[j][e] += __shfl_xor_sync(0xffffffffu, aw[j][e], 16);
            if (sub == 0 && c < octets) red[warp * a.cols + c * 8 + e] = aw[j][e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.cols; i += kThreads) {
        float w = 0.f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) w += red[k * a.cols + i];
        out[i] = w;
    }
}

// dgamma[i] = the sum of the partial rows: 32 threads of a column add every 32nd row, one adds their sums, always in the
// same order
template <typename T>
__global__ void __launch_bounds__(1024) add_norm_sum_kernel(const float* __restrict__ partial, T* __restrict__ dgamma, int n_partials, int cols) {
    chain_release();
    chain_wait();
    __shared__ float sums[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int i = blockIdx.x * 32 + tx;
    float w = 0.f;
    if (i < cols)
        for (int p = ty; p < n_partials; p += 32) w += partial[static_cast<int64_t>(p) * cols + i];
    sums[ty][tx] = w;
    __syncthreads();
    if (ty == 0 && i < cols) {
        w = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) w += sums[k][tx];
        dgamma[i] = from_float<T>(w);
    }
}

// How a row of `octets` is laid over lanes: half a warp, a warp with 1 to 4 octets a lane, or a CTA
struct Shape {
    int g, opt, threads, rows_per_cta;
};
Shape shape_of(int octets) {
    if (octets <= 16) return {16, 1, kThreads, 2 * kWarps};
    if (octets <= 128) return {32, (octets + 31) / 32, kThreads, kWarps};
    const int opt = octets <= 256 ? 1 : (octets <= 512 ? 2 : 4);
    return {0, opt, ((octets + opt - 1) / opt + 31) / 32 * 32, 1};
}

int grid_of(int64_t rows, int rows_per_cta, int per_sm) {
    int64_t ctas = (rows + rows_per_cta - 1) / rows_per_cta;
    const int64_t cap = static_cast<int64_t>(device_info().sm_count) * per_sm;
    if (ctas > cap) ctas = cap;
    return ctas < 1 ? 1 : static_cast<int>(ctas);
}

#define TB200_AN_SHAPES(CALL) \
    switch (sh.g * 8 + sh.opt) { \
        case 16 * 8 + 1: CALL(1, 16); break; \
        case 32 * 8 + 1: CALL(1, 32); break; \
        case 32 * 8 + 2: CALL(2, 32); break; \
        case 32 * 8 + 3: CALL(3, 32); break; \
        case 32 * 8 + 4: CALL(4, 32); break; \
        case 1: CALL(1, 0); break; \
        case 2: CALL(2, 0); break; \
        default: CALL(4, 0); break; \
    }

template <typename T, int SC>
void launch_fwd(const FwdArgs<T>& a, cudaStream_t st) {
    const Shape sh = shape_of(a.cols >> 3);
    const int grid = grid_of(a.rows, sh.rows_per_cta, sh.g == 0 ? 16 : 8);
#define TB200_AN_FWD(OPT, G) launch_chained(add_norm_kernel<T, OPT, G, SC>, grid, sh.threads, 0, st, a)
    TB200_AN_SHAPES(TB200_AN_FWD)
#undef TB200_AN_FWD
    count_launch();
}

template <typename T>
int fwd(const void* x, const void* residual, const void* gamma, void* total, void* normed, void* q, void* scales, int kind, int64_t rows,
        int32_t cols, float eps, cudaStream_t st) {
    const FwdArgs<T> a{static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(gamma), static_cast<T*>(total),
                       static_cast<T*>(normed), static_cast<uint32_t*>(q), scales, rows, cols, eps};
    switch (kind) {
        case kNoQuant: launch_fwd<T, kNoQuant>(a, st); break;
        case kAmax: launch_fwd<T, kAmax>(a, st); break;
        default: launch_fwd<T, kMx>(a, st); break;
    }
    return launch_status();
}

template <typename T>
int bwd(const void* total, const void* gamma, const void* dn, const void* dt, void* d, void* dgamma, float* work, int64_t rows, int32_t cols,
        float eps, cudaStream_t st) {
    const BwdArgs<T> a{static_cast<const T*>(total), static_cast<const T*>(gamma), static_cast<const T*>(dn), static_cast<const T*>(dt),
                       static_cast<T*>(d), work, rows, cols, eps};
    const Shape sh = shape_of(cols >> 3);
    int grid = 0;
    if (rows > 0) {
        grid = grid_of(rows, sh.rows_per_cta, sh.g == 0 ? 2 : 4);
        if (grid > kMaxPartials) grid = kMaxPartials;
        const size_t smem = sh.g == 0 ? 0 : static_cast<size_t>(kWarps) * cols * sizeof(float);    // at most 32 KB
#define TB200_AN_BWD(OPT, G) launch_chained(add_norm_bwd_kernel<T, OPT, G>, grid, sh.threads, smem, st, a)
        TB200_AN_SHAPES(TB200_AN_BWD)
#undef TB200_AN_BWD
        count_launch();
        const int code = launch_status();
        if (code != TB200_OK) return code;
    }
    launch_chained(add_norm_sum_kernel<T>, (cols + 31) / 32, 1024, 0, st, work, static_cast<T*>(dgamma), grid, cols);
    count_launch();
    return launch_status();
}

bool width_served(int32_t cols) { return cols >= 8 && cols % 8 == 0 && cols <= kMaxCols; }

}  // namespace
}  // namespace tb200

extern "C" int tb200_add_rmsnorm_fwd(const void* x, const void* residual, const void* gamma, void* total, void* normed, void* q, void* scales,
                                     int32_t scale_kind, int64_t rows, int32_t cols, float eps, int dtype, void* stream) {
    using namespace tb200;
    if (rows < 0 || cols < 1) return TB200_ERR_SHAPE;
    if (dtype_size(dtype) == 0) return TB200_ERR_DTYPE;
    if (scale_kind < kNoQuant || scale_kind > kMx) return TB200_ERR_UNSUPPORTED;
    if (!width_served(cols) || (scale_kind != kNoQuant && cols % 128 != 0)) return TB200_ERR_UNSUPPORTED;
    if (rows == 0) return TB200_OK;
    if (x == nullptr || gamma == nullptr || (total == nullptr && normed == nullptr && q == nullptr)) return TB200_ERR_NULL;
    if (scale_kind != kNoQuant && (q == nullptr || scales == nullptr)) return TB200_ERR_NULL;
    if (scale_kind == kNoQuant && q != nullptr) return TB200_ERR_UNSUPPORTED;
    for (const void* p : {x, residual, gamma, static_cast<const void*>(total), static_cast<const void*>(normed), static_cast<const void*>(q),
                          static_cast<const void*>(scales)})
        if (p != nullptr && !aligned16(p)) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case TB200_F32: return fwd<float>(x, residual, gamma, total, normed, q, scales, scale_kind, rows, cols, eps, st);
        case TB200_F16: return fwd<__half>(x, residual, gamma, total, normed, q, scales, scale_kind, rows, cols, eps, st);
        default: return fwd<__nv_bfloat16>(x, residual, gamma, total, normed, q, scales, scale_kind, rows, cols, eps, st);
    }
}

extern "C" int64_t tb200_add_rmsnorm_bwd_workspace_bytes(int32_t cols) {
    return cols < 1 ? 0 : static_cast<int64_t>(tb200::kMaxPartials) * cols * static_cast<int64_t>(sizeof(float));
}

extern "C" int tb200_add_rmsnorm_bwd(const void* total, const void* gamma, const void* d_normed, const void* d_total, void* d_in, void* dgamma,
                                     float* workspace, int64_t rows, int32_t cols, float eps, int dtype, void* stream) {
    using namespace tb200;
    if (rows < 0 || cols < 1) return TB200_ERR_SHAPE;
    if (dtype_size(dtype) == 0) return TB200_ERR_DTYPE;
    if (!width_served(cols)) return TB200_ERR_UNSUPPORTED;
    if (gamma == nullptr || dgamma == nullptr || workspace == nullptr || (rows > 0 && (total == nullptr || d_normed == nullptr || d_in == nullptr)))
        return TB200_ERR_NULL;
    for (const void* p : {total, gamma, d_normed, d_total, static_cast<const void*>(d_in), static_cast<const void*>(workspace)})
        if (p != nullptr && !aligned16(p)) return TB200_ERR_ALIGN;
    if (!device_info().valid) return TB200_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case TB200_F32: return bwd<float>(total, gamma, d_normed, d_total, d_in, dgamma, workspace, rows, cols, eps, st);
        case TB200_F16: return bwd<__half>(total, gamma, d_normed, d_total, d_in, dgamma, workspace, rows, cols, eps, st);
        default: return bwd<__nv_bfloat16>(total, gamma, d_normed, d_total, d_in, dgamma, workspace, rows, cols, eps, st);
    }
}
