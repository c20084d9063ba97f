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
// of fp32), so that 16 neighbouring lanes hold a block of 128 columns whatever the type.  Forward, rows of up to 1024 columns belong
// to a warp (to half of one at 128 columns): four octets a lane at most, the row's sums are shuffles alone, and the next
// row's pieces are requested before the current row is worked on; wider rows belong to a CTA.
#include "quant.cuh"
#include "tb200_common.cuh"

namespace tb200 {
void count_launch();

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxWideThreads = 512;
constexpr int kMaxCols = kMaxWideThreads * 4 * 8;

enum Scales : int { kNoQuant = 0, kAmax = 1, kMx = 2 };

// Sums over the lanes of a row.  G: lanes of a row inside a warp, 0: `warps` warps from warp `first` on, whose sums everyone adds in
// order (`slot` alternates so that a row's sums are not overwritten while a slower warp still reads them).
template <int G>
__device__ __forceinline__ float2 row_sum(float2 v, float2* slot, int first, int warps) {
#pragma unroll
    for (int o = (G == 0 ? 16 : G >> 1); o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (G == 0) {
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + first), "r"(warps * 32) : "memory");
        v = make_float2(0.f, 0.f);
        for (int w = 0; w < warps; ++w) {
            v.x += slot[first + w].x;
            v.y += slot[first + w].y;
        }
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

// Between these the quotient 448 / amax and its quick form are accurate: a divisor above 2^126 gives the quick form 0, and below
// 448 / 2^128 the quotient is infinite, though amax / 448 is a number at both ends.
constexpr float kLeastAmax = 0x1p-100f, kMostAmax = 0x1p100f;

// The factor of a block outside of them, which takes n by 2^+-100 nearer to 1 first (exact, but for values that are nothing beside the
// block's largest).  It is the reciprocal of the scale as it is stored, which has few bits where it is subnormal.  A scale that
// rounds to zero becomes 1: the block's values, below 2^-141, are zeros.  Infinity makes the whole block NaN.
__device__ __forceinline__ float far_factor(float amax, float* scale, float2 (&n)[4]) {
    if (!(*scale > 0.f)) {
        *scale = 1.0f;
        return 1.0f;
    }
    const float nearer = amax > 1.0f ? 0x1p-100f : 0x1p100f;
#pragma unroll
    for (int e = 0; e < 4; ++e) n[e] = __fmul2_rn(n[e], make_float2(nearer, nearer));
    return __fdividef(1.0f, *scale * nearer);
}

// CTAs an SM that the registers are held to, where the rare branch of far_factor would take some more and a CTA with them: 262144 x 512
// bf16 and fp16 159 us instead of 152, 20000 x 2048 bf16 61 instead of 53.  0: as the compiler has it
template <typename T, int OPT, int G, int SC>
constexpr int fwd_ctas() { return SC == kAmax && ((G == 32 && OPT == 2 && sizeof(T) == 2) || (G == 0 && OPT == 1)) ? 3 : 0; }

// OPT: octets of a lane; G: see row_sum; SC: kind of scales
template <typename T, int OPT, int G, int SC>
__global__ void __launch_bounds__(G == 0 ? kMaxWideThreads : kThreads, fwd_ctas<T, OPT, G, SC>())
add_norm_kernel(const FwdArgs<T> a) {
    __shared__ float2 slots[2][kMaxWideThreads / 32];
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
        float2 t[OPT][4];
        float2 ss = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            float2 r[4];
            nx[j].unpack2(t[j]);
            nr[j].unpack2(r);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                t[j][e] = __fadd2_rn(t[j][e], r[e]);
                ss = __ffma2_rn(t[j][e], t[j][e], ss);
            }
        }
        if (AHEAD) fetch(row + step);
        const float s = rsqrtf(row_sum<G>(make_float2(ss.x + ss.y, 0.f), slots[parity], 0, blockDim.x >> 5).x * inv_cols + a.eps);
        const float2 s2 = make_float2(s, s);
#pragma unroll
        for (int j = 0; j < OPT; ++j) {
            const int c = lg + j * lanes;
            const bool in = live && c < octets;
            const int64_t at = row * a.cols + static_cast<int64_t>(c) * 8;
            if (in && a.total != nullptr) Octet<T>::store2(a.total + at, t[j]);
            float2 w[4];
            gm[j].unpack2(w);
            float amax = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                t[j][e] = __fmul2_rn(__fmul2_rn(t[j][e], s2), w[e]);
                if (SC != kNoQuant) amax = fmaxf(amax, fmaxf(fabsf(t[j][e].x), fabsf(t[j][e].y)));
            }
            if (in && a.normed != nullptr) Octet<T>::store2(a.normed + at, t[j]);
            if (SC != kNoQuant) {                            // columns are whole blocks: 16 neighbouring lanes hold one
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                float inv, scale = 1.0f;
                uint32_t byte = 0;
                if (SC == kAmax) {                           // the rule of tb200_quant_act_1x128, on the unrounded n
                    // the product and the quick quotient are within 2^-22: every lane forms them, a division would cost a quarter
                    // of the kernel's instructions.
                    scale = amax * (1.0f / 448.0f);
                    inv = __fdividef(448.0f, amax);
                    if (!(amax >= kLeastAmax && amax <= kMostAmax)) inv = far_factor(amax, &scale, t[j]);      // the block's 16 lanes alike
                } else {
                    byte = pow2_scale(amax, &inv);
                }
                const float2 inv2 = make_float2(inv, inv);
#pragma unroll
                for (int e = 0; e < 4; ++e) t[j][e] = __fmul2_rn(t[j][e], inv2);
                if (in) {
                    *reinterpret_cast<uint2*>(a.q + (at >> 2)) =
                        make_uint2(pack_e4m3x4(t[j][0].x, t[j][0].y, t[j][1].x, t[j][1].y), pack_e4m3x4(t[j][2].x, t[j][2].y, t[j][3].x, t[j][3].y));
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

// How many rows a thread has on their way: cp.async into slots of its own, 100 KB of a CTA at most (two on an SM) where that is
// two rows or more, else what one CTA has.
template <int PPL, int G>
constexpr int bwd_stage_bytes() { return (G == 1 ? kMaxWideThreads : kThreads) * PPL * 48; }
template <int PPL, int G>
constexpr int bwd_stages() {
    const int stage = bwd_stage_bytes<PPL, G>();
    const int two = 100 * 1024 / stage, one = 200 * 1024 / stage;
    return two >= 4 ? 4 : (two >= 2 ? two : (one >= 2 ? 2 : 1));
}
template <int N>
__device__ __forceinline__ void async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// PPL: 16-byte pieces of a row for a lane (neighbouring lanes hold neighbouring pieces).  G: lanes of a row (half a warp or a
// warp), 0: as many warps as it takes, several rows a CTA where there is room, 1: the same of up to 512 threads.
//
// With p = sum(g t) the gradient is d = s (g - t s^2 p / cols) + dt, so that both sums of a row are formed in one go and the row
// is reduced once.  What keeps HBM busy are the bytes on their way, and registers for the next row's pieces leave too few
// warps: every thread copies its pieces of the next rows into shared memory ahead of their turn (cp.async, read back by the
// thread that asked for them, so that nothing waits for another thread) and reads them where they are used.  65536 x 512 bf16
// took 61 us with the next row in registers, 46 so (with packed arithmetic and the single reduction): 5.8 TB/s.
template <typename T, int PPL, int G>
__global__ void __launch_bounds__(G == 1 ? kMaxWideThreads : kThreads, bwd_stages<PPL, G>() * bwd_stage_bytes<PPL, G>() > 100 * 1024 ? 1 : 2)
add_norm_bwd_kernel(const BwdArgs<T> a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 slots[2][kMaxWideThreads / 32];
    constexpr int S = bwd_stages<PPL, G>(), N = Vec16<T>::N, H = N / 2;
    chain_release();
    chain_wait();
    const int pieces = a.cols / N;
    const int lanes = G <= 1 ? ((pieces + PPL - 1) / PPL + 31) / 32 * 32 : G;      // of a row
    const int groups = static_cast<int>(blockDim.x) / lanes, group = static_cast<int>(threadIdx.x) / lanes;
    const int lg = static_cast<int>(threadIdx.x) - group * lanes;
    const int warp0 = group * lanes / 32, warps = lanes / 32;                      // G <= 1: the group's
    const float inv_cols = 1.0f / static_cast<float>(a.cols);
    uint4 gm[PPL];
    float2 aw[PPL][H];
#pragma unroll
    for (int j = 0; j < PPL; ++j) {
        gm[j] = lg + j * lanes < pieces ? __ldg(reinterpret_cast<const uint4*>(a.gamma) + lg + j * lanes) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < H; ++e) aw[j][e] = make_float2(0.f, 0.f);
    }
    // piece j of tensor w (total, d_normed, d_total) in a stage
    const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16, pitch = blockDim.x * 16;
    auto slot = [&](int stage, int w, int j) { return base + ((stage * 3 + w) * PPL + j) * pitch; };
    auto ask = [&](int64_t row, int stage) {
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            const int c = lg + j * lanes;
            const bool in = row < a.rows && c < pieces;
            const int64_t at = in ? row * a.cols + static_cast<int64_t>(c) * N : 0;
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                const T* from = (w == 0 ? a.total : (w == 1 ? a.dn : (a.dt != nullptr ? a.dt : a.dn))) + at;
                const int bytes = in && (w < 2 || a.dt != nullptr) ? 16 : 0;       // the rest is filled with zeros
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot(stage, w, j)), "l"(from), "r"(bytes) : "memory");
            }
        }
    };
    auto get = [&](int stage, int w, int j, float2 (&f)[H]) {
        uint4 v;      // volatile: read again in the second half instead of held over the reduction
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(slot(stage, w, j)));
        Vec16<T>::unpack2(v, f);
    };
    // a warp's lanes walk the same number of rows: the shuffles name all of them
    const int64_t step = static_cast<int64_t>(gridDim.x) * groups;
    const int64_t uneven = G == 16 ? group & 1 : 0;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * groups + group;
#pragma unroll
    for (int k = 0; k < S - 1; ++k) {
        ask(first + k * step, k);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int parity = 0, stage = 0;
    for (int64_t row = first; row - uneven < a.rows; row += step, parity ^= 1) {
        // the slots of the row before this one are free
        ask(row + (S - 1) * step, stage == 0 ? S - 1 : stage - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        async_wait<S - 1>();
        float2 ss = make_float2(0.f, 0.f), gt = ss;
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            float2 t[H], n[H], w[H];
            get(stage, 0, j, t);
            get(stage, 1, j, n);
            Vec16<T>::unpack2(gm[j], w);
#pragma unroll
            for (int e = 0; e < H; ++e) {
                ss = __ffma2_rn(t[e], t[e], ss);
                gt = __ffma2_rn(__fmul2_rn(n[e], w[e]), t[e], gt);
            }
        }
        const float2 sums = row_sum<G <= 1 ? 0 : G>(make_float2(ss.x + ss.y, gt.x + gt.y), slots[parity], warp0, warps);
        // without a row (half of a last warp) s is 1, so that nothing is added to dw: with eps = 0 it would be 0 x infinity
        const float s = rsqrtf(sums.x * inv_cols + (G == 16 && row >= a.rows ? 1.0f : a.eps));
        const float2 s2 = make_float2(s, s), k2 = make_float2(-(s * s) * (sums.y * inv_cols), -(s * s) * (sums.y * inv_cols));
#pragma unroll
        for (int j = 0; j < PPL; ++j) {
            const int c = lg + j * lanes;
            float2 t[H], n[H], w[H], o[H];
            get(stage, 0, j, t);
            get(stage, 1, j, n);
            get(stage, 2, j, o);
            asm volatile("" : "+r"(gm[j].x), "+r"(gm[j].y), "+r"(gm[j].z), "+r"(gm[j].w));      // unpacked again, not held
            Vec16<T>::unpack2(gm[j], w);
#pragma unroll
            for (int e = 0; e < H; ++e) {
                aw[j][e] = __ffma2_rn(n[e], __fmul2_rn(t[e], s2), aw[j][e]);
                o[e] = __ffma2_rn(s2, __ffma2_rn(t[e], k2, __fmul2_rn(n[e], w[e])), o[e]);
            }
            if (row < a.rows && c < pieces) *reinterpret_cast<uint4*>(a.d + row * a.cols + static_cast<int64_t>(c) * N) = Vec16<T>::pack2(o);
        }
        if (++stage == S) stage = 0;
    }
    async_wait<0>();
    __syncthreads();                      // the slots become the CTA's sums
    // the CTA's partial sums of dw: its groups in order
    float* red = reinterpret_cast<float*>(smem);
    float* out = a.partial + static_cast<int64_t>(blockIdx.x) * a.cols;
    float* mine = groups > 1 ? red + group * a.cols : out;
#pragma unroll
    for (int j = 0; j < PPL; ++j) {
        const int c = lg + j * lanes;
        if (c < pieces) {
#pragma unroll
            for (int e = 0; e < H; e += 2)
                *reinterpret_cast<float4*>(mine + c * N + 2 * e) = make_float4(aw[j][e].x, aw[j][e].y, aw[j][e + 1].x, aw[j][e + 1].y);
        }
    }
    if (groups == 1) return;
    __syncthreads();
    for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
        float w = 0.f;
        for (int k = 0; k < groups; ++k) w += red[k * a.cols + i];
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
    if (i < cols) {
#pragma unroll 8
        for (int p = ty; p < n_partials; p += 32) w += __ldcg(partial + static_cast<int64_t>(p) * cols + i);
    }
    sums[ty][tx] = w;
    __syncthreads();
    if (ty == 0 && i < cols) {
        w = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) w += sums[k][tx];
        dgamma[i] = from_float<T>(w);
    }
}

// How a row of `octets` is laid over lanes
struct Shape {
    int g, opt, threads, rows_per_cta;      // opt: octets (backward: 16-byte pieces) of a lane
};
// half a warp, a warp with up to four octets a lane, or a CTA
Shape fwd_shape(int octets) {
    if (octets <= 16) return {16, 1, kThreads, 2 * kWarps};
    if (octets <= 128) return {32, (octets + 31) / 32, kThreads, kWarps};
    const int opt = octets <= 256 ? 1 : (octets <= 512 ? 2 : 4);
    return {0, opt, ((octets + opt - 1) / opt + 31) / 32 * 32, 1};
}
// Half a warp, a warp with one or two pieces a lane, or several warps with two at least: with one piece a thread the barrier of a
// row comes too often (65536 x 640 bf16: 118 us, 1024 columns 40000 rows 73).
Shape bwd_shape(int pieces) {
    if (pieces <= 16) return {16, 1, kThreads, 2 * kWarps};
    if (pieces <= 64) return {32, (pieces + 31) / 32, kThreads, kWarps};
    int per = pieces <= 2 * kThreads ? 2 : 4;
    if (pieces > per * kMaxWideThreads) per = 8;
    const int lanes = ((pieces + per - 1) / per + 31) / 32 * 32;
    const int rows = lanes > kThreads / 2 ? 1 : kThreads / lanes;
    return {lanes > kThreads ? 1 : 0, per, rows * lanes, rows};
}
constexpr int kBwdCtas = 4;      // CTAs of an SM at most

int grid_of(int64_t rows, int rows_per_cta, int per_sm) {
    int64_t ctas = (rows + rows_per_cta - 1) / rows_per_cta;
    const int64_t cap = static_cast<int64_t>(device_info().sm_count) * per_sm;
    if (ctas > cap) ctas = cap;
    return ctas < 1 ? 1 : static_cast<int>(ctas);
}

template <typename T, int SC>
void launch_fwd(const FwdArgs<T>& a, cudaStream_t st) {
    const Shape sh = fwd_shape(a.cols >> 3);
    const int grid = grid_of(a.rows, sh.rows_per_cta, sh.g == 0 ? 16 : 8);
#define TB200_AN_FWD(OPT, G) launch_chained(add_norm_kernel<T, OPT, G, SC>, grid, sh.threads, 0, st, a)
    switch (sh.g * 8 + sh.opt) {
        case 16 * 8 + 1: TB200_AN_FWD(1, 16); break;
        case 32 * 8 + 1: TB200_AN_FWD(1, 32); break;
        case 32 * 8 + 2: TB200_AN_FWD(2, 32); break;
        case 32 * 8 + 3: TB200_AN_FWD(3, 32); break;
        case 32 * 8 + 4: TB200_AN_FWD(4, 32); break;
        case 1: TB200_AN_FWD(1, 0); break;
        case 2: TB200_AN_FWD(2, 0); break;
        default: TB200_AN_FWD(4, 0); break;
    }
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

// -> the number of CTAs: rows of the partial table
template <typename T, int PPL, int G>
int launch_bwd(const BwdArgs<T>& a, const Shape& sh, cudaStream_t st) {
    const size_t smem = static_cast<size_t>(bwd_stages<PPL, G>()) * sh.threads * PPL * 48;
    static bool attr_set[64] = {};
    const DeviceInfo& dev = device_info();
    if (!attr_set[dev.index]) {
        cudaFuncSetAttribute(add_norm_bwd_kernel<T, PPL, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        attr_set[dev.index] = true;
    }
    int per_sm = static_cast<int>(224 * 1024 / (smem + 2048));
    const int by_registers = 512 / sh.threads;                       // 128 a thread
    if (per_sm > by_registers) per_sm = by_registers;
    if (per_sm > kBwdCtas) per_sm = kBwdCtas;
    if (per_sm < 1) per_sm = 1;
    const int grid = grid_of(a.rows, sh.rows_per_cta, per_sm);
    launch_chained(add_norm_bwd_kernel<T, PPL, G>, grid, sh.threads, smem, st, a);
    return grid;
}

template <typename T>
int bwd(const void* total, const void* gamma, const void* dn, const void* dt, void* d, void* dgamma, float* work, int64_t rows, int32_t cols,
        float eps, cudaStream_t st) {
    const BwdArgs<T> a{static_cast<const T*>(total), static_cast<const T*>(gamma), static_cast<const T*>(dn), static_cast<const T*>(dt),
                       static_cast<T*>(d), work, rows, cols, eps};
    const Shape sh = bwd_shape(cols / Vec16<T>::N);
    int grid = 0;
    if (rows > 0) {
        switch (sh.g * 16 + sh.opt) {
            case 16 * 16 + 1: grid = launch_bwd<T, 1, 16>(a, sh, st); break;
            case 32 * 16 + 1: grid = launch_bwd<T, 1, 32>(a, sh, st); break;
            case 32 * 16 + 2: grid = launch_bwd<T, 2, 32>(a, sh, st); break;
            case 2: grid = launch_bwd<T, 2, 0>(a, sh, st); break;
            case 4: grid = launch_bwd<T, 4, 0>(a, sh, st); break;
            case 16 + 4: grid = launch_bwd<T, 4, 1>(a, sh, st); break;
            default: grid = launch_bwd<T, 8, 1>(a, sh, st); break;
        }
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
    using namespace tb200;
    if (cols < 1) return 0;
    const int sms = device_info().valid ? device_info().sm_count : 148;
    return static_cast<int64_t>(sms) * kBwdCtas * cols * static_cast<int64_t>(sizeof(float));
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
