// Root-mean-square norm with the residual's addition in front and, on request, its result in 8 bits with a scale per row and 128
// channels; and the quantisers for rows that no such norm wrote.
//   s = x + residual (rounded to the storage type once: what is stored is what is normalised)
//   y = s * (mean(s^2) + eps)^-1/2 * weight,  in float32, rounded once: to the storage type, or straight to e4m3 under the
//   block's scale (a rounding to bfloat16 in between would move one value in 16 by a step of e4m3)
// A warp reads a block of 128 channels at once, four channels a lane: a block's largest magnitude is one warp reduction, its
// 8-bit result one 128-byte store.  All kernels are bound by memory: every input is read once, into registers, however
// often it is used.
#include "common.cuh"
#include "fp8.cuh"

namespace convnn {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;

struct NormParams {
    const void *x, *residual, *weight;
    void *sum, *y;                      // sum: with a residual; y, or the 8-bit result:
    uint8_t* q;
    float* scales;
    long long ldx, ldr, lds, ldy, scale_row, scale_block;
    long long rows;
    int D;
    float eps, inv_d;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A lane has four neighbouring channels of the block that starts at channel c0, read and written at once (VEC: D a multiple of four
// and every row on a boundary of four values) or one by one: the sums, and so the results, are the same bits either way.
template <typename T> struct Raw4;
template <> struct Raw4<float> { float4 v; };
template <> struct Raw4<__nv_bfloat16> { uint2 v; };

template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* row, int c0, int lane, int D, float (&v)[4]) {
    if (VEC) {
        v[0] = v[1] = v[2] = v[3] = 0.f;
        if (c0 + 4 * lane < D) {
            const Raw4<T> r = *reinterpret_cast<const Raw4<T>*>(row + c0 + 4 * lane);
            const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = to_f32<T>(e[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + 4 * lane + j;
            v[j] = c < D ? to_f32<T>(row[c]) : 0.f;
        }
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T* row, int c0, int lane, int D, const float (&v)[4]) {
    if (VEC) {
        if (c0 + 4 * lane < D) {
            Raw4<T> r;
            T* e = reinterpret_cast<T*>(&r);
#pragma unroll
            for (int j = 0; j < 4; ++j) e[j] = from_f32<T>(v[j]);
            *reinterpret_cast<Raw4<T>*>(row + c0 + 4 * lane) = r;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + 4 * lane + j;
            if (c < D) row[c] = from_f32<T>(v[j]);
        }
    }
}
// The warp's block v under its scale, which is returned.
template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int c0, int lane, int D, const float (&v)[4], float scale) {
    const float inv = __frcp_rn(scale);
    const uint32_t w = e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    if (VEC) {
        if (c0 + 4 * lane < D) *reinterpret_cast<uint32_t*>(row + c0 + 4 * lane) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = c0 + 4 * lane + j;
            if (c < D) row[c] = (uint8_t)(w >> (8 * j));
        }
    }
}
__device__ __forceinline__ uint32_t amax4(const float (&v)[4]) {
    return max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
}

// x + residual as it is stored.
template <typename T, bool VEC>
__device__ __forceinline__ void load_sum(const NormParams& p, long long row, int c0, int lane, float (&v)[4]) {
    load4<T, VEC>(static_cast<const T*>(p.x) + row * p.ldx, c0, lane, p.D, v);
    if (p.residual) {
        float r[4];
        load4<T, VEC>(static_cast<const T*>(p.residual) + row * p.ldr, c0, lane, p.D, r);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_f32<T>(from_f32<T>(v[j] + r[j]));
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void finish_block(const NormParams& p, long long row, int b, int lane, const float (&v)[4],
                                             const float (&w)[4], float rstd) {
    const int c0 = b * kFp8Block;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = v[j] * rstd * w[j];
    if (p.q) {
        const float scale = fp8_scale(__reduce_max_sync(0xffffffffu, amax4(y)));
        store_e4m3<VEC>(p.q + row * p.ldy, c0, lane, p.D, y, scale);
        if (lane == 0) p.scales[row * p.scale_row + b * p.scale_block] = scale;
    } else {
        store4<T, VEC>(static_cast<T*>(p.y) + row * p.ldy, c0, lane, p.D, y);
    }
}

// WPR warps per row, each with NB blocks of it in registers; R rows at a time, where a row is short.
template <typename T, int NB, int R, int WPR, bool VEC>
__global__ void __launch_bounds__(kThreads) rms_norm_kernel(const NormParams p) {
    static_assert(WPR == 1 || R == 1, "rows shared by warps come one at a time");
    __shared__ float part[kWarps];
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wi = warp % WPR;
    const long long row0 = ((long long)blockIdx.x * (kWarps / WPR) + warp / WPR) * R;
    const int blocks = (p.D + kFp8Block - 1) / kFp8Block;
    float v[R][NB][4];
    float w[NB][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int b = wi + WPR * i;
            if (row0 + r < p.rows && b < blocks) load_sum<T, VEC>(p, row0 + r, b * kFp8Block, lane, v[r][i]);
            else v[r][i][0] = v[r][i][1] = v[r][i][2] = v[r][i][3] = 0.f;
        }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int b = wi + WPR * i;
        if (b < blocks) load4<T, VEC>(static_cast<const T*>(p.weight), b * kFp8Block, lane, p.D, w[i]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int b = wi + WPR * i;
            if (p.residual && row0 + r < p.rows && b < blocks)
                store4<T, VEC>(static_cast<T*>(p.sum) + (row0 + r) * p.lds, b * kFp8Block, lane, p.D, v[r][i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) ss = fmaf(v[r][i][j], v[r][i][j], ss);
        }
        ss = warp_sum(ss);
        if (WPR > 1) {
            if (lane == 0) part[warp] = ss;
            __syncthreads();
            ss = 0.f;
#pragma unroll
            for (int k = 0; k < WPR; ++k) ss += part[warp - wi + k];
        }
        const float rstd = rsqrtf(ss * p.inv_d + p.eps);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int b = wi + WPR * i;
            if (row0 + r < p.rows && b < blocks) finish_block<T, VEC>(p, row0 + r, b, lane, v[r][i], w[i], rstd);
        }
    }
}

// Rows that do not fit in a CTA's registers: read twice.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) rms_norm_wide_kernel(const NormParams p) {
    __shared__ float part[kWarps];
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = blockIdx.x;
    const int blocks = (p.D + kFp8Block - 1) / kFp8Block;
    float ss = 0.f;
    for (int b = warp; b < blocks; b += kWarps) {
        float v[4];
        load_sum<T, VEC>(p, row, b * kFp8Block, lane, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(v[j], v[j], ss);
    }
    ss = warp_sum(ss);
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) ss += part[k];
    const float rstd = rsqrtf(ss * p.inv_d + p.eps);
    for (int b = warp; b < blocks; b += kWarps) {
        float v[4], w[4];
        load_sum<T, VEC>(p, row, b * kFp8Block, lane, v);
        if (p.residual) store4<T, VEC>(static_cast<T*>(p.sum) + row * p.lds, b * kFp8Block, lane, p.D, v);
        load4<T, VEC>(static_cast<const T*>(p.weight), b * kFp8Block, lane, p.D, w);
        finish_block<T, VEC>(p, row, b, lane, v, w, rstd);
    }
}

struct QuantParams {
    const void* x;
    uint8_t* q;
    float* scales;
    long long ldx, ldq, scale_row, scale_block, rows;
    int D;
};

// A scale per row and block: a warp takes eight blocks of the flattened (row, block) list, all requested before the first is
// used.
constexpr int kTasks = 8;
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantParams p) {
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = (p.D + kFp8Block - 1) / kFp8Block;
    const long long t0 = ((long long)blockIdx.x * kWarps + warp) * kTasks;
    const long long first = t0 / blocks;
    float v[kTasks][4];
    long long row = first;
    int b = (int)(t0 - first * blocks);
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        if (row < p.rows) load4<T, VEC>(static_cast<const T*>(p.x) + row * p.ldx, b * kFp8Block, lane, p.D, v[t]);
        if (++b == blocks) { b = 0; ++row; }
    }
    row = first;
    b = (int)(t0 - first * blocks);
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        if (row < p.rows) {
            const float scale = fp8_scale(__reduce_max_sync(0xffffffffu, amax4(v[t])));
            store_e4m3<VEC>(p.q + row * p.ldq, b * kFp8Block, lane, p.D, v[t], scale);
            if (lane == 0) p.scales[row * p.scale_row + b * p.scale_block] = scale;
        }
        if (++b == blocks) { b = 0; ++row; }
    }
}

// A scale per 128 x 128 block: a CTA holds the block in registers, sixteen rows a warp.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const QuantParams p) {
    __shared__ uint32_t top[kWarps];
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = (p.D + kFp8Block - 1) / kFp8Block;
    const long long rb = blockIdx.x / blocks;
    const int b = (int)(blockIdx.x - rb * blocks), c0 = b * kFp8Block;
    constexpr int N = kFp8Block / kWarps;
    float v[N][4];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const long long row = rb * kFp8Block + warp + kWarps * i;
        if (row < p.rows) load4<T, VEC>(static_cast<const T*>(p.x) + row * p.ldx, c0, lane, p.D, v[i]);
        else v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, amax4(v[i]));
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) top[warp] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) m = max(m, top[k]);
    const float scale = fp8_scale(m);
    if (threadIdx.x == 0) p.scales[rb * p.scale_row + b * p.scale_block] = scale;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const long long row = rb * kFp8Block + warp + kWarps * i;
        if (row < p.rows) store_e4m3<VEC>(p.q + row * p.ldq, c0, lane, p.D, v[i], scale);
    }
}

// Whether rows of `elt`-byte values can be read four at a time.
bool fours(const void* p, long long ld, size_t elt) {
    return ld % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & (4 * elt - 1)) == 0;
}

template <typename T, int NB, int R, int WPR>
int launch_norm(const NormParams& p, bool vec, cudaStream_t st) {
    const long long per = (long long)(kWarps / WPR) * R, grid = (p.rows + per - 1) / per;
    if (grid > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "rms_norm: %lld rows", p.rows);
    if (vec) launch_chained(rms_norm_kernel<T, NB, R, WPR, true>, (unsigned)grid, kThreads, 0, st, p);
    else launch_chained(rms_norm_kernel<T, NB, R, WPR, false>, (unsigned)grid, kThreads, 0, st, p);
    CONVNN_CHECK_LAUNCH("rms_norm");
    return CONVNN_OK;
}

template <typename T>
int norm_of(const NormParams& p, cudaStream_t st) {
    const bool vec = p.D % 4 == 0 && fours(p.x, p.ldx, sizeof(T)) && fours(p.weight, 0, sizeof(T)) &&
                     (!p.residual || (fours(p.residual, p.ldr, sizeof(T)) && fours(p.sum, p.lds, sizeof(T)))) &&
                     (p.q ? fours(p.q, p.ldy, 1) : fours(p.y, p.ldy, sizeof(T)));
    const int blocks = (p.D + kFp8Block - 1) / kFp8Block;
    if (blocks <= 1) return launch_norm<T, 1, 8, 1>(p, vec, st);
    if (blocks <= 2) return launch_norm<T, 2, 4, 1>(p, vec, st);
    if (blocks <= 4) return launch_norm<T, 4, 2, 1>(p, vec, st);
    if (blocks <= 8) return launch_norm<T, 8, 1, 1>(p, vec, st);
    if (blocks <= 32) return launch_norm<T, 4, 1, 8>(p, vec, st);
    if (blocks <= 64) return launch_norm<T, 8, 1, 8>(p, vec, st);
    if (p.rows > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "rms_norm: %lld rows", p.rows);
    if (vec) launch_chained(rms_norm_wide_kernel<T, true>, (unsigned)p.rows, kThreads, 0, st, p);
    else launch_chained(rms_norm_wide_kernel<T, false>, (unsigned)p.rows, kThreads, 0, st, p);
    CONVNN_CHECK_LAUNCH("rms_norm");
    return CONVNN_OK;
}

template <typename T>
int quantize_of(const QuantParams& p, int block_rows, cudaStream_t st) {
    const bool vec = p.D % 4 == 0 && fours(p.x, p.ldx, sizeof(T)) && fours(p.q, p.ldq, 1);
    const long long blocks = (p.D + kFp8Block - 1) / kFp8Block;
    const long long grid = block_rows == 1 ? (p.rows * blocks + kWarps * kTasks - 1) / (kWarps * kTasks)
                                           : (p.rows + kFp8Block - 1) / kFp8Block * blocks;
    if (grid > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "quantize_fp8: %lld rows of %d", p.rows, p.D);
    if (block_rows == 1) {
        if (vec) launch_chained(quantize_rows_kernel<T, true>, (unsigned)grid, kThreads, 0, st, p);
        else launch_chained(quantize_rows_kernel<T, false>, (unsigned)grid, kThreads, 0, st, p);
    } else {
        if (vec) launch_chained(quantize_blocks_kernel<T, true>, (unsigned)grid, kThreads, 0, st, p);
        else launch_chained(quantize_blocks_kernel<T, false>, (unsigned)grid, kThreads, 0, st, p);
    }
    CONVNN_CHECK_LAUNCH("quantize_fp8");
    return CONVNN_OK;
}

}  // namespace

int launch_rms_norm(int dtype, const void* x, long long ldx, const void* residual, long long ldr, const void* weight, float eps,
                    void* sum, long long lds, void* y, void* q, long long ldy, float* scales, long long scale_row,
                    long long scale_block, long long rows, int D, cudaStream_t st) {
    NormParams p{};
    p.x = x; p.residual = residual; p.weight = weight; p.sum = sum; p.y = y;
    p.q = static_cast<uint8_t*>(q); p.scales = scales;
    p.ldx = ldx; p.ldr = ldr; p.lds = lds; p.ldy = ldy; p.scale_row = scale_row; p.scale_block = scale_block;
    p.rows = rows; p.D = D; p.eps = eps; p.inv_d = 1.0f / (float)D;
    return dtype == CONVNN_F32 ? norm_of<float>(p, st) : norm_of<__nv_bfloat16>(p, st);
}

int launch_quantize_fp8(int dtype, const void* x, long long ldx, int block_rows, void* q, long long ldq, float* scales,
                        long long scale_row, long long scale_block, long long rows, int D, cudaStream_t st) {
    QuantParams p{};
    p.x = x; p.q = static_cast<uint8_t*>(q); p.scales = scales;
    p.ldx = ldx; p.ldq = ldq; p.scale_row = scale_row; p.scale_block = scale_block; p.rows = rows; p.D = D;
    return dtype == CONVNN_F32 ? quantize_of<float>(p, block_rows, st) : quantize_of<__nv_bfloat16>(p, block_rows, st);
}

}  // namespace convnn
