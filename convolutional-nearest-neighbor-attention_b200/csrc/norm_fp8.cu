// Root-mean-square norm with the residual's addition in front and, on request, its result in 8 bits with a scale per row and 128
// channels; and the quantisers for rows that no such norm wrote.
//   s = x + residual (rounded to the storage type once: what is stored is what is normalised)
//   y = s * (mean(s^2) + eps)^-1/2 * weight,  in float32, rounded once: to the storage type, or straight to e4m3 under the
//   block's scale (a rounding to bfloat16 in between would move one value in 16 by a step of e4m3)
// A lane reads eight neighbouring channels at once, sixteen lanes a block: its largest magnitude is four exchanges, its 8-bit
// result one 128-byte store.  All kernels are bound by memory as long as their loads are all requested before the first is used (raw,
// into registers: every input is read once) and their instructions stay under about 90 per 256 channels: 131072 x 768 bfloat16 with
// residual and 8-bit result 106 us, 708 MB at 6.6 TB/s (79 % of the memory's cycles); the same with loads that branched and four
// channels a lane 366.  Rows of one vector (50432 x 192: 15.3 us, 68 MB) start and end more often than they stream.
#include "common.cuh"
#include "f32x2.cuh"
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
    bool weight16;                      // weight on a 16-byte boundary
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Eight neighbouring channels as they are stored, and as four pairs of float32.
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };

// What a lane requests of SEG lanes' 8 * SEG channels, and how it comes to its own eight.  U = 8: D a multiple of eight and rows on
// 16-byte boundaries (8-bit rows: 8), read and written eight values at a time, without a branch for a tail (which kept the loads
// from being requested together: 131072 x 768 107 -> 116 us).  Otherwise the lanes read side by side, two values at a time where D and
// the rows' starts are even, and exchange them through shared memory (`room`, 8 * 32 values a warp): 4099 x 1001 float32 26 -> 9.8 us
// against eight strided reads and writes a lane.  The sums, and so the results, are the same bits either way.
template <typename T, int U> struct Unit;
template <> struct Unit<float, 1> { using type = uint32_t; };
template <> struct Unit<float, 2> { using type = uint2; };
template <> struct Unit<__nv_bfloat16, 1> { using type = uint16_t; };
template <> struct Unit<__nv_bfloat16, 2> { using type = uint32_t; };
template <typename T, int U> struct Held { typename Unit<T, U>::type e[8 / U]; };
template <typename T> struct Held<T, 8> { Raw8<T> raw; };

template <typename T, int U, int SEG>
__device__ __forceinline__ Held<T, U> fetch(const T* row, int c0, int lane, int D) {
    Held<T, U> h;
    if constexpr (U == 8) {
        const int c = c0 + 8 * (lane % SEG);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) h.raw.v[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            if (c < D) h.raw.v[i] = reinterpret_cast<const uint4*>(row + c)[i];
    } else {
        using E = typename Unit<T, U>::type;
#pragma unroll
        for (int j = 0; j < 8 / U; ++j) {
            const int c = c0 + U * (SEG * j + lane % SEG);
            h.e[j] = E{};
            if (c < D) h.e[j] = *reinterpret_cast<const E*>(row + c);
        }
    }
    return h;
}
template <typename T, int U, int SEG>
__device__ __forceinline__ Raw8<T> own8(const Held<T, U>& h, T* room, int lane) {
    if constexpr (U == 8) {
        return h.raw;
    } else {
        T* seg = room + lane / SEG * (8 * SEG);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8 / U; ++j) reinterpret_cast<typename Unit<T, U>::type*>(seg)[SEG * j + lane % SEG] = h.e[j];
        __syncwarp();
        return *reinterpret_cast<const Raw8<T>*>(seg + 8 * (lane % SEG));
    }
}
// 32 lanes' eight channels each from c0 on -> row.
template <typename T, int U>
__device__ __forceinline__ void store256(T* row, int c0, int lane, int D, const Raw8<T>& r, T* room) {
    if constexpr (U == 8) {
        const int c = c0 + 8 * lane;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            if (c < D) reinterpret_cast<uint4*>(row + c)[i] = r.v[i];
    } else {
        using E = typename Unit<T, U>::type;
        __syncwarp();
        *reinterpret_cast<Raw8<T>*>(room + 8 * lane) = r;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8 / U; ++j) {
            const int c = c0 + U * (32 * j + lane);
            if (c < D) *reinterpret_cast<E*>(row + c) = reinterpret_cast<const E*>(room)[32 * j + lane];
        }
    }
}
// A lane's eight of the norm's weights, which are few and stay in the caches.
template <typename T, int U>
__device__ __forceinline__ Raw8<T> weights8(const T* w, int c, int D, bool sixteen) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = make_uint4(0, 0, 0, 0);
    if (U == 8 || (sixteen && c + 8 <= D)) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            if (c < D) r.v[i] = reinterpret_cast<const uint4*>(w + c)[i];
    } else {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < D) e[j] = w[c + j];
    }
    return r;
}
__device__ __forceinline__ void widen(const Raw8<__nv_bfloat16>& r, f32x2 (&v)[4]) { bf16x8_to_f32x2(r.v[0], v); }
__device__ __forceinline__ void widen(const Raw8<float>& r, f32x2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[2 * i] = pack2(__uint_as_float(r.v[i].x), __uint_as_float(r.v[i].y));
        v[2 * i + 1] = pack2(__uint_as_float(r.v[i].z), __uint_as_float(r.v[i].w));
    }
}
__device__ __forceinline__ void narrow(const f32x2 (&v)[4], Raw8<__nv_bfloat16>& r) { r.v[0] = f32x2_to_bf16x8(v); }
__device__ __forceinline__ void narrow(const f32x2 (&v)[4], Raw8<float>& r) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float f[4];
        unpack2(v[2 * i], f[0], f[1]);
        unpack2(v[2 * i + 1], f[2], f[3]);
        r.v[i] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
}
__device__ __forceinline__ uint32_t amax8(const f32x2 (&v)[4]) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2(v[i], a, b);
        m[i] = max_nan(fabsf(a), fabsf(b));
    }
    return abs_bits(max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3])));
}
__device__ __forceinline__ uint32_t amax8(const Raw8<float>& r) {
    f32x2 v[4];
    widen(r, v);
    return amax8(v);
}
// (the magnitudes of bfloat16 values order like their bits)
__device__ __forceinline__ uint32_t amax8(const Raw8<__nv_bfloat16>& r) {
    constexpr uint32_t MAG = 0x7fff7fffu;
    const uint32_t m = __vmaxu2(__vmaxu2(r.v[0].x & MAG, r.v[0].y & MAG), __vmaxu2(r.v[0].z & MAG, r.v[0].w & MAG));
    return max(m << 16, m & 0xffff0000u);
}
// Over the sixteen lanes of a block.
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
template <int U>
__device__ __forceinline__ void store_e4m3(uint8_t* p, int valid, const f32x2 (&v)[4], float scale) {
    const float inv = __frcp_rn(scale);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2(mul2(v[i], pack2(inv, inv)), f[2 * i], f[2 * i + 1]);
    const uint2 w = make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
    if (U == 8) {
        if (valid > 0) *reinterpret_cast<uint2*>(p) = w;
    } else if (valid >= 8 && (reinterpret_cast<uintptr_t>(p) & 7u) == 0) {
        *reinterpret_cast<uint2*>(p) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < valid) p[j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
    }
}

// x + residual as it is stored, widened again.
template <typename T>
__device__ __forceinline__ Raw8<T> add_residual(const Raw8<T>& res, f32x2 (&v)[4]) {
    f32x2 r[4];
    widen(res, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = add2(v[i], r[i]);
    Raw8<T> s;
    narrow(v, s);
    widen(s, v);
    return s;
}
__device__ __forceinline__ float squares(const f32x2 (&v)[4], float ss) {
    f32x2 a = mul2(v[0], v[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) a = fma2(v[i], v[i], a);
    float x, y;
    unpack2(a, x, y);
    return ss + (x + y);
}
// The result of a warp's 256 channels from c0 on.
template <typename T, int U>
__device__ __forceinline__ void finish256(const NormParams& p, long long row, int c0, int lane, bool inside, const f32x2 (&v)[4],
                                          const f32x2 (&w)[4], float rstd, T* room) {
    f32x2 y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = mul2(mul2(v[i], pack2(rstd, rstd)), w[i]);
    if (p.q) {
        const float scale = fp8_scale(block_max(amax8(y)));
        const int c = c0 + 8 * lane, valid = inside ? p.D - c : 0;
        store_e4m3<U>(p.q + row * p.ldy + c, valid, y, scale);
        if (valid > 0 && lane % 16 == 0) p.scales[row * p.scale_row + c / kFp8Block * p.scale_block] = scale;
    } else if (inside) {
        Raw8<T> o;
        narrow(y, o);
        store256<T, U>(static_cast<T*>(p.y) + row * p.ldy, c0, lane, p.D, o, room);
    }
}

// WPR warps per row, each with NV vectors of 256 channels of it in registers; R rows at a time, where a row is short.
template <typename T, int NV, int R, int WPR, int U>
__global__ void __launch_bounds__(kThreads) rms_norm_kernel(const NormParams p) {
    static_assert(WPR == 1 || R == 1, "rows shared by warps come one at a time");
    __shared__ float part[kWarps];
    __shared__ __align__(16) T rooms[U == 8 ? 1 : kWarps][U == 8 ? 1 : 256];
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wi = warp % WPR;
    T* room = rooms[U == 8 ? 0 : warp];
    const long long row0 = ((long long)blockIdx.x * (kWarps / WPR) + warp / WPR) * R;
    const T* x = static_cast<const T*>(p.x);
    const T* res = static_cast<const T*>(p.residual);
    Held<T, U> raw[R][NV], extra[R][NV];
    Raw8<T> wr[NV];
    int c0[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) c0[i] = (wi + WPR * i) * 256;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            raw[r][i] = fetch<T, U, 32>(x + (row0 + r) * p.ldx, c0[i], lane, row0 + r < p.rows ? p.D : 0);
    if (res) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                extra[r][i] = fetch<T, U, 32>(res + (row0 + r) * p.ldr, c0[i], lane, row0 + r < p.rows ? p.D : 0);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) wr[i] = weights8<T, U>(static_cast<const T*>(p.weight), c0[i] + 8 * lane, p.D, p.weight16);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const bool inside = row0 + r < p.rows;
        f32x2 v[NV][4];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            widen(own8<T, U, 32>(raw[r][i], room, lane), v[i]);
            if (res) {
                const Raw8<T> s = add_residual<T>(own8<T, U, 32>(extra[r][i], room, lane), v[i]);
                if (inside) store256<T, U>(static_cast<T*>(p.sum) + (row0 + r) * p.lds, c0[i], lane, p.D, s, room);
            }
            ss = squares(v[i], ss);
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
        for (int i = 0; i < NV; ++i) {
            f32x2 w[4];
            widen(wr[i], w);
            finish256<T, U>(p, row0 + r, c0[i], lane, inside, v[i], w, rstd, room);
        }
    }
}

// Rows that do not fit in a CTA's registers: read twice.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) rms_norm_wide_kernel(const NormParams p) {
    __shared__ float part[kWarps];
    __shared__ __align__(16) T rooms[U == 8 ? 1 : kWarps][U == 8 ? 1 : 256];
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    T* room = rooms[U == 8 ? 0 : warp];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ldr : nullptr;
    float rstd = 0.f;
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
        float ss = 0.f;
#pragma unroll 2
        for (int c0 = warp * 256; c0 < p.D; c0 += kWarps * 256) {
            const Held<T, U> raw = fetch<T, U, 32>(x, c0, lane, p.D);
            Held<T, U> extra;
            Raw8<T> wr;
            if (res) extra = fetch<T, U, 32>(res, c0, lane, p.D);
            if (pass) wr = weights8<T, U>(static_cast<const T*>(p.weight), c0 + 8 * lane, p.D, p.weight16);
            f32x2 v[4];
            widen(own8<T, U, 32>(raw, room, lane), v);
            if (res) {
                const Raw8<T> s = add_residual<T>(own8<T, U, 32>(extra, room, lane), v);
                if (pass) store256<T, U>(static_cast<T*>(p.sum) + row * p.lds, c0, lane, p.D, s, room);
            }
            if (!pass) {
                ss = squares(v, ss);
            } else {
                f32x2 w[4];
                widen(wr, w);
                finish256<T, U>(p, row, c0, lane, true, v, w, rstd, room);
            }
        }
        if (!pass) {
            ss = warp_sum(ss);
            if (lane == 0) part[warp] = ss;
            __syncthreads();
            ss = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) ss += part[k];
            rstd = rsqrtf(ss * p.inv_d + p.eps);
        }
    }
}

struct QuantParams {
    const void* x;
    uint8_t* q;
    float* scales;
    long long ldx, ldq, scale_row, scale_block, rows;
    int D;
};

// A scale per row and block: a half-warp takes G neighbouring blocks of R rows.
template <typename T, int U, int G, int R>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantParams p, int groups) {
    __shared__ __align__(16) T rooms[U == 8 ? 1 : kWarps][U == 8 ? 1 : 256];
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, at = (lane & 15) * 8;
    T* room = rooms[U == 8 ? 0 : warp];
    const long long task = ((long long)blockIdx.x * kWarps + warp) * 2 + (lane >> 4), set = task / groups, row0 = set * R;
    const int b0 = (int)(task - set * groups) * G, c0 = b0 * kFp8Block;
    const T* x = static_cast<const T*>(p.x) + row0 * p.ldx;
    Held<T, U> held[R][G];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int g = 0; g < G; ++g)
            held[r][g] = fetch<T, U, 16>(x + r * p.ldx, c0 + g * kFp8Block, lane, row0 + r < p.rows ? p.D : 0);
    uint8_t* q = p.q + row0 * p.ldq + c0 + at;
    float* scales = p.scales + row0 * p.scale_row + b0 * p.scale_block;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const Raw8<T> raw = own8<T, U, 16>(held[r][g], room, lane);
            const float scale = fp8_scale(block_max(amax8(raw)));
            const int valid = row0 + r < p.rows ? p.D - c0 - g * kFp8Block - at : 0;
            f32x2 v[4];
            widen(raw, v);
            store_e4m3<U>(q + r * p.ldq + g * kFp8Block, valid, v, scale);
            if (valid > 0 && at == 0) scales[r * p.scale_row + g * p.scale_block] = scale;
        }
}

// A scale per 128 x 128 block: a CTA holds the block in registers, eight rows a half-warp.
template <typename T, int U>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const QuantParams p) {
    __shared__ uint32_t top[kWarps];
    __shared__ __align__(16) T rooms[U == 8 ? 1 : kWarps][U == 8 ? 1 : 256];
    chain_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    T* room = rooms[U == 8 ? 0 : warp];
    const int blocks = (p.D + kFp8Block - 1) / kFp8Block;
    const long long rb = blockIdx.x / blocks;
    const int b = (int)(blockIdx.x - rb * blocks), c = b * kFp8Block + (lane & 15) * 8;
    constexpr int N = kFp8Block / (2 * kWarps);
    const long long row0 = rb * kFp8Block + 2 * warp + (lane >> 4);
    Held<T, U> held[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const long long row = row0 + 2 * kWarps * i;
        held[i] = fetch<T, U, 16>(static_cast<const T*>(p.x) + row * p.ldx, b * kFp8Block, lane, row < p.rows ? p.D : 0);
    }
    Raw8<T> raw[N];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        raw[i] = own8<T, U, 16>(held[i], room, lane);
        m = max(m, amax8(raw[i]));
    }
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
        const long long row = row0 + 2 * kWarps * i;
        f32x2 v[4];
        widen(raw[i], v);
        store_e4m3<U>(p.q + row * p.ldq + c, row < p.rows ? p.D - c : 0, v, scale);
    }
}

bool on_boundary(const void* p, long long ld_bytes, int bytes) {
    return ld_bytes % bytes == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0;
}
template <typename T> bool rows_on(const void* p, long long ld, int bytes) { return on_boundary(p, ld * (long long)sizeof(T), bytes); }

// EIGHT: for rows of a multiple of eight channels too.
template <typename T, int NV, int R, int WPR, bool EIGHT = true>
int launch_norm(const NormParams& p, int unit, cudaStream_t st) {
    const long long per = (long long)(kWarps / WPR) * R, grid = (p.rows + per - 1) / per;
    if (grid > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "rms_norm: %lld rows", p.rows);
    if (EIGHT && unit == 8) launch_chained(rms_norm_kernel<T, NV, R, WPR, EIGHT ? 8 : 1>, (unsigned)grid, kThreads, 0, st, p);
    else if (unit == 2) launch_chained(rms_norm_kernel<T, NV, R, WPR, 2>, (unsigned)grid, kThreads, 0, st, p);
    else launch_chained(rms_norm_kernel<T, NV, R, WPR, 1>, (unsigned)grid, kThreads, 0, st, p);
    CONVNN_CHECK_LAUNCH("rms_norm");
    return CONVNN_OK;
}

template <typename T>
int norm_of(const NormParams& p, cudaStream_t st) {
    auto starts_on = [&](int bytes) {
        return rows_on<T>(p.x, p.ldx, bytes) && (!p.residual || (rows_on<T>(p.residual, p.ldr, bytes) && rows_on<T>(p.sum, p.lds, bytes))) &&
               (p.q || rows_on<T>(p.y, p.ldy, bytes));
    };
    const bool eight = p.D % 8 == 0 && starts_on(16) && p.weight16 && (!p.q || on_boundary(p.q, p.ldy, 8));
    const int unit = eight ? 8 : p.D % 2 == 0 && starts_on(2 * (int)sizeof(T)) ? 2 : 1;
    const int vectors = (p.D + 255) / 256;
    // Several rows a warp where one leaves it little to wait for: 50432 rows of 192 bfloat16 channels 16.8 us with one, 15.5 with four, 22.3
    // with eight; of 256 float32 channels 26.7, 28.6 with four; 117861 odd rows of 133 bfloat16 channels 51.7, 69.7 with four.
    if (vectors <= 1) return sizeof(T) == 2 && unit == 8 ? launch_norm<T, 1, 4, 1>(p, unit, st) : launch_norm<T, 1, 2, 1>(p, unit, st);
    if (vectors <= 2) return launch_norm<T, 2, 1, 1>(p, unit, st);
    if (vectors <= 3) return launch_norm<T, 3, 1, 1>(p, unit, st);
    // As many warps a row as leave each a few vectors and none without: bfloat16 with residual and 8-bit result, 16001 rows of 1536
    // channels 28 us in two warps, 31 in four, 38 in eight (49 in eight with room for two vectors each); of 2048 36 in four, 37 in two,
    // 42 in eight; 10001 of 2560 31 in four, 36 in eight.  float32 keeps more registers a vector (1536: 54 in two, 48 in four, 49 in
    // eight; 2048: 33 in four and eight), and rows of other channels more yet: 50001 of 1001 92 in two warps, 125 in one; 16001
    // of 1501 61 in two, 54 in four, 52 in eight; 10001 of 2501 70 in four, 64 in eight.  The choice is one by width and type, not
    // by where rows start, so that a view's results are those of its copy.
    const bool whole = p.D % 8 == 0;
    if (vectors <= 4) return whole ? launch_norm<T, 4, 1, 1>(p, unit, st) : launch_norm<T, 2, 1, 2, false>(p, unit, st);
    if constexpr (sizeof(T) == 2) {
        if (whole && vectors <= 6) return launch_norm<T, 3, 1, 2>(p, unit, st);
        if (whole && vectors <= 8) return launch_norm<T, 2, 1, 4>(p, unit, st);
        if (whole && vectors <= 12) return launch_norm<T, 3, 1, 4>(p, unit, st);
    }
    if (vectors <= 8) return launch_norm<T, 1, 1, 8, sizeof(T) == 4>(p, unit, st);
    if (vectors <= 16) return launch_norm<T, 2, 1, 8>(p, unit, st);
    // (6001 of 6144: 40 with room for three vectors a warp, 47 for four)
    if (vectors <= 24) return launch_norm<T, 3, 1, 8>(p, unit, st);
    if (vectors <= 32) return launch_norm<T, 4, 1, 8>(p, unit, st);
    if (p.rows > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "rms_norm: %lld rows", p.rows);
    if (unit == 8) launch_chained(rms_norm_wide_kernel<T, 8>, (unsigned)p.rows, kThreads, 0, st, p);
    else if (unit == 2) launch_chained(rms_norm_wide_kernel<T, 2>, (unsigned)p.rows, kThreads, 0, st, p);
    else launch_chained(rms_norm_wide_kernel<T, 1>, (unsigned)p.rows, kThreads, 0, st, p);
    CONVNN_CHECK_LAUNCH("rms_norm");
    return CONVNN_OK;
}

template <typename T, int G, int R>
int launch_quantize_rows(const QuantParams& p, int unit, cudaStream_t st) {
    const int groups = ((p.D + kFp8Block - 1) / kFp8Block + G - 1) / G;
    const long long tasks = (p.rows + R - 1) / R * groups, grid = (tasks + 2 * kWarps - 1) / (2 * kWarps);
    if (grid > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "quantize_fp8: %lld rows of %d", p.rows, p.D);
    if (unit == 8) launch_chained(quantize_rows_kernel<T, 8, G, R>, (unsigned)grid, kThreads, 0, st, p, groups);
    else if (unit == 2) launch_chained(quantize_rows_kernel<T, 2, G, R>, (unsigned)grid, kThreads, 0, st, p, groups);
    else launch_chained(quantize_rows_kernel<T, 1, G, R>, (unsigned)grid, kThreads, 0, st, p, groups);
    CONVNN_CHECK_LAUNCH("quantize_fp8");
    return CONVNN_OK;
}

template <typename T>
int quantize_of(const QuantParams& p, int block_rows, cudaStream_t st) {
    const bool eight = p.D % 8 == 0 && rows_on<T>(p.x, p.ldx, 16) && on_boundary(p.q, p.ldq, 8);
    const int unit = eight ? 8 : p.D % 2 == 0 && rows_on<T>(p.x, p.ldx, 2 * (int)sizeof(T)) ? 2 : 1;
    const int blocks = (p.D + kFp8Block - 1) / kFp8Block;
    if (block_rows == 1) {
        // three or four blocks a half-warp, whichever leaves fewer out of the last one; rows of one or two blocks, several rows
        if (blocks == 1) return launch_quantize_rows<T, 1, 4>(p, unit, st);
        if (blocks == 2) return launch_quantize_rows<T, 2, 2>(p, unit, st);
        if ((blocks + 2) / 3 * 3 < (blocks + 3) / 4 * 4) return launch_quantize_rows<T, 3, 2>(p, unit, st);
        return launch_quantize_rows<T, 4, 1>(p, unit, st);
    }
    const long long grid = (p.rows + kFp8Block - 1) / kFp8Block * blocks;
    if (grid > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "quantize_fp8: %lld rows of %d", p.rows, p.D);
    if (unit == 8) launch_chained(quantize_blocks_kernel<T, 8>, (unsigned)grid, kThreads, 0, st, p);
    else if (unit == 2) launch_chained(quantize_blocks_kernel<T, 2>, (unsigned)grid, kThreads, 0, st, p);
    else launch_chained(quantize_blocks_kernel<T, 1>, (unsigned)grid, kThreads, 0, st, p);
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
    p.weight16 = aligned16(weight);
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
