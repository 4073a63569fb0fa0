// Matrix product of 8-bit values (e4m3) with a float32 scale per row of A and block of 128 channels, and per 128 x 128 block of W:
//   out[m, n] = [gelu](sum_b sa[m, b] sw[n / 128, b] (sum_{k in b} a[m, k] w[n, k]) + bias[n]) + residual[m, n]
// The inner sums run on tcgen05 (kind::f8f6f4, 128 channels = four instructions = one row of a 128-byte-swizzled tile) into an
// accumulator of their own in TMEM, which the epilogue warps add up in registers, scaled, in ascending b, while the next block
// is multiplied into the next buffer.  The scales are any float32 values, so they cannot be the tensor cores' own powers of two.
// Everything after the sum stays in float32 until the one rounding of the store: to bfloat16, not at all, or to e4m3 under the
// scale of the row's block of 128 columns.
//
// Two kernels, by the number of tiles (see launch_linear_fp8):
//   linear_fp8_kernel: one CTA, or a cluster that shares the blocks of k, per tile of 128 x BN; few tiles
//   linear_fp8_pair_kernel: persistent CTA pairs on tiles of 256 x 256; many tiles
// Every mbarrier wait is bounded (see sm100.cuh); an expiry latches the device status.
#include "common.cuh"
#include "sm100.cuh"
#include "f32x2.cuh"
#include "fp8.cuh"

namespace convnn {

__device__ int g_linear_fp8_status = 0;   // error latch of this translation unit

namespace {

using namespace sm100;

constexpr int BP = 128;                   // rows of P in a tile
constexpr int KB = kFp8Block;             // channels (= bytes) of a block
constexpr int NTHREADS = 320;
constexpr int MAX_STAGES = 12;

enum OutKind : int { OUT_F32 = 0, OUT_BF16 = 1, OUT_E4M3 = 2 };

struct LinearFp8Params {
    const float *sa, *sw;                 // scales; strides in elements
    long long sa_row, sa_block, sw_row, sw_block;
    const void *bias, *residual;          // of `io`
    void* out;
    float* so;                            // OUT_E4M3: scales out
    long long ldr, ldo, so_row, so_block;
    int M, N, blocks;                     // blocks of k
    int out_kind, io, gelu;               // io: convnn_dtype of bias, residual (and out)
    int stages, splits;                   // CTAs of the cluster
    bool bias16, residual16, out16;       // their rows start on 16-byte boundaries
    bool out_tma;                         // and those of out end on one: a copy by TMA writes on to it, over what lies behind the last column
    bool residual4, out4;                 // on 4-byte boundaries (residual: and N is even, two bfloat16 values at a time)
};

__device__ __forceinline__ void fail(volatile int* abort_flag, int code) {
    *abort_flag = 1;
    atomicCAS(&g_linear_fp8_status, 0, code);
}

// D format F32 (bit 4), A / B format E4M3 (0 in bits 7-9, 10-12), N >> 3 in bits 17-22, M >> 4 in bits 24-28.
__host__ __device__ constexpr uint32_t idesc_e4m3_f32(int M, int N) {
    return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void mma_e4m3_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

// x * Phi(x), for results that stay in float32.
__device__ __forceinline__ float gelu_erf(float x) { return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f)); }
// The same for results of 8 or 16 bits: max(x, 0) - a Q(a) with a = |x| and Q = 1 - Phi = exp(-a^2 / 2) R(a), R the polynomial of degree 7
// in t = 1 / (1 + 0.35 a) that comes nearest to erfcx(a / sqrt 2) / 2 on [0, 13.5] relative to it (Hastings' form, fitted by
// weighted least squares: 3.1e-7).  Q is off by 2^-19 + a^2 2^-24 of itself at most as it is evaluated here, so that a block of 128
// channels that lies wholly in the tail has its own scale and values (an approximation near in absolute terms does not: a polynomial of
// degree 14 within 1.1e-7 of Q was 3 % off at -4.5 and constant below -5).  Below -13.2 the result is zero; -inf gives NaN as the
// formula does, since the positive part is made as x / 2 + |x| / 2.
// Four pairs side by side, in an order that the compiler keeps: it strings single instructions up value by value, each waiting for
// the last.  A value's two approximations (16 cycles of a warp's scheduler) run beside its 14 multiply-adds: 50432 x 768 x 192 into 8 bits
// 52.0 us, 51.4 with that polynomial; one reciprocal for two values 53.5.
__device__ __forceinline__ f32x2 fma2_here(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2_here(f32x2 a, f32x2 b) {
    f32x2 r;
    asm volatile("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float rcp_here(float x) {
    float r;
    asm volatile("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float ex2_here(float x) {
    float r;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void gelu8(float* x) {
    constexpr float C[8] = {2.73154092e-05f, -0.140270337f, -0.133355111f, -0.155961424f, 0.0170232989f,
                            -0.240640655f, 0.202119172f, -0.0489424132f};
    f32x2 a[4], t[4], e[4], q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = pack2(fminf(fabsf(x[2 * j]), 14.0f), fminf(fabsf(x[2 * j + 1]), 14.0f));
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = fma2_here(a[j], pack2(0.35f, 0.35f), pack2(1.0f, 1.0f));
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = mul2_here(mul2(a[j], pack2(-0.72134752f, -0.72134752f)), a[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float u, v;
        unpack2(t[j], u, v);
        t[j] = pack2(rcp_here(u), rcp_here(v));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = fma2_here(t[j], pack2(C[7], C[7]), pack2(C[6], C[6]));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float u, v;
        unpack2(e[j], u, v);
        e[j] = pack2(ex2_here(u), ex2_here(v));
    }
#pragma unroll
    for (int i = 5; i >= 0; --i)
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = fma2_here(q[j], t[j], pack2(C[i], C[i]));
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = mul2_here(q[j], e[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float u = 0.5f * x[2 * j], v = 0.5f * x[2 * j + 1];
        unpack2(fma2_here(a[j], q[j], pack2(u + fabsf(u), v + fabsf(v))), x[2 * j], x[2 * j + 1]);
    }
}

// Eight values of a row from column n on: neighbours, 16 bytes at a time where `vec` and all are inside, or one by one, `step` apart.
template <typename T> struct Eight { uint4 v[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Eight<T> load8(const void* base, long long at, int left, int step, bool vec) {
    const T* p = static_cast<const T*>(base) + at;
    Eight<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = make_uint4(0, 0, 0, 0);
    if (vec && left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j * step < left) e[j] = p[j * step];
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store8(void* base, long long at, int left, int step, bool vec, const float (&v)[8]) {
    T* p = static_cast<T*>(base) + at;
    if (vec && left >= 8) {
        Eight<T> r;
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = from_f32<T>(v[j]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.v[i];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j * step < left) p[j * step] = from_f32<T>(v[j]);
    }
}
template <typename T>
__device__ __forceinline__ void add8(float (&v)[8], const Eight<T>& r) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += to_f32<T>(e[j]);
}

// Eight outputs of row m from column n on, `step` apart, `left` columns before the end (<= 0: none); `sum` gives their sums, which are
// asked for after the bias and the residual.  Sixteen neighbouring lanes hold a row's block of 128 columns and come here together.
template <typename IO, typename Sum>
__device__ __forceinline__ void finish8(const LinearFp8Params& p, long long m, int n, int left, int step, const Sum& sum) {
    Eight<IO> bias, residual;
    const bool near = step == 1;
    if (p.bias) bias = load8<IO>(p.bias, n, left, step, p.bias16 && near);
    if (p.residual) residual = load8<IO>(p.residual, m * p.ldr + n, left, step, p.residual16 && near);
    float v[8];
    sum(v);
    if (p.bias) add8<IO>(v, bias);
    if (p.gelu && p.out_kind == OUT_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = gelu_erf(v[j]);
    } else if (p.gelu) {
        gelu8(v);
    }
    if (p.residual) add8<IO>(v, residual);
    if (p.out_kind == OUT_E4M3) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) top = max(top, abs_bits(v[j]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float scale = fp8_scale(top), inv = __frcp_rn(scale);
        if (left > 0) {
            uint2 w;
            w.x = e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
            w.y = e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
            uint8_t* q = static_cast<uint8_t*>(p.out) + m * p.ldo + n;
            if (p.out16 && left >= 8) *reinterpret_cast<uint2*>(q) = w;
            else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) q[j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
            }
            if (n % KB == 0) p.so[m * p.so_row + (n / KB) * p.so_block] = scale;
        }
    } else if (left > 0) {
        store8<IO>(p.out, m * p.ldo + n, left, step, p.out16 && near, v);
    }
}

// Tiles of 128 x BN: 128 rows of P, whose rows are TMEM lanes, times BN rows of Q.  P are the activations and BN = 128 (more rows),
// or P are the weights and Q 16, 32 or 64 tokens (SWAP).  Where tiles are few the CTAs of a cluster share a tile's blocks of k;
// their partial tiles, in shared memory, are added up in rank order.
//   warp 0     TMA producer (ring of P and Q blocks)
//   warp 1     MMA issuer
//   warps 2-9  scaled sums (two warps per lane quarter, half of the columns each), then with the others the output
template <int BN, bool SWAP>
__global__ void __launch_bounds__(NTHREADS, BN >= 64 ? 2 : 1)
linear_fp8_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, const LinearFp8Params p) {
    static_assert(SWAP ? BN <= 64 : BN == 128, "see the scales of the two forms");
    constexpr int CW = BN / 2;                               // columns of a warp
    constexpr int NBUF = BN == 128 ? 2 : 4;
    constexpr uint32_t TCOLS = NBUF * BN < 32 ? 32 : NBUF * BN;
    constexpr int AHEAD = 4;                                 // scales requested so many blocks before their use
    // the summed tile, rows of the output by its columns
    constexpr int ROWS = SWAP ? BN : BP, COLS = SWAP ? BP : BN, PITCH = COLS + 4;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr uint32_t P_BYTES = BP * KB, Q_BYTES = BN * KB;
    const uint32_t STAGES = p.stages;
    uint8_t* sP = smem;
    uint8_t* sQ = sP + STAGES * P_BYTES;
    float* tile = reinterpret_cast<float*>(smem);            // in the place of the ring, once that is read
    __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], tfull[NBUF], tempty[NBUF];
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t counts[2];                           // blocks of k asked for, and multiplied
    __shared__ int abort_word;
    __shared__ __align__(16) float col_scale[SWAP ? 8 : 1][2][SWAP ? 32 : 1];
    volatile int* abort_flag = &abort_word;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = p.splits > 1 ? (int)cluster_ctarank() : 0;
    const int unit = blockIdx.x / p.splits;
    // tiles of one block of weights after another, or of one block of rows after another
    const int n_q = SWAP ? (p.M + BN - 1) / BN : (p.N + BN - 1) / BN;
    const int pt = unit / n_q, qt = unit - pt * n_q;
    const int kb0 = (int)((long long)p.blocks * rank / p.splits), kb1 = (int)((long long)p.blocks * (rank + 1) / p.splits);

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < NBUF; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 8); }
        abort_word = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmP);
        prefetch_tensormap(&tmQ);
    }
    if (warp == 1) { tmem_alloc(&tmem_slot, TCOLS); tmem_relinquish(); }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    chain_begin();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            int kb = kb0;
            for (; kb < kb1; ++kb) {
                if (!mbar_wait(&empty[s], ph ^ 1u, abort_flag)) { fail(abort_flag, 121); break; }
                mbar_expect_tx(&full[s], P_BYTES + Q_BYTES);
                tma_load_2d(sP + s * P_BYTES, &tmP, &full[s], kb * KB, pt * BP);
                tma_load_2d(sQ + s * Q_BYTES, &tmQ, &full[s], kb * KB, qt * BN);
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
            counts[0] = (uint32_t)(kb - kb0);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_e4m3_f32(BP, BN);
        const uint64_t hi = kmajor_desc_hi(KB);
        const uint32_t full0 = smem_u32(full), tempty0 = smem_u32(tempty), empty0 = smem_u32(empty), tfull0 = smem_u32(tfull);
        const uint32_t sP0 = smem_u32(sP), sQ0 = smem_u32(sQ);
        uint32_t s = 0, ph = 0, buf = 0, tph = 0;
        int kb = kb0;
        for (; kb < kb1; ++kb) {
            if (!mbar_wait_warp(tempty0 + 8 * buf, tph ^ 1u, abort_flag)) { if (lane == 0) fail(abort_flag, 122); break; }
            if (!mbar_wait_warp(full0 + 8 * s, ph, abort_flag)) { if (lane == 0) fail(abort_flag, 123); break; }
            tc_fence_after_sync();
            if (elect_one()) {
                const uint64_t ad = hi | (uint64_t)(((sP0 + s * P_BYTES) & 0x3FFFFu) >> 4);
                const uint64_t bd = hi | (uint64_t)(((sQ0 + s * Q_BYTES) & 0x3FFFFu) >> 4);
                const uint32_t d = tmem_base + buf * BN;
#pragma unroll
                for (int i = 0; i < 4; ++i) mma_e4m3_ss(d, ad + 2 * i, bd + 2 * i, idesc, i > 0);
                mma_commit_a(empty0 + 8 * s);
                mma_commit_a(tfull0 + 8 * buf);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1u; }
            if (++buf == NBUF) { buf = 0; tph ^= 1u; }
        }
        if (lane == 0) counts[1] = (uint32_t)(kb - kb0);
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;   // (a warp reads the TMEM lanes of its number mod 4)
        const int c0 = half * CW, row = quarter * 32 + lane;
        f32x2 acc[CW / 2];
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) acc[j] = pack2(0.f, 0.f);
        // The scale of this lane's row (its column, where SWAP) times the one that the whole tile shares.  Rows past the end hold
        // zeros and are never stored.
        const int mine = SWAP ? qt * BN + c0 + lane : pt * BP + row;
        const bool have = mine < p.M && (!SWAP || lane < CW);
        const float* sa = p.sa + (have ? (long long)mine * p.sa_row : 0);
        const float* sw = p.sw + (long long)(SWAP ? pt : qt) * p.sw_row;
        auto scale_of = [&](int kb) {
            if (!have || kb >= kb1) return 0.f;
            return sa[kb * p.sa_block] * sw[kb * p.sw_block];
        };
        float next[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) next[i] = scale_of(kb0 + i);
        uint32_t buf = 0, tph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            const float s = next[0];
#pragma unroll
            for (int i = 0; i + 1 < AHEAD; ++i) next[i] = next[i + 1];
            next[AHEAD - 1] = scale_of(kb + AHEAD);
            float* sc = SWAP ? col_scale[warp - 2][kb & 1] : nullptr;
            if (SWAP) {
                sc[lane] = s;
                __syncwarp();
            }
            if (!__all_sync(0xffffffffu, mbar_wait(&tfull[buf], tph, abort_flag))) { if (lane == 0) fail(abort_flag, 124); break; }
            tc_fence_after_sync();
            const uint32_t t = tmem_base + buf * BN + c0 + ((uint32_t)(quarter * 32) << 16);
            constexpr int STEP = CW < 16 ? CW : 16;
#pragma unroll
            for (int c = 0; c < CW; c += STEP) {
                uint32_t r[STEP];
                if constexpr (STEP == 8) tmem_ld_x8(t + c, r);
                else tmem_ld_x16(t + c, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < STEP; j += 2) {
                    const f32x2 part = pack2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
                    const f32x2 by = SWAP ? *reinterpret_cast<const f32x2*>(sc + c + j) : pack2(s, s);
                    acc[(c + j) / 2] = fma2(part, by, acc[(c + j) / 2]);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[buf]);
            if (++buf == NBUF) { buf = 0; tph ^= 1u; }
        }
        // The last product has read the ring, and nothing more is copied into it.
#pragma unroll
        for (int j = 0; j < CW / 2; ++j) {
            float a, b;
            unpack2(acc[j], a, b);
            if (SWAP) {
                tile[(c0 + 2 * j) * PITCH + row] = a;
                tile[(c0 + 2 * j + 1) * PITCH + row] = b;
            } else {
                *reinterpret_cast<float2*>(tile + row * PITCH + c0 + 2 * j) = make_float2(a, b);
            }
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    if (*abort_flag && warp == 1) {
        // A wait gave up: what was asked for lands and what was issued ends before the CTA leaves and its tensor memory is another's.
        int never = 0;
        for (uint32_t f = counts[0] > STAGES ? counts[0] - STAGES : 0; f < counts[0]; ++f)
            mbar_wait_warp(smem_u32(&full[f % STAGES]), (f / STAGES) & 1u, &never);
        if (counts[1] > 0) {
            const uint32_t last = counts[1] - 1;
            mbar_wait_warp(smem_u32(&empty[last % STAGES]), (last / STAGES) & 1u, &never);
            mbar_wait_warp(smem_u32(&tfull[last % NBUF]), (last / NBUF) & 1u, &never);
        }
    }
    if (warp == 1) tmem_dealloc(tmem_base, TCOLS);
    // After a wait that gave up, the tiles of the cluster are not whole, and what is written is undefined.
    const int row_a = ROWS * rank / p.splits, row_b = ROWS * (rank + 1) / p.splits;
    constexpr int GROUPS = COLS / 8;                         // sixteen, in both forms
    static_assert(GROUPS == 16, "sixteen lanes hold a row");
    // A lane takes eight neighbouring columns of a row; sixteen apart where rows of the output start anywhere, so that the sixteen lanes
    // of a row write side by side.  (Every warp goes round as often as the others: the lanes of a row exchange their largest values.)
    const int step = p.out16 || p.out_kind == OUT_E4M3 ? 1 : GROUPS;
    for (int u = row_a * GROUPS + (int)threadIdx.x; u - lane < row_b * GROUPS; u += NTHREADS) {
        const int r = u / GROUPS, g = u % GROUPS, c = step == 1 ? 8 * g : g;
        const long long m = (long long)(SWAP ? qt * BN : pt * BP) + r;
        const int n = (SWAP ? pt * BP : qt * BN) + c, left = r < row_b && m < p.M ? p.N - n : 0;
        const float* from = tile + (r < row_b ? r : row_a) * PITCH + c;
        auto sum = [&](float (&v)[8]) {
            if (p.splits == 1) {
                if (step == 1) {
                    const float4 a = *reinterpret_cast<const float4*>(from), b = *reinterpret_cast<const float4*>(from + 4);
                    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = from[GROUPS * j];
                }
                return;
            }
            // two CTAs' parts at once: what takes time is the way there
            const uint32_t off = smem_u32(from);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
            for (int k = 0; k < p.splits; k += 2) {
                const uint32_t at0 = map_to_cta(off, k), at1 = map_to_cta(off, k + 1);
                float w0[8], w1[8];
                if (step == 1) {
                    const float4 a = ld_cluster_f32x4(at0), b = ld_cluster_f32x4(at0 + 16), c = ld_cluster_f32x4(at1),
                                 d = ld_cluster_f32x4(at1 + 16);
                    w0[0] = a.x; w0[1] = a.y; w0[2] = a.z; w0[3] = a.w; w0[4] = b.x; w0[5] = b.y; w0[6] = b.z; w0[7] = b.w;
                    w1[0] = c.x; w1[1] = c.y; w1[2] = c.z; w1[3] = c.w; w1[4] = d.x; w1[5] = d.y; w1[6] = d.z; w1[7] = d.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) w0[j] = ld_cluster_f32(at0 + 4 * GROUPS * j);
#pragma unroll
                    for (int j = 0; j < 8; ++j) w1[j] = ld_cluster_f32(at1 + 4 * GROUPS * j);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (v[j] + w0[j]) + w1[j];
            }
        };
        if (p.io == CONVNN_F32) finish8<float>(p, m, n, left, step, sum);
        else finish8<__nv_bfloat16>(p, m, n, left, step, sum);
    }
    if (p.splits > 1) cluster_sync_all();                    // the others may still read this CTA's tile
}

// CTAs that share the blocks of k of a tile: as many as leave every CTA an SM and two blocks.  (Two CTAs per SM load no faster: 1 x 4096 x
// 4096 7.6 -> 9.5 us with 256 CTAs instead of 128.  With fewer blocks the sum of the parts takes longer: 128 x 1024 x 1024 9.1 -> 10.8.)
int splits_of(long long tiles, int blocks) {
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= device_sms() && blocks >= 4 * splits) splits *= 2;
    return splits;
}

template <int BN, bool SWAP>
int launch_tiles(const CUtensorMap& tmP, const CUtensorMap& tmQ, LinearFp8Params p, cudaStream_t st) {
    constexpr size_t STAGE = (size_t)(BP + BN) * KB;
    constexpr size_t TILE = (size_t)(SWAP ? BN * (BP + 4) : BP * (BN + 4)) * 4;
    const long long tiles = SWAP ? (long long)((p.N + BP - 1) / BP) * ((p.M + BN - 1) / BN)
                                 : (long long)((p.M + BP - 1) / BP) * ((p.N + BN - 1) / BN);
    if (tiles * 8 > 0x7fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "linear_fp8: %d x %d is too many tiles", p.M, p.N);
    p.splits = splits_of(tiles, p.blocks);
    const int per = (p.blocks + p.splits - 1) / p.splits;
    p.stages = SWAP ? MAX_STAGES : 3;
    while (p.stages > per && p.stages > 2) --p.stages;
    // (two CTAs per SM where there are more tiles: 1 x 20480 x 4096 30.4 -> 19.8 us, 64 x 20480 x 4096 44.2 -> 28.0)
    const size_t room = (size_t)(tiles * p.splits > device_sms() ? 108 : 200) * 1024;
    while (p.stages * STAGE > room) --p.stages;
    size_t smem = p.stages * STAGE;
    if (smem < TILE) smem = TILE;
    smem += 1024;
    auto kern = linear_fp8_kernel<BN, SWAP>;
    CONVNN_ENSURE_SMEM(kern, smem);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0] = chained_attribute(st);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(tiles * p.splits)); cfg.blockDim = dim3(NTHREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = p.splits > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tmP, tmQ, p);
    if (e != cudaSuccess) return set_error(CONVNN_E_CUDA, "linear_fp8 launch: %s", cudaGetErrorString(e));
    CONVNN_CHECK_LAUNCH("linear_fp8");
    return CONVNN_OK;
}

// ---- CTA pairs ------------------------------------------------------------------------------------------------------
// Two CTAs of a cluster (cta_group::2) have tiles of 256 x 256: 128 rows of a each, whose sums are in their own TMEM, and half of
// the rows of w each, so that a CTA copies 32 KB for 512 cycles of products (a lone CTA's 128 x 256 tile: 48 KB).
//   warp 0      TMA producer of its CTA's operands, credited to the even CTA's barriers
//   warp 1      MMA issuer (even CTA), a block of k into one of two buffers of 256 columns
//   warps 2, 3  the scales of four blocks of k at a time
//   warps 4-11  epilogue: a warp has 32 rows and 128 columns, its sums in registers (128 of 224), and after the last block bias, GELU,
//               residual, rounding; the results leave through its two slabs of shared memory, 32 rows of 128 bytes in the order
//               of the 128-byte swizzle, by TMA where rows start and end on 16-byte boundaries.  Meanwhile the next tile's first two
//               blocks are multiplied.
// Twelve warps are launched with 168 registers a thread; the first four keep 56, which leaves the others 224: 4 * 32 * 56 + 8 * 32 * 224
// = 12 * 32 * 168.
// What bounds it: 16384 x 4096 x 4096 runs at 1.68 PFLOP/s under the 1000 W power cap (1.86 for ten launches), 1.2 times what a bfloat16
// library product sustains there; a block of k takes about 1000 cycles, of them 512 to 600 the tensor cores', the rest the way from
// the product to the sums and back with two buffers, and the sums' own reads of TMEM (128 columns of two warps per scheduler: 290
// cycles at the port's rate).  Few blocks of k: the output, GELU's 14 multiply-adds a value (50432 x 768 x 192).
// Slower, ten launches of 16384 x 4096 x 4096: sixteen epilogue warps of 64 columns 418 us, lone CTAs of 128 x 256 330, waits that spin
// 309, where pairs took 296; halves of a tile one after the other with buffers of their own 292 -> 419 (50432 x 768 x 192 with
// GELU 57.7 -> 62.4).  Sums as float32 pairs do not stay in registers; 48 columns in flight instead of 32 change nothing.
constexpr int PAIR_WARPS = 8, PAIR_THREADS = 128 + 32 * PAIR_WARPS;
constexpr int PAIR_N = 256;
constexpr uint32_t PAIR_STAGE = 2 * BP * KB, SLAB = 4096;
constexpr int PAIR_STAGES = 4;
constexpr int SCALE_GROUP = 4, SCALE_SLOTS = 4;              // blocks of k whose scales come together, and how many times that is held
constexpr uint32_t SCALE_BYTES = SCALE_GROUP * (BP + 2) * 4 + 96;        // the rows', the two column blocks'; a multiple of 128

__device__ __forceinline__ void mma_e4m3_ss_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                                 uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tma_store_2d_a(const CUtensorMap* m, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(m)), "r"(src), "r"(c0), "r"(c1)
                 : "memory");
}
__device__ __forceinline__ void add_scaled(float* acc, const uint32_t (&part)[16], float scale) {
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = fmaf(__uint_as_float(part[j]), scale, acc[j]);
}
// Four bytes to shared memory; zero, and nothing read, where not `in`.
__device__ __forceinline__ void copy4(uint32_t to, const float* base, const float* from, bool in) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(in ? from : base), "r"(in ? 4 : 0) : "memory");
}
// Whether a phase is over, without waiting for it.
__device__ __forceinline__ bool mbar_test_a(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t at, const uint4& v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// 16 bytes of a warp's slab: row r of 128 bytes, slot s of 16, placed as the 128-byte swizzle does: neither eight lanes on neighbouring
// rows nor eight on one row meet in a bank.
__device__ __forceinline__ uint32_t slab_at(uint32_t slab, int r, int s) { return slab + r * 128 + ((s ^ (r & 7)) << 4); }

template <typename T> struct Values16 { static constexpr int N = 16 / sizeof(T); };
// acc += the values of 16 bytes.
__device__ __forceinline__ void add16(const uint4& v, float* acc, __nv_bfloat16) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        acc[2 * i] += __uint_as_float(w[i] << 16);
        acc[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void add16(const uint4& v, float* acc, float) {
    acc[0] += __uint_as_float(v.x); acc[1] += __uint_as_float(v.y);
    acc[2] += __uint_as_float(v.z); acc[3] += __uint_as_float(v.w);
}
// Rows that start anywhere: a row's 128 bytes from column n on as lanes side by side, B bytes each.  B is T's size, or 4 for pairs.
template <typename T, int B> struct Bytes { using type = T; };
template <> struct Bytes<__nv_bfloat16, 2> { using type = uint16_t; };
template <> struct Bytes<__nv_bfloat16, 4> { using type = uint32_t; };
template <typename T, int B>
__device__ __forceinline__ void rows_to_slab(const T* base, long long ld, int M, int N, long long m0, int n, uint32_t slab, int lane) {
    using E = typename Bytes<T, B>::type;
    constexpr int U = 4 / B, AT_ONCE = 8 / U;
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
        E v[AT_ONCE][U];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int col = n + (32 * u + lane) * B / (int)sizeof(T);
                v[i][u] = E{};
                if (m0 + r0 + i < M && col < N) v[i][u] = *reinterpret_cast<const E*>(base + (m0 + r0 + i) * ld + col);
            }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = (32 * u + lane) * B;
                const uint32_t to = slab_at(slab, r0 + i, at >> 4) + (at & 15);
                if constexpr (B == 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(reinterpret_cast<const uint32_t&>(v[i][u])) : "memory");
                else asm volatile("st.shared.b16 [%0], %1;" ::"r"(to), "h"(reinterpret_cast<const uint16_t&>(v[i][u])) : "memory");
            }
    }
}
template <typename T>
__device__ __forceinline__ void slab_to_rows(T* base, long long ld, int M, int N, long long m0, int n, uint32_t slab, int lane) {
    using E = typename Bytes<T, sizeof(T)>::type;
    constexpr int B = sizeof(T), U = 4 / B;
#pragma unroll 4
    for (int r = 0; r < 32; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = (32 * u + lane) * B, col = n + 32 * u + lane;
            const uint32_t from = slab_at(slab, r, at >> 4) + (at & 15);
            E v;
            if constexpr (B == 4) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(reinterpret_cast<uint32_t&>(v)) : "r"(from) : "memory");
            else if constexpr (B == 2) asm volatile("ld.shared.b16 %0, [%1];" : "=h"(reinterpret_cast<uint16_t&>(v)) : "r"(from) : "memory");
            else {
                uint32_t w;
                asm volatile("ld.shared.u8 %0, [%1];" : "=r"(w) : "r"(from) : "memory");
                v = (E)w;
            }
            if (m0 + r < M && col < N) *reinterpret_cast<E*>(base + (m0 + r) * ld + col) = v;
        }
}
// The same for rows on 4-byte boundaries: two bfloat16 values a lane, or the last of a row.
__device__ __forceinline__ void slab_to_rows4(__nv_bfloat16* base, long long ld, int M, int N, long long m0, int n, uint32_t slab, int lane) {
    const int col = n + 2 * lane;
#pragma unroll 4
    for (int r = 0; r < 32; ++r) {
        uint32_t v;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(slab_at(slab, r, lane >> 2) + ((4 * lane) & 15)) : "memory");
        __nv_bfloat16* to = base + (m0 + r) * ld + col;
        if (m0 + r >= M || col >= N) continue;
        if (col + 1 < N) *reinterpret_cast<uint32_t*>(to) = v;
        else *reinterpret_cast<uint16_t*>(to) = (uint16_t)v;
    }
}
// 8-bit rows on 16-byte boundaries: sixteen a lane, the last of a row in smaller pieces.  (50432 x 1000 x 768 into 8 bits 72 us, four a lane 82;
// by TMA, over what lies behind, 63.  The whole slabs of a row by TMA and this for its last: 70, but 28.7 instead of 27.9 for 768 columns.)
__device__ __forceinline__ void slab_to_rows16(uint8_t* base, long long ld, int M, int N, long long m0, int n, uint32_t slab, int lane) {
    const int left = N - n - 16 * (lane & 7);
    uint8_t* to = base + (m0 + (lane >> 3)) * ld + n + 16 * (lane & 7);
#pragma unroll 2
    for (int r = lane >> 3; r < 32; r += 4, to += 4 * ld) {
        const uint4 v = lds128(slab_at(slab, r, lane & 7));
        if (m0 + r >= M || left <= 0) continue;
        if (left >= 16) {
            *reinterpret_cast<uint4*>(to) = v;
        } else {
            uint32_t w[3] = {v.x, v.y, v.z};
            uint8_t* p = to;
            if (left & 8) { *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]); w[0] = w[2]; w[1] = v.w; p += 8; }
            if (left & 4) { *reinterpret_cast<uint32_t*>(p) = w[0]; w[0] = w[1]; p += 4; }
            if (left & 2) { *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0]; w[0] >>= 16; p += 2; }
            if (left & 1) *p = (uint8_t)w[0];
        }
    }
}

// The residual of 32 rows and 128 bytes of columns from column n on into the slab: asked for here, there after residual_arrived().
template <typename T>
__device__ __forceinline__ void request_residual(const LinearFp8Params& p, long long m0, int n, uint32_t slab, int lane) {
    const T* base = static_cast<const T*>(p.residual);
    if (p.residual16) {
        constexpr int V = Values16<T>::N;
        const int col = n + (lane & 7) * V, valid = p.N - col;
        const T* from = base + (m0 + (lane >> 3)) * p.ldr + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            const bool in = m0 + r < p.M && valid > 0;
            const uint32_t bytes = in ? min(16u, (uint32_t)valid * (uint32_t)sizeof(T)) : 0u;      // the rest is filled with zeros
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slab_at(slab, r, lane & 7)), "l"(in ? from : base), "r"(bytes)
                         : "memory");
            from += 4 * p.ldr;
        }
    } else if (sizeof(T) == 4 || !p.residual4) {
        rows_to_slab<T, sizeof(T)>(base, p.ldr, p.M, p.N, m0, n, slab, lane);
    } else {
        rows_to_slab<T, 4>(base, p.ldr, p.M, p.N, m0, n, slab, lane);
    }
}
__device__ __forceinline__ void residual_arrived() {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
}
// acc += this lane's row of the slab.
template <typename T>
__device__ __forceinline__ void add_row(uint32_t slab, int lane, float* acc) {
#pragma unroll
    for (int s = 0; s < 8; ++s) add16(lds128(slab_at(slab, lane, s)), acc + s * Values16<T>::N, T());
}
// The slab's 32 rows of 128 bytes -> out, from column n on.
template <typename T>
__device__ __forceinline__ void store_slab(const LinearFp8Params& p, const CUtensorMap* tmO, long long m0, int n, uint32_t slab, int lane) {
    if (p.out_tma) {
        fence_proxy_async();
        __syncwarp();
        if (lane == 0 && m0 < p.M && n < p.N) tma_store_2d_a(tmO, slab, n, (int)m0);
        if (lane == 0) tma_store_commit();
        return;
    }
    __syncwarp();
    T* out = static_cast<T*>(p.out);
    if constexpr (sizeof(T) == 1) {
        if (p.out16) slab_to_rows16(out, p.ldo, p.M, p.N, m0, n, slab, lane);
        else slab_to_rows<T>(out, p.ldo, p.M, p.N, m0, n, slab, lane);
    } else if constexpr (sizeof(T) == 2) {
        if (p.out4) slab_to_rows4(out, p.ldo, p.M, p.N, m0, n, slab, lane);
        else slab_to_rows<T>(out, p.ldo, p.M, p.N, m0, n, slab, lane);
    } else {
        slab_to_rows<T>(out, p.ldo, p.M, p.N, m0, n, slab, lane);
    }
    __syncwarp();
}

template <int OUT, bool GELU>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
linear_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ CUtensorMap tmO, const LinearFp8Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* slabs = smem + PAIR_STAGES * PAIR_STAGE;         // two a warp
    float* scales = reinterpret_cast<float*>(slabs + 2 * PAIR_WARPS * SLAB);       // [slot]: [block of the group][row], [block][half of the columns]
    __shared__ uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], tfull[2], tempty[2], sfull[SCALE_SLOTS], sempty[SCALE_SLOTS];
    __shared__ uint32_t tmem_slot;
    __shared__ uint32_t counts[3];                           // fills by the even and by the odd CTA, blocks of k multiplied
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < PAIR_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 2 * PAIR_WARPS); }
        for (int b = 0; b < SCALE_SLOTS; ++b) { mbar_init(&sfull[b], 64); mbar_init(&sempty[b], PAIR_WARPS); }
        abort_word = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmA);
        prefetch_tensormap(&tmW);
        prefetch_tensormap(&tmO);
    }
    __syncthreads();
    if (warp == 1) { tmem_alloc_pair(&tmem_slot, 512); tmem_relinquish_pair(); }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();                                      // both CTAs' barriers exist before any remote signal
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    const uint32_t peer_abort = map_to_cta(smem_u32(&abort_word), rank ^ 1u);
    auto give_up = [&](int code) {
        st_cluster_u32(peer_abort, 1u);
        fail(abort_flag, code);
    };
    auto tell = [&](uint32_t i, uint32_t n) {                // both CTAs
        if (lane == 0) {
            counts[i] = n;
            st_cluster_u32(map_to_cta(smem_u32(&counts[i]), rank ^ 1u), n);
        }
    };
    chain_begin();

    const int n_n = (p.N + PAIR_N - 1) / PAIR_N, n_m = (p.M + 2 * BP - 1) / (2 * BP);
    const int tiles = n_n * n_m, first = blockIdx.x >> 1, step = gridDim.x >> 1;
    const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), tfull0 = smem_u32(tfull), tempty0 = smem_u32(tempty);
    const uint32_t s0 = smem_u32(smem);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            const uint32_t lead_full0 = map_to_cta(full0, 0);
            uint32_t s = 0, ph = 0, fills = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                const int m0 = t / n_n * 2 * BP + (int)rank * BP, n0 = t % n_n * PAIR_N + (int)rank * BP;
                for (int kb = 0; kb < p.blocks; ++kb) {
                    if (!mbar_wait_warp(empty0 + 8 * s, ph ^ 1u, abort_flag)) { if (lane == 0) give_up(125); ok = false; break; }
                    if (elect_one()) {
                        if (rank == 0) mbar_expect_tx_a(full0 + 8 * s, 2 * PAIR_STAGE);
                        tma_load_2d_pair(s0 + s * PAIR_STAGE, &tmA, lead_full0 + 8 * s, kb * KB, m0);
                        tma_load_2d_pair(s0 + s * PAIR_STAGE + BP * KB, &tmW, lead_full0 + 8 * s, kb * KB, n0);
                    }
                    __syncwarp();
                    ++fills;
                    if (++s == PAIR_STAGES) { s = 0; ph ^= 1u; }
                }
            }
            // the last signals to this CTA's barriers have come before it leaves
            for (uint32_t i = 0; i < PAIR_STAGES && i < fills && ok; ++i) {
                if (s == 0) { s = PAIR_STAGES; ph ^= 1u; }
                --s;
                ok = mbar_wait_warp(empty0 + 8 * s, ph, abort_flag);
            }
            tell(rank, fills);
        } else if (warp == 1) {
            if (rank == 0) {
                constexpr uint32_t idesc = idesc_e4m3_f32(2 * BP, PAIR_N);
                const uint64_t hi = kmajor_desc_hi(KB);
                uint32_t s = 0, ph = 0, buf = 0, tph = 0, issued = 0;
                bool ok = true;
                for (int t = first; t < tiles && ok; t += step) {
                    for (int kb = 0; kb < p.blocks; ++kb) {
                        if (!mbar_wait_warp(full0 + 8 * s, ph, abort_flag)) { if (lane == 0) give_up(127); ok = false; break; }
                        if (!mbar_wait_warp(tempty0 + 8 * buf, tph ^ 1u, abort_flag)) { if (lane == 0) give_up(126); ok = false; break; }
                        tc_fence_after_sync();
                        if (elect_one()) {
                            const uint64_t ad = hi | (uint64_t)(((s0 + s * PAIR_STAGE) & 0x3FFFFu) >> 4);
                            const uint64_t bd = hi | (uint64_t)(((s0 + s * PAIR_STAGE + BP * KB) & 0x3FFFFu) >> 4);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                mma_e4m3_ss_pair(tmem_base + buf * PAIR_N, ad + 2 * i, bd + 2 * i, idesc, i > 0);
                            mma_commit_pair_both(empty0 + 8 * s);
                            mma_commit_pair_both(tfull0 + 8 * buf);
                        }
                        __syncwarp();
                        if (++s == PAIR_STAGES) { s = 0; ph ^= 1u; }
                        buf ^= 1u;
                        if (buf == 0) tph ^= 1u;
                        ++issued;
                    }
                }
                tell(2, issued);
            }
        } else {
            // copied straight to shared memory, zeros where there is nothing; a warp has two blocks of a group
            const int i0 = 2 * (warp - 2);
            const long long rows32 = 32 * p.sa_row;
            uint32_t slot = 0, ph = 0;
            bool ok = true;
            for (int t = first; t < tiles && ok; t += step) {
                const int m0 = t / n_n * 2 * BP + (int)rank * BP + lane, n = t % n_n * PAIR_N + (lane & 1) * KB;
                for (int kb0 = 0; kb0 < p.blocks; kb0 += SCALE_GROUP) {
                    if (!mbar_wait_warp(smem_u32(&sempty[slot]), ph ^ 1u, abort_flag)) { if (lane == 0) give_up(129); ok = false; break; }
                    const uint32_t to = smem_u32(scales) + slot * SCALE_BYTES;
#pragma unroll
                    for (int i = i0; i < i0 + 2; ++i) {
                        const bool in = kb0 + i < p.blocks;
                        const float* from = p.sa + (long long)m0 * p.sa_row + (kb0 + i) * p.sa_block;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            copy4(to + (i * BP + 32 * j + lane) * 4, p.sa, from, in && m0 + 32 * j < p.M);
                            from += rows32;
                        }
                        if (lane < 2)
                            copy4(to + (SCALE_GROUP * BP + 2 * i + lane) * 4, p.sw, p.sw + (long long)(n / KB) * p.sw_row + (kb0 + i) * p.sw_block,
                                  in && n < p.N);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sfull[slot])) : "memory");
                    if (++slot == SCALE_SLOTS) { slot = 0; ph ^= 1u; }
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quarter = warp & 3, half = (warp - 4) >> 2, row = quarter * 32 + lane;
        const uint32_t slab0 = smem_u32(slabs) + (warp - 4) * (2 * SLAB);
        const uint32_t bias0 = smem_u32(scales) + SCALE_SLOTS * SCALE_BYTES + (warp - 4) * 512;
        const uint32_t lead_tempty0 = map_to_cta(tempty0, 0);
        const uint32_t taddr = tmem_base + half * KB + ((uint32_t)(quarter * 32) << 16);
        const uint32_t sc0 = smem_u32(scales), sfull0 = smem_u32(sfull);
        uint32_t slot = 0, sph = 0, buf = 0, tph = 0;
        bool ok = true;
        uint32_t even[16], odd[16];
        // The scale of block kb; a group of them is waited for with its first one, which comes when the last group has been read.
        auto scale_of = [&](int kb) {
            const int i = kb % SCALE_GROUP;
            if (i == 0) {
                if (kb > 0) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sempty[slot]);
                    if (++slot == SCALE_SLOTS) { slot = 0; sph ^= 1u; }
                }
                if (ok && !mbar_wait_warp(sfull0 + 8 * slot, sph, abort_flag)) { if (lane == 0) give_up(130); ok = false; }
            }
            float a, w;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(a) : "r"(sc0 + slot * SCALE_BYTES + (i * BP + row) * 4) : "memory");
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(w) : "r"(sc0 + slot * SCALE_BYTES + (SCALE_GROUP * BP + 2 * i + half) * 4) : "memory");
            return a * w;
        };
        for (int t = first; t < tiles; t += step) {
            const long long m0 = (long long)(t / n_n) * 2 * BP + rank * BP + quarter * 32;      // of the warp
            const int n = t % n_n * PAIR_N + half * KB;
            if (p.residual) {
                if (lane == 0) tma_store_wait_read<0>();     // the last tile's results have left the slabs
                __syncwarp();
                if (p.io == CONVNN_F32) {
                    request_residual<float>(p, m0, n, slab0, lane);
                    request_residual<float>(p, m0, n + 32, slab0 + SLAB, lane);
                } else {
                    request_residual<__nv_bfloat16>(p, m0, n, slab0, lane);
                    request_residual<__nv_bfloat16>(p, m0, n + 64, slab0 + SLAB, lane);
                }
            }
            // four columns' bias a lane, as they are stored
            uint4 bias = make_uint4(0, 0, 0, 0);
            if (p.bias) {
                const int c = n + 4 * lane;
                if (p.bias16 && c + 4 <= p.N) {
                    if (p.io == CONVNN_F32) {
                        bias = *reinterpret_cast<const uint4*>(static_cast<const float*>(p.bias) + c);
                    } else {
                        const uint2 two = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.bias) + c);
                        bias.x = two.x; bias.y = two.y;
                    }
                } else if (p.io == CONVNN_F32) {
                    const uint32_t* from = static_cast<const uint32_t*>(p.bias) + c;
                    if (c < p.N) bias.x = from[0];
                    if (c + 1 < p.N) bias.y = from[1];
                    if (c + 2 < p.N) bias.z = from[2];
                    if (c + 3 < p.N) bias.w = from[3];
                } else {
                    const uint16_t* from = static_cast<const uint16_t*>(p.bias) + c;
                    if (c < p.N) bias.x = from[0];
                    if (c + 1 < p.N) bias.x |= (uint32_t)from[1] << 16;
                    if (c + 2 < p.N) bias.y = from[2];
                    if (c + 3 < p.N) bias.y |= (uint32_t)from[3] << 16;
                }
            }
            float acc[128];                                  // (pairs, as elsewhere, do not stay in registers here)
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j) odd[j] = 0u;
            float last = 0.f;
            float scale = scale_of(0);
            bool ready = false;
#pragma unroll 1
            for (int kb = 0; kb < p.blocks; ++kb) {
                if (!__all_sync(0xffffffffu, ready) && ok && !mbar_wait_warp(tfull0 + 8 * buf, tph, abort_flag)) {
                    if (lane == 0) give_up(128);
                    ok = false;
                }
                tc_fence_after_sync();
                // sixteen columns are added up while the next are on their way, the last under the next block's first; the next block's
                // scale and barrier are asked for in between
                const uint32_t from = taddr + buf * PAIR_N;
                float next = 0.f;
                tmem_ld_x16(from, even);
                add_scaled(acc + 112, odd, last);
#pragma unroll
                for (int c = 0; c < 8; c += 2) {
                    tmem_ld_wait();
                    tmem_ld_x16(from + 16 * (c + 1), odd);
                    add_scaled(acc + 16 * c, even, scale);
                    if (c == 0 && kb + 1 < p.blocks) next = scale_of(kb + 1);
                    if (c == 4) {
                        buf ^= 1u;
                        if (buf == 0) tph ^= 1u;
                        ready = mbar_test_a(tfull0 + 8 * buf, tph);
                    }
                    tmem_ld_wait();
                    if (c == 6) break;
                    tmem_ld_x16(from + 16 * (c + 2), even);
                    add_scaled(acc + 16 * (c + 1), odd, scale);
                }
                last = scale;
                scale = next;
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(lead_tempty0 + 8 * (buf ^ 1u));
            }
            if (lane == 0) mbar_arrive(&sempty[slot]);
            if (++slot == SCALE_SLOTS) { slot = 0; sph ^= 1u; }
            add_scaled(acc + 112, odd, last);
            if (p.bias) {
                if (p.io != CONVNN_F32) bias = make_uint4(bias.x << 16, bias.x & 0xffff0000u, bias.y << 16, bias.y & 0xffff0000u);
                sts128(bias0 + 16 * lane, bias);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 128; j += 4) add16(lds128(bias0 + 4 * j), acc + j, 0.f);
                __syncwarp();
            }
            if (GELU && OUT == OUT_F32) {
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j] = gelu_erf(acc[j]);
            } else if (GELU) {
#pragma unroll
                for (int j = 0; j < 128; j += 8) gelu8(acc + j);
            }
            if (!p.residual) {
                if (lane == 0) tma_store_wait_read<0>();
                __syncwarp();
            } else {
                residual_arrived();
                if (p.io == CONVNN_F32) {
                    add_row<float>(slab0, lane, acc);
                    add_row<float>(slab0 + SLAB, lane, acc + 32);
                    __syncwarp();
                    request_residual<float>(p, m0, n + 64, slab0, lane);
                    request_residual<float>(p, m0, n + 96, slab0 + SLAB, lane);
                    residual_arrived();
                    add_row<float>(slab0, lane, acc + 64);
                    add_row<float>(slab0 + SLAB, lane, acc + 96);
                } else {
                    add_row<__nv_bfloat16>(slab0, lane, acc);
                    add_row<__nv_bfloat16>(slab0 + SLAB, lane, acc + 64);
                }
            }
            // (a lane writes the row of the slab that it has read)
            if (OUT == OUT_BF16) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint32_t slab = slab0 + q * SLAB;
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const float* v = acc + 64 * q + 8 * s;
                        const f32x2 four[4] = {pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
                        sts128(slab_at(slab, lane, s), f32x2_to_bf16x8(four));
                    }
                    store_slab<__nv_bfloat16>(p, &tmO, m0, n + 64 * q, slab, lane);
                }
            } else if (OUT == OUT_F32) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint32_t slab = slab0 + (q & 1) * SLAB;
                    if (q >= 2) {
                        if (lane == 0) tma_store_wait_read<1>();
                        __syncwarp();
                    }
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const float* f = acc + 32 * q + 4 * s;
                        sts128(slab_at(slab, lane, s), make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                                                  __float_as_uint(f[3])));
                    }
                    store_slab<float>(p, &tmO, m0, n + 32 * q, slab, lane);
                }
            } else {
                float most[4] = {0.f, 0.f, 0.f, 0.f};
                if (n + KB <= p.N) {
#pragma unroll
                    for (int j = 0; j < 128; ++j) most[j & 3] = max_nan(most[j & 3], fabsf(acc[j]));
                } else {
#pragma unroll
                    for (int j = 0; j < 128; ++j)
                        if (n + j < p.N) most[j & 3] = max_nan(most[j & 3], fabsf(acc[j]));
                }
                const uint32_t top = abs_bits(max_nan(max_nan(most[0], most[1]), max_nan(most[2], most[3])));
                const float to = fp8_scale(top), inv = __frcp_rn(to);
                const uint32_t slab = slab0;
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float* f = acc + 16 * s + 4 * i;
                        w[i] = e4m3x4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
                    }
                    sts128(slab_at(slab, lane, s), make_uint4(w[0], w[1], w[2], w[3]));
                }
                if (m0 + lane < p.M && n < p.N) p.so[(m0 + lane) * p.so_row + n / KB * p.so_block] = to;
                store_slab<uint8_t>(p, &tmO, m0, n, slab, lane);
            }
        }
        if (lane == 0) tma_store_wait<0>();
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();                                      // the peer no longer signals or reads this CTA
    if (*abort_flag) {
        // A wait gave up (in both CTAs, give_up() has seen to that): what was asked for lands and what was issued ends before
        // either of them leaves.
        if (warp == 0 && lane == 0) {
            int never = 0;
            if (rank == 0) drain_pair_ring(full0, PAIR_STAGES, PAIR_STAGE, counts[0], counts[1]);
            if (counts[2] > 0) {
                const uint32_t last = counts[2] - 1;
                mbar_wait_a(empty0 + 8 * (last % PAIR_STAGES), (last / PAIR_STAGES) & 1u, &never);
                mbar_wait_a(tfull0 + 8 * (last & 1u), (last >> 1) & 1u, &never);
            }
        }
        __syncwarp();
        cluster_sync_all();
    }
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

template <int OUT, bool GELU>
int launch_pairs(const CUtensorMap& tmA, const CUtensorMap& tmW, const LinearFp8Params& p, cudaStream_t st) {
    CUtensorMap tmO = tmA;                                   // (unused where rows of the output start or end anywhere)
    if (p.out_tma) {
        const int elt = OUT == OUT_F32 ? 4 : OUT == OUT_BF16 ? 2 : 1;
        const uint64_t dims[2] = {(uint64_t)p.N, (uint64_t)p.M}, strides[1] = {(uint64_t)p.ldo * elt};
        const uint32_t box[2] = {(uint32_t)(128 / elt), 32};
        const bool ok = OUT == OUT_F32    ? encode_tensor_map_f32(&tmO, p.out, 2, dims, strides, box, 128)
                        : OUT == OUT_BF16 ? encode_tensor_map_bf16(&tmO, p.out, 2, dims, strides, box, 128)
                                          : encode_tensor_map_u8(&tmO, p.out, 2, dims, strides, box, 128);
        if (!ok) return CONVNN_E_CUDA;
    }
    constexpr size_t smem = PAIR_STAGES * PAIR_STAGE + 2 * PAIR_WARPS * SLAB + SCALE_SLOTS * SCALE_BYTES + PAIR_WARPS * 512 + 1024;
    const long long tiles = (long long)((p.M + 2 * BP - 1) / (2 * BP)) * ((p.N + PAIR_N - 1) / PAIR_N);
    if (tiles > 0x3fffffffll) return set_error(CONVNN_E_UNSUPPORTED, "linear_fp8: %d x %d is too many tiles", p.M, p.N);
    auto kern = linear_fp8_pair_kernel<OUT, GELU>;
    CONVNN_ENSURE_SMEM(kern, smem);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(PAIR_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
    cfg.gridDim = dim3(2);
    static ClusterLimit fit{};
    int pairs = 0;
    if (const int rc = fit.query(reinterpret_cast<const void*>(kern), &cfg, &pairs)) return rc;
    cfg.gridDim = dim3(2 * (unsigned)(tiles < pairs ? tiles : pairs));
    attr[1] = chained_attribute(st); cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tmA, tmW, tmO, p);
    if (e != cudaSuccess) return set_error(CONVNN_E_CUDA, "linear_fp8 pair launch: %s", cudaGetErrorString(e));
    CONVNN_CHECK_LAUNCH("linear_fp8_pair");
    return CONVNN_OK;
}

bool encode_rows(CUtensorMap* m, const void* base, long long rows, int K, long long ld, int box_rows) {
    const uint64_t dims[2] = {(uint64_t)K, (uint64_t)rows}, strides[1] = {(uint64_t)ld};
    const uint32_t box[2] = {(uint32_t)KB, (uint32_t)box_rows};
    return encode_tensor_map_u8(m, base, 2, dims, strides, box, 128);
}

}  // namespace

int launch_linear_fp8(const void* a, long long lda, const float* sa, long long sa_row, long long sa_block, const void* w,
                      long long ldw, const float* sw, long long sw_row, long long sw_block, const void* bias, const void* residual,
                      long long ldr, int io, void* out, long long ldo, float* so, long long so_row, long long so_block, int M, int N,
                      int K, int gelu, cudaStream_t st) {
    LinearFp8Params p{};
    p.sa = sa; p.sa_row = sa_row; p.sa_block = sa_block;
    p.sw = sw; p.sw_row = sw_row; p.sw_block = sw_block;
    p.bias = bias; p.residual = residual; p.out = out; p.so = so;
    p.ldr = ldr; p.ldo = ldo; p.so_row = so_row; p.so_block = so_block;
    p.M = M; p.N = N; p.blocks = (K + KB - 1) / KB;
    p.io = io; p.gelu = gelu;
    p.out_kind = so ? OUT_E4M3 : io == CONVNN_F32 ? OUT_F32 : OUT_BF16;
    const long long per16 = io == CONVNN_F32 ? 4 : 8;
    const long long elt = io == CONVNN_F32 ? 4 : 2, out_elt = so ? 1 : elt;
    auto on = [](const void* q, long long ld_bytes, int n) { return ((uintptr_t)ld_bytes | reinterpret_cast<uintptr_t>(q)) % n == 0; };
    p.bias16 = on(bias, 0, 16);
    p.residual16 = on(residual, ldr * elt, 16); p.residual4 = on(residual, ldr * elt, 4) && N % 2 == 0;
    p.out16 = on(out, ldo * out_elt, 16); p.out_tma = p.out16 && N * out_elt % 16 == 0; p.out4 = on(out, ldo * out_elt, 4);
    const long long pair_tiles = (long long)((M + 2 * BP - 1) / (2 * BP)) * ((N + PAIR_N - 1) / PAIR_N);
    // Pairs from a tile per five SMs on: 512 x 4096 x 4096 (32 tiles) 31.4 -> 24.2 us, 3152 x 768 x 768 (39) 10.9 -> 9.0; with fewer the
    // clusters that share a tile's sum are faster (256 x 4096 x 4096, 16 tiles: 16.7 against 23.6).  Up to 128 rows half a tile is empty.
    if (M > 128 && pair_tiles * 5 >= device_sms()) {
        CUtensorMap tmA, tmW;
        if (!encode_rows(&tmA, a, M, K, lda, BP) || !encode_rows(&tmW, w, N, K, ldw, BP)) return CONVNN_E_CUDA;
        if (p.out_kind == OUT_F32) return gelu ? launch_pairs<OUT_F32, true>(tmA, tmW, p, st) : launch_pairs<OUT_F32, false>(tmA, tmW, p, st);
        if (p.out_kind == OUT_BF16) return gelu ? launch_pairs<OUT_BF16, true>(tmA, tmW, p, st) : launch_pairs<OUT_BF16, false>(tmA, tmW, p, st);
        return gelu ? launch_pairs<OUT_E4M3, true>(tmA, tmW, p, st) : launch_pairs<OUT_E4M3, false>(tmA, tmW, p, st);
    }
    // The weights as the 128 rows of a tile, tokens as its columns: always up to 64 tokens; with more, 64 at a time, where that is at
    // most one tile per SM and at most eight blocks of k per CTA: what takes time then is the output, of which a CTA has half
    // as much (197 x 2304 x 768 8.6 -> 7.2 us, 582 x 1000 x 494 8.3 -> 6.8; 256 x 4096 x 4096, 32 blocks, 16.4 -> 20.1).
    const long long small_tiles = (long long)((N + BP - 1) / BP) * ((M + 63) / 64);
    const bool swap = M <= 64 || (small_tiles <= device_sms() && p.blocks <= 8 * splits_of(small_tiles, p.blocks));
    const int bn = !swap ? 128 : M <= 16 ? 16 : M <= 32 ? 32 : 64;
    CUtensorMap tmP, tmQ;
    if (!encode_rows(&tmP, swap ? w : a, swap ? N : M, K, swap ? ldw : lda, BP)) return CONVNN_E_CUDA;
    if (!encode_rows(&tmQ, swap ? a : w, swap ? M : N, K, swap ? lda : ldw, bn)) return CONVNN_E_CUDA;
    if (bn == 16) return launch_tiles<16, true>(tmP, tmQ, p, st);
    if (bn == 32) return launch_tiles<32, true>(tmP, tmQ, p, st);
    if (bn == 64) return launch_tiles<64, true>(tmP, tmQ, p, st);
    return launch_tiles<128, false>(tmP, tmQ, p, st);
}

int read_linear_fp8_status(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_linear_fp8_status, sizeof(int));
    if (e != cudaSuccess) return set_error(CONVNN_E_CUDA, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(e));
    *out = v;
    return CONVNN_OK;
}

}  // namespace convnn
