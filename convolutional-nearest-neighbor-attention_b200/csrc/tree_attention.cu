// Attention of a tree of drafted tokens over a paged cache (one token per sequence: ordinary decoding).
//   s_ij = scale * q_i . k_j over the cached entries j < length and those drafted tokens whose bit is set in i's mask
//   out_i = sum_j 2^(s_ij log2(e) - m_i) v_j / sum_j 2^(s_ij log2(e) - m_i);  nothing to attend to: zeros
// One pass over the keys with a running maximum and sum in float32.  The query heads that share a key head, for all of a sequence's
// tokens, are the rows of one product, so that keys and values are read once.  With few rows reading them is all that takes time.
//
// rows_kernel (bfloat16, up to 16 rows): mma.sync.  Each of four warps walks every fourth slice of 16 keys by itself, copies of its next
// slices in flight, and the four join at the unit's end: no barrier between slices.  48 sequences of 4096 to 16384 entries, 8 key heads of
// 128: 308 us for 1.87 GB, 6.05 TB/s (92 % of a plain copy's rate; 5.4 after a second of it, when the clock falls to 1700 MHz).  Three slices
// in flight per warp instead of two (the queries' room for the warps' sums) gain nothing: 324 us; pages asked for a slice ahead 316.
// scalar_kernel (float32): 16 rows on the fp32 pipes, tiles of 32 keys through a ring of the whole CTA, four rows by four keys or channels a
// thread; 64 units of 4096 entries of 128 channels 81 us, twice what their bytes take.  Three barriers a tile are what is waited for.
// tree_attention_tc.cu (bfloat16, more rows, up to 128 channels, pages of a multiple of 16 entries): tcgen05.  16 sequences of 32 to 64 tokens, 32
// query heads: 1536 us with rows_kernel, 16 rows at a time.
// join_kernel: units that several CTAs had, and rows without anything.
// Where the cache is short, the second kernel costs more than the even division gains: a cluster of up to sixteen CTAs has a unit, and they
// join through their shared memories (one token of 12 heads over 1000 entries: 10.6 us with two kernels, 5.6 in one, of which 0.6 us
// are each of the lengths, the table and the first keys, read one after the other).  The host goes by what the tables could hold: a table
// 64 times as wide as those entries need is divided evenly (9.3 us).
#include <math.h>

#include <type_traits>

#include "paged_attention.cuh"
#include "sm100.cuh"

namespace convnn {
namespace {

using namespace paged;

constexpr int ROWS = 16, kThreads = 128, kWarps = 4;

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 16 bytes, zeros where there is nothing to copy.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two values >= 0 as the next bfloat16 below them, and what is left as bfloat16: off by 2^-15 of the value (a step is 2^-7, half a step of
// the rest 2^-8 of it).  Below, not nearest: neither part of a value above zero is zero or negative, so that an infinite value in the
// product stays what it is.
__device__ __forceinline__ uint32_t split2(float x, float y, uint32_t& rest) {
    const uint32_t hx = max(__float_as_uint(x), 1u) - 1u, hy = max(__float_as_uint(y), 1u) - 1u;
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x - __uint_as_float(hx & 0xffff0000u), y - __uint_as_float(hy & 0xffff0000u));
    rest = *reinterpret_cast<const uint32_t*>(&lo);
    return __byte_perm(hx, hy, 0x7632);
}

__device__ __forceinline__ void push4(uint32_t at, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void push2(uint32_t at, float x, float y) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
template <typename T>
__device__ __forceinline__ void write_four(const Params& p, const Sequence& s, int b, int h, int row, int col, const float4& sum, float inv,
                                           bool bad) {
    const int t = row / p.G, g = row - t * p.G;
    float x[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
    if (bad) {
        const unsigned long long mask = seen_by(p, s, b, row);
        for (int e = 0; e < 4; ++e) x[e] += not_finite_seen<T>(p, s, b, h, mask, col + e);
    }
    T* out = static_cast<T*>(p.out) + b * p.os[0] + t * p.os[1] + (h * p.G + g) * p.os[2] + col;
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
        __nv_bfloat162 w[2] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3])};
        *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(w);
    }
}
constexpr int MOST_PARTS = 16;
// Bytes that join_cluster() needs for `fours` groups of four channels.
__host__ __device__ inline int join_bytes(int fours) { return (ROWS * fours + MOST_PARTS) * 24 + 4 * MOST_PARTS; }
// The whole cluster, behind a cluster_arrive() at the kernel's start: joins the parts of the unit's rows and writes them, zeros where a
// row is not there or attends to nothing.  Every CTA has an even share of the groups of four channels of all rows, and the others
// store theirs into its memory (`room`), which nobody waits for; reading them instead, 64 loads one after the other, took 4 us.
// part_of(row, four, sums, maximum, sum of weights) says what this CTA has.
template <typename T, typename F>
__device__ __forceinline__ void join_cluster(const Params& p, const Sequence& s, int b, int h, int rt, uint8_t* room, bool bad, const F& part_of) {
    const int part = blockIdx.x % p.split, fours = p.D / 4, items = min(ROWS, p.T * p.G - rt * ROWS) * fours;
    const int share = (items + p.split - 1) / p.split, all = share * p.split;
    const uint32_t sums = smem_at(room), weights = sums + 16 * all, bads = weights + 8 * all;
    cluster_wait();                                                  // (the others run)
    for (int i = threadIdx.x; i < items; i += blockDim.x) {
        const int owner = i / share, at = part * share + i - owner * share, r = i / fours;
        float4 x;
        float m, l;
        part_of(r, i - r * fours, x, m, l);
        push4(sm100::map_to_cta(sums, owner) + 16 * at, x);
        push2(sm100::map_to_cta(weights, owner) + 8 * at, m, l);
    }
    if (threadIdx.x < p.split) sm100::st_cluster_u32(sm100::map_to_cta(bads, threadIdx.x) + 4 * part, bad);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const float4* got = reinterpret_cast<const float4*>(room);
    const float2* got_weights = reinterpret_cast<const float2*>(got + all);
    const uint32_t* got_bads = reinterpret_cast<const uint32_t*>(got_weights + all);
    for (int j = threadIdx.x; j < share && part * share + j < items; j += blockDim.x) {
        const int i = part * share + j, r = i / fours, row = rt * ROWS + r;
        float top = -CUDART_INF_F, sum = 0.f;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        bool any_bad = false;
        if (row < s.count * p.G) {
            for (int c = 0; c < p.split; ++c) top = fmaxf(top, got_weights[c * share + j].x);
#pragma unroll 4
            for (int c = 0; c < p.split; ++c) {
                const float2 w = got_weights[c * share + j];
                const float4 x = got[c * share + j];
                const float f = w.x == top ? 1.f : ex2(w.x - top);   // (nothing anywhere: zeros, once each)
                sum = fmaf(w.y, f, sum);
                y.x = fmaf(x.x, f, y.x); y.y = fmaf(x.y, f, y.y);
                y.z = fmaf(x.z, f, y.z); y.w = fmaf(x.w, f, y.w);
                any_bad |= got_bads[c] != 0;
            }
        }
        write_four<T>(p, s, b, h, row, 4 * (i - r * fours), y, inverse_of(p, s, b, row, sum), any_bad);
    }
}
// A part without keys.
struct NoPart {
    __device__ __forceinline__ void operator()(int, int, float4& x, float& m, float& l) const {
        x = make_float4(0.f, 0.f, 0.f, 0.f);
        m = -CUDART_INF_F;
        l = 0.f;
    }
};

// ---- bfloat16: 16 rows a tile on mma.sync ---------------------------------------------------------------------------------------

// DS steps of 16 channels (D rounded up; the channels behind D are zeros), STAGES slices in flight per warp.
template <int DS, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(kThreads) rows_kernel(const Params p) {
    constexpr int DP = 16 * DS, CH = DP / 8, PITCH = (CH | 1) * 16;      // an odd number of 16-byte columns: no bank conflicts
    constexpr int SLICE = 16 * PITCH, STAGE = 2 * SLICE, OP = DP + 8;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* sQ = smem;                                                  // [16][PITCH]
    float* sO = reinterpret_cast<float*>(sQ + SLICE);                    // [16][OP]: one warp's sums on their way to the next
    float* sM = sO + ROWS * OP;                                          // [4][16] maxima
    float* sL = sM + kWarps * ROWS;                                      // [16] sums
    int* sBad = reinterpret_cast<int*>(sL + ROWS);
    uint8_t* ring = reinterpret_cast<uint8_t*>(sBad + 4);
    uint8_t* room = ring + kWarps * STAGES * STAGE;                      // (SPLIT)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t own = smem_at(ring) + warp * (STAGES * STAGE);

    if (p.D != DP) {                                                     // channels behind D are zeros
        for (int i = threadIdx.x; i < (SLICE + kWarps * STAGES * STAGE) / 16; i += kThreads) {
            uint8_t* at = i < SLICE / 16 ? sQ + 16 * i : ring + 16 * (i - SLICE / 16);
            *reinterpret_cast<uint4*>(at) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }
    if (SPLIT) cluster_arrive();
    chain_begin();

    Cursor at;
    if (SPLIT) at.start_part(p, blockIdx.x);
    else at.start(p, blockIdx.x);
    if (at.left == 0) {                                                  // (the whole CTA)
        if (SPLIT) join_cluster<__nv_bfloat16>(p, at.s, at.b, at.h, at.rt, room, false, NoPart());
        return;
    }
    Cursor ahead = at;
    const int chunks = p.D / 8;
    // a slice lies in one page, where its rows' distances fit 32 bits
    const bool one_page = p.page_size % 16 == 0 && p.ks[2] < (1 << 26) && p.vs[2] < (1 << 26);
    const int k_row = (int)p.ks[2], v_row = (int)p.vs[2];

    // The page of a lane's row of this warp's slice of ahead's tile; lanes 16 apart have one row.  In a cluster it is asked for a slice before
    // it is copied, in the even division where it is (sooner is slower there, see above).
    int next_row = 0, next_page = -1;
    auto look_up = [&]() {
        const int first = ahead.tile * 64 + warp * 16, entry = one_page ? first : first + (lane & 15), slot = p.slot_at(entry);
        next_page = -1;
        next_row = entry - slot * p.page_size + (one_page ? lane & 15 : 0);
        if (ahead.left > 0 && entry < ahead.s.total) next_page = p.table[ahead.b * p.table_stride + slot];
    };
    // this warp's slice of ahead's tile into `stage`
    auto fetch = [&](int stage) {
        if (!SPLIT) look_up();
        if (ahead.left > 0) {
            const int first = ahead.tile * 64 + warp * 16;
            const bool any = first < ahead.s.total, there = (unsigned)next_page < (unsigned)p.pages && first + (lane & 15) < ahead.s.total;
            const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(p.k) + ahead.h * p.ks[1];
            const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(p.v) + ahead.h * p.vs[1];
            const uint32_t dst = own + stage * STAGE;
            if (one_page && !SPLIT) {
                // one place for all rows, and what lies between them and their columns does not change (48 sequences 391 -> 380 us; in a cluster,
                // whose CTAs are few, all copies of a slice at once take longer: 8 units of 4096 entries 28.4 -> 32.6)
                const int page = (unsigned)next_page < (unsigned)p.pages ? next_page : -1, row = next_row - (lane & 15);
                const int rows = page < 0 ? 0 : ahead.s.total - first;
                if (page >= 0) {
                    k += page * p.ks[0] + row * p.ks[2];
                    v += page * p.vs[0] + row * p.vs[2];
                }
                ahead.next(p);
                if (rows >= 16) {
#pragma unroll
                    for (int i = 0; i < DS; ++i) {
                        const int c = i * 32 + lane, r = c / CH, col = c - r * CH;
                        if (col < chunks) {
                            copy16(dst + r * PITCH + col * 16, k + (r * k_row + col * 8), true);
                            copy16(dst + SLICE + r * PITCH + col * 16, v + (r * v_row + col * 8), true);
                        }
                    }
                } else if (any) {
#pragma unroll
                    for (int i = 0; i < DS; ++i) {
                        const int c = i * 32 + lane, r = c / CH, col = c - r * CH;
                        if (col < chunks) {
                            copy16(dst + r * PITCH + col * 16, k + (r < rows ? r * k_row + col * 8 : 0), r < rows);
                            copy16(dst + SLICE + r * PITCH + col * 16, v + (r < rows ? r * v_row + col * 8 : 0), r < rows);
                        }
                    }
                }
            } else {
                const long long kr = there ? next_page * p.ks[0] + next_row * p.ks[2] : 0, vr = there ? next_page * p.vs[0] + next_row * p.vs[2] : 0;
                ahead.next(p);
                if (SPLIT) look_up();
                if (any) {
#pragma unroll
                    for (int i = 0; i < DS; ++i) {
                        const int c = i * 32 + lane, r = c / CH, col = c - r * CH;
                        const long long ko = __shfl_sync(0xffffffffu, kr, r), vo = __shfl_sync(0xffffffffu, vr, r);
                        const bool copied = __shfl_sync(0xffffffffu, (int)there, r);
                        if (col < chunks) {
                            copy16(dst + r * PITCH + col * 16, k + ko + col * 8, copied);
                            copy16(dst + SLICE + r * PITCH + col * 16, v + vo + col * 8, copied);
                        }
                    }
                }
            }
        }
        copies_end();
    };
    if (SPLIT) look_up();
    // the rows of q (zeros where a token is not there), with the first slice's copies where there is one unit
    auto copy_rows = [&]() {
        for (int i = threadIdx.x; i < ROWS * chunks; i += kThreads) {
            const int r = i / chunks, col = i - r * chunks, row = at.rt * ROWS + r, t = row / p.G;
            const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q);
            if (t < at.s.count) q += at.b * p.qs[0] + t * p.qs[1] + (at.h * p.G + row - t * p.G) * p.qs[2] + col * 8;
            copy16(smem_at(sQ) + r * PITCH + col * 16, q, t < at.s.count);
        }
    };
    if (SPLIT) copy_rows();
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);

    const uint32_t q_at = smem_at(sQ) + (lane & 15) * PITCH + (lane >> 4) * 16;
    const uint32_t k_lane = ((lane & 7) + (lane >> 4) * 8) * PITCH + ((lane >> 3) & 1) * 16;
    const uint32_t v_lane = ((lane & 7) + ((lane >> 3) & 1) * 8) * PITCH + (lane >> 4) * 16;
    int stage = 0;
    bool first_unit = true;
    while (at.left > 0) {
        // ---- a unit: its rows
        const Sequence s = at.s;
        const int b = at.b, h = at.h, row0 = at.rt * ROWS, tile0 = at.tile;
        if (!SPLIT)
            for (int i = threadIdx.x; i < ROWS * chunks; i += kThreads) {
                const int r = i / chunks, col = i - r * chunks, t = (row0 + r) / p.G, g = row0 + r - t * p.G;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (t < s.count)
                    v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + b * p.qs[0] + t * p.qs[1] +
                                                        (h * p.G + g) * p.qs[2] + col * 8);
                *reinterpret_cast<uint4*>(sQ + r * PITCH + col * 16) = v;
            }
        if (threadIdx.x == 0) *sBad = 0;
        const unsigned long long mask0 = seen_by(p, s, b, row0 + lane / 4), mask1 = seen_by(p, s, b, row0 + lane / 4 + 8);
        if (SPLIT) copies_wait<STAGES - 2>();
        __syncthreads();
        float o[2 * DS][4], m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int n = 0; n < 2 * DS; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
        bool bad = false, end, at_end;
        do {
            // ---- a tile: this warp's slice of it
            fetch(stage == 0 ? STAGES - 1 : stage - 1);
            copies_wait<STAGES - 1>();
            __syncwarp();
            const int first = at.tile * 64 + warp * 16;
            if (first < s.total) {
                const uint32_t sk = own + stage * STAGE + k_lane, sv = own + stage * STAGE + SLICE + v_lane;
                float c[2][4] = {};
#pragma unroll
                for (int d = 0; d < DS; ++d) {
                    uint32_t qa[4], kb[4];
                    ldsm4(qa, q_at + d * 32);
                    ldsm4(kb, sk + d * 32);
                    mma(c[0], qa, kb[0], kb[1]);
                    mma(c[1], qa, kb[2], kb[3]);
                }
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[n][e] *= p.scale_log2;
                if (first + 16 > s.length) {
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = first + n * 8 + (lane & 3) * 2 + (e & 1) - s.length;
                            const bool seen = j < 0 || (j < s.total - s.length && ((e < 2 ? mask0 : mask1) >> j & 1));
                            if (!seen) c[n][e] = -CUDART_INF_F;
                        }
                    // what is not finite among the drafted tokens' values: a zero in its place, for now
                    const int lr = lane & 15;
                    if (first + lr >= s.length) {
                        uint8_t* row = ring + warp * (STAGES * STAGE) + stage * STAGE + SLICE + lr * PITCH;
                        for (int col = lane >> 4; col < chunks; col += 2) {
                            uint4* w = reinterpret_cast<uint4*>(row + col * 16);
                            uint32_t x[4] = {w->x, w->y, w->z, w->w};
                            bool hit = false;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if ((x[e] & 0x7f80u) == 0x7f80u) { x[e] &= 0xffff0000u; hit = true; }
                                if ((x[e] & 0x7f800000u) == 0x7f800000u) { x[e] &= 0xffffu; hit = true; }
                            }
                            if (hit) {
                                *w = make_uint4(x[0], x[1], x[2], x[3]);
                                bad = true;
                            }
                        }
                    }
                    __syncwarp();
                }
                float x0 = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1]));
                float x1 = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
#pragma unroll
                for (int w = 1; w <= 2; w <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, w));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, w));
                }
                if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
                    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
                    const float f0 = m0 == n0 ? 1.f : ex2(m0 - n0), f1 = m1 == n1 ? 1.f : ex2(m1 - n1);
                    m0 = n0; m1 = n1;
                    l0 *= f0; l1 *= f1;
#pragma unroll
                    for (int n = 0; n < 2 * DS; ++n) {
                        o[n][0] *= f0; o[n][1] *= f0;
                        o[n][2] *= f1; o[n][3] *= f1;
                    }
                }
                const float z0 = m0 == -CUDART_INF_F ? 0.f : m0, z1 = m1 == -CUDART_INF_F ? 0.f : m1;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    c[n][0] = ex2(c[n][0] - z0); c[n][1] = ex2(c[n][1] - z0);
                    c[n][2] = ex2(c[n][2] - z1); c[n][3] = ex2(c[n][3] - z1);
                    l0 += c[n][0] + c[n][1];
                    l1 += c[n][2] + c[n][3];
                }
                // The weights as the sum of two bfloat16: a rounding to one would cost as much as the result's own, and the second
                // product is free while memory is what is waited for.
                uint32_t pa[4], pr[4];
                pa[0] = split2(c[0][0], c[0][1], pr[0]);
                pa[1] = split2(c[0][2], c[0][3], pr[1]);
                pa[2] = split2(c[1][0], c[1][1], pr[2]);
                pa[3] = split2(c[1][2], c[1][3], pr[3]);
#pragma unroll
                for (int d = 0; d < DS; ++d) {
                    uint32_t vb[4];
                    ldsm4_t(vb, sv + d * 32);
                    mma(o[2 * d], pa, vb[0], vb[1]);
                    mma(o[2 * d + 1], pa, vb[2], vb[3]);
                    mma(o[2 * d], pr, vb[0], vb[1]);
                    mma(o[2 * d + 1], pr, vb[2], vb[3]);
                }
                __syncwarp();                                            // (the stage is filled again)
            }
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            end = at.last_of_unit();
            at_end = at.tile + 1 == s.tiles;
            at.next(p);
        } while (!end);

        // ---- the four warps' sums: maxima first, then one after the other
        if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(sBad, 1);
#pragma unroll
        for (int w = 1; w <= 2; w <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, w);
            l1 += __shfl_xor_sync(0xffffffffu, l1, w);
        }
        const int r0 = lane / 4, r1 = r0 + 8;
        if ((lane & 3) == 0) {
            sM[warp * ROWS + r0] = m0;
            sM[warp * ROWS + r1] = m1;
        }
        if (SPLIT) {
            // one unit: the ring is free, a warp's own part of it takes its sums
            float* mine = reinterpret_cast<float*>(ring + warp * (STAGES * STAGE));
            __syncwarp();
#pragma unroll
            for (int n = 0; n < 2 * DS; ++n) {
                *reinterpret_cast<float2*>(mine + r0 * OP + n * 8 + (lane & 3) * 2) = make_float2(o[n][0], o[n][1]);
                *reinterpret_cast<float2*>(mine + r1 * OP + n * 8 + (lane & 3) * 2) = make_float2(o[n][2], o[n][3]);
            }
            if ((lane & 3) == 0) {
                sO[warp * ROWS + r0] = l0;
                sO[warp * ROWS + r1] = l1;
            }
            __syncthreads();
            join_cluster<__nv_bfloat16>(p, s, b, h, row0 / ROWS, room, *sBad != 0, [&](int r, int four, float4& x, float& m, float& l) {
                m = fmaxf(fmaxf(sM[r], sM[ROWS + r]), fmaxf(sM[2 * ROWS + r], sM[3 * ROWS + r]));
                x = make_float4(0.f, 0.f, 0.f, 0.f);
                l = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float4 y = *reinterpret_cast<const float4*>(ring + w * (STAGES * STAGE) + 4 * (r * OP + 4 * four));
                    const float f = sM[w * ROWS + r] == m ? 1.f : ex2(sM[w * ROWS + r] - m);
                    l = fmaf(sO[w * ROWS + r], f, l);
                    x.x = fmaf(y.x, f, x.x); x.y = fmaf(y.y, f, x.y);
                    x.z = fmaf(y.z, f, x.z); x.w = fmaf(y.w, f, x.w);
                }
            });
            break;
        }
        __syncthreads();
        float t0 = sM[r0], t1 = sM[r1];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            t0 = fmaxf(t0, sM[w * ROWS + r0]);
            t1 = fmaxf(t1, sM[w * ROWS + r1]);
        }
        const float f0 = m0 == -CUDART_INF_F ? 0.f : ex2(m0 - t0), f1 = m1 == -CUDART_INF_F ? 0.f : ex2(m1 - t1);
        l0 *= f0; l1 *= f1;
#pragma unroll 1
        for (int w = kWarps - 1; w >= 0; --w) {
            if (warp == w) {
#pragma unroll
                for (int n = 0; n < 2 * DS; ++n) {
                    float2* y0 = reinterpret_cast<float2*>(sO + r0 * OP + n * 8 + (lane & 3) * 2);
                    float2* y1 = reinterpret_cast<float2*>(sO + r1 * OP + n * 8 + (lane & 3) * 2);
                    // (what no key of this warp went into is zero times a factor of zero)
                    float2 a = make_float2(o[n][0] * f0, o[n][1] * f0), c = make_float2(o[n][2] * f1, o[n][3] * f1);
                    if (w != kWarps - 1) {
                        const float2 u = *y0, v = *y1;
                        a.x += u.x; a.y += u.y;
                        c.x += v.x; c.y += v.y;
                    }
                    *y0 = a;
                    *y1 = c;
                }
                if ((lane & 3) == 0) {
                    sL[r0] = w == kWarps - 1 ? l0 : sL[r0] + l0;
                    sL[r1] = w == kWarps - 1 ? l1 : sL[r1] + l1;
                }
            }
            __syncthreads();
        }
        // ---- handed on, or the result
        const bool whole = tile0 == 0 && at_end;
        float* slot = slot_of(p, blockIdx.x, first_unit);
        const bool any_bad = *sBad;
        for (int i = threadIdx.x; i < ROWS * chunks; i += kThreads) {
            const int r = i / chunks, col = i - r * chunks;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = sO[r * OP + col * 8 + e];
            if (whole) {
                const int t = (row0 + r) / p.G, g = row0 + r - t * p.G;
                if (t >= s.count) continue;
                const float inv = inverse_of(p, s, b, row0 + r, sL[r]);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] *= inv;
                if (any_bad) {
                    const unsigned long long mask = seen_by(p, s, b, row0 + r);
                    for (int e = 0; e < 8; ++e) y[e] += not_finite_seen<__nv_bfloat16>(p, s, b, h, mask, col * 8 + e);
                }
                __nv_bfloat162 w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = __floats2bfloat162_rn(y[2 * e], y[2 * e + 1]);
                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + b * p.os[0] + t * p.os[1] + (h * p.G + g) * p.os[2] +
                                          col * 8) = *reinterpret_cast<uint4*>(w);
            } else {
                float4* dst = reinterpret_cast<float4*>(slot + r * p.D + col * 8);
                dst[0] = make_float4(y[0], y[1], y[2], y[3]);
                dst[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
        }
        if (!whole) {
            float* tail = slot + ROWS * p.D;
            if (threadIdx.x < ROWS) {
                const int r = threadIdx.x;
                tail[r] = fmaxf(fmaxf(sM[r], sM[ROWS + r]), fmaxf(sM[2 * ROWS + r], sM[3 * ROWS + r]));
                tail[ROWS + r] = sL[r];
            }
            if (threadIdx.x == 0) tail[2 * ROWS] = any_bad ? 1.f : 0.f;
        }
        first_unit = false;
        __syncthreads();                                                 // (sQ, sO, sM, sL of the next unit)
    }
    copies_wait<0>();
}

// ---- float32: 16 rows a tile on the fp32 pipes ----------------------------------------------------------------------------------

// Scores: every warp all 16 x 32 of them, over a part of the channels (a lane four rows by four keys: eight reads of 16 bytes, one
// wavefront each, for 64 multiply-adds), added by the warp that owns the row, two a warp, a lane a key.  Sums: a lane four rows by four
// channels, a warp eight such columns, warps that are left over another part of the keys.  A lane with one key or one group of channels for
// all its rows reads five times as much of shared memory, which then is all that takes time: 4900 cycles a tile of 80 channels.
constexpr int SW = 8, kScalarThreads = 32 * SW, TILE = 32, SP = 40, PP = 36;   // pitches of the scores and of the weights
template <int STAGES, bool SPLIT>
__global__ void __launch_bounds__(kScalarThreads) scalar_kernel(const Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    const int pitch = p.D + 4;                                           // floats (rows start on 16-byte boundaries: D is a multiple of 4)
    const int pieces = p.D / 4;
    float* sQ = reinterpret_cast<float*>(smem);                          // [16][pitch]
    float* sS = sQ + ROWS * pitch;                                       // [8][16][SP]
    float* sP = sS + SW * ROWS * SP;                                     // [16][PP]
    float *sF = sP + ROWS * PP, *sTop = sF + ROWS, *sSum = sTop + ROWS;  // [16] each
    int* sBad = reinterpret_cast<int*>(sSum + ROWS);                     // (4 words)
    float* ring = sSum + ROWS + 4;
    const int stage_floats = 2 * TILE * pitch;
    uint8_t* room = reinterpret_cast<uint8_t*>(ring + STAGES * stage_floats);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lr = lane >> 3, lc = lane & 7;   // rows lr + 4 i
    const int columns = (pieces + 7) / 8, parts = SW / columns;          // warps over the channels; parts of the keys
    const int my_part = warp / columns, col = (warp - my_part * columns) * 8 + lc;
    const bool sums_here = my_part < parts && col < pieces;
    const int keys = TILE / parts / 4 * 4, key0 = my_part * keys, key1 = my_part + 1 == parts ? TILE : key0 + keys;
    if (SPLIT) cluster_arrive();
    chain_begin();

    Cursor at;
    if (SPLIT) at.start_part(p, blockIdx.x);
    else at.start(p, blockIdx.x);
    if (at.left == 0) {
        if (SPLIT) join_cluster<float>(p, at.s, at.b, at.h, at.rt, room, false, NoPart());
        return;
    }
    Cursor ahead = at;
    // The page of this thread's row (eight threads a row) of ahead's tile is asked for a tile before its row is copied.
    int next_row = 0, next_page = -1;
    auto look_up = [&]() {
        const int entry = ahead.tile * TILE + (threadIdx.x >> 3), slot = p.slot_at(entry);
        next_page = -1;
        next_row = entry - slot * p.page_size;
        if (ahead.left > 0 && entry < ahead.s.total) next_page = p.table[ahead.b * p.table_stride + slot];
    };
    auto fetch = [&](int stage) {
        if (ahead.left > 0) {
            const bool there = (unsigned)next_page < (unsigned)p.pages;
            const long long page = there ? next_page : 0, row = there ? next_row : 0;
            const float* k = static_cast<const float*>(p.k) + ahead.h * p.ks[1] + page * p.ks[0] + row * p.ks[2];
            const float* v = static_cast<const float*>(p.v) + ahead.h * p.vs[1] + page * p.vs[0] + row * p.vs[2];
            const uint32_t dst = smem_at(ring + stage * stage_floats + (threadIdx.x >> 3) * pitch);
            ahead.next(p);
            look_up();
            for (int c = threadIdx.x & 7; c < pieces; c += 8) {
                copy16(dst + 16 * c, k + 4 * c, there);
                copy16(dst + 4 * TILE * pitch + 16 * c, v + 4 * c, there);
            }
        }
        copies_end();
    };
    look_up();
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);
    int stage = 0;
    bool first_unit = true;
    while (at.left > 0) {
        const Sequence s = at.s;
        const int b = at.b, h = at.h, row0 = at.rt * ROWS, tile0 = at.tile;
        for (int i = threadIdx.x; i < ROWS * pieces; i += kScalarThreads) {
            const int r = i / pieces, c = i - r * pieces, t = (row0 + r) / p.G, g = row0 + r - t * p.G;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (t < s.count)
                v = *reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + b * p.qs[0] + t * p.qs[1] +
                                                     (h * p.G + g) * p.qs[2] + c * 4);
            *reinterpret_cast<float4*>(sQ + r * pitch + c * 4) = v;
        }
        if (threadIdx.x == 0) *sBad = 0;
        const unsigned long long mask[2] = {seen_by(p, s, b, row0 + 2 * warp), seen_by(p, s, b, row0 + 2 * warp + 1)};
        float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
        float4 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int live = min(ROWS, s.count * p.G - row0);                // rows; of up to four a lane has one
        bool end, at_end;
        do {
            copies_wait<STAGES - 2>();
            __syncthreads();                                             // the tile is there, and the one before it read
            fetch(stage == 0 ? STAGES - 1 : stage - 1);
            const float* sk = ring + stage * stage_floats;
            float* sv = ring + stage * stage_floats + TILE * pitch;
            const bool drafts = at.tile * TILE + TILE > s.length;
            // what is not finite among the drafted tokens' values: a zero in its place, for now (read behind two more barriers)
            if (const int entry = at.tile * TILE + (threadIdx.x >> 3); drafts && entry >= s.length && entry < s.total) {
                for (int c = threadIdx.x & 7; c < pieces; c += 8) {
                    float4* at16 = reinterpret_cast<float4*>(sv + (threadIdx.x >> 3) * pitch + 4 * c);
                    const float4 v = *at16;
                    if (isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w)) continue;
                    *at16 = make_float4(isfinite(v.x) ? v.x : 0.f, isfinite(v.y) ? v.y : 0.f, isfinite(v.z) ? v.z : 0.f,
                                        isfinite(v.w) ? v.w : 0.f);
                    *sBad = 1;
                }
            }
            auto scores = [&](auto rows) {
                constexpr int R = decltype(rows)::value;
                float c[R][4] = {};
#pragma unroll 2
                for (int d = warp; d < pieces; d += SW) {
                    float4 q[R], k[4];
#pragma unroll
                    for (int i = 0; i < R; ++i) q[i] = *reinterpret_cast<const float4*>(sQ + (lr + 4 * i) * pitch + 4 * d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const float4*>(sk + (lc + 8 * i) * pitch + 4 * d);
#pragma unroll
                    for (int i = 0; i < R; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            c[i][j] = fmaf(q[i].x, k[j].x, c[i][j]);
                            c[i][j] = fmaf(q[i].y, k[j].y, c[i][j]);
                            c[i][j] = fmaf(q[i].z, k[j].z, c[i][j]);
                            c[i][j] = fmaf(q[i].w, k[j].w, c[i][j]);
                        }
                }
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sS[(warp * ROWS + lr + 4 * i) * SP + lc + 8 * j] = c[i][j];
            };
            if (live <= 4) scores(std::integral_constant<int, 1>());
            else scores(std::integral_constant<int, 4>());
            __syncthreads();
            const int j = at.tile * TILE + lane - s.length;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 2 * warp + i;
                if (r >= live) continue;
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < SW; ++w) x += sS[(w * ROWS + r) * SP + lane];
                x *= p.scale_log2;
                if (drafts && j >= 0 && !(j < s.total - s.length && (mask[i] >> j & 1))) x = -CUDART_INF_F;
                float top = x;
#pragma unroll
                for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                const float n = fmaxf(m[i], top), f = m[i] == n ? 1.f : ex2(m[i] - n);
                m[i] = n;
                const float w = ex2(x - (n == -CUDART_INF_F ? 0.f : n));
                l[i] = fmaf(l[i], f, w);
                sP[r * PP + lane] = w;
                if (lane == 0) sF[r] = f;
            }
            __syncthreads();
            auto sums = [&](auto rows) {
                constexpr int R = decltype(rows)::value;
                float4 part[R];                                          // (a tile's own, so that what is added to a long sum is not small)
                float f[R];
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    part[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    f[i] = sF[lr + 4 * i];
                }
#pragma unroll 2
                for (int e = key0; e < key1; e += 4) {
                    float4 w[R], v[4];
#pragma unroll
                    for (int i = 0; i < R; ++i) w[i] = *reinterpret_cast<const float4*>(sP + (lr + 4 * i) * PP + e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const float4*>(sv + (e + i) * pitch + 4 * col);
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        const float ws[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            part[i].x = fmaf(ws[x], v[x].x, part[i].x);
                            part[i].y = fmaf(ws[x], v[x].y, part[i].y);
                            part[i].z = fmaf(ws[x], v[x].z, part[i].z);
                            part[i].w = fmaf(ws[x], v[x].w, part[i].w);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    o[i].x = fmaf(o[i].x, f[i], part[i].x); o[i].y = fmaf(o[i].y, f[i], part[i].y);
                    o[i].z = fmaf(o[i].z, f[i], part[i].z); o[i].w = fmaf(o[i].w, f[i], part[i].w);
                }
            };
            if (sums_here) {
                if (live <= 4) sums(std::integral_constant<int, 1>());
                else sums(std::integral_constant<int, 4>());
            }
            stage = stage + 1 == STAGES ? 0 : stage + 1;
            end = at.last_of_unit();
            at_end = at.tile + 1 == s.tiles;
            at.next(p);
        } while (!end);

        // ---- the parts of the keys, then the unit
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
            if (lane == 0) {
                sTop[2 * warp + i] = m[i];
                sSum[2 * warp + i] = l[i];
            }
        }
        if (sums_here && my_part)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(sS + ((my_part - 1) * ROWS + lr + 4 * i) * p.D + 4 * col) = o[i];
        __syncthreads();                                                 // (the scores of the last tile are read)
        const bool whole = tile0 == 0 && at_end, any_bad = *sBad != 0;
        float* slot = slot_of(p, blockIdx.x, first_unit);
        if (sums_here && my_part == 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = lr + 4 * i, t = (row0 + r) / p.G, g = row0 + r - t * p.G;
                float4 y = o[i];
                for (int w = 0; w < parts - 1; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(sS + (w * ROWS + r) * p.D + 4 * col);
                    y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
                }
                if (SPLIT) {
                    *reinterpret_cast<float4*>(sQ + r * pitch + 4 * col) = y;        // (one unit: the queries are read)
                } else if (!whole) {
                    *reinterpret_cast<float4*>(slot + r * p.D + 4 * col) = y;
                } else if (t < s.count) {
                    const float inv = inverse_of(p, s, b, row0 + r, sSum[r]);
                    y.x *= inv; y.y *= inv; y.z *= inv; y.w *= inv;
                    if (any_bad) {
                        const unsigned long long seen = seen_by(p, s, b, row0 + r);
                        y.x += not_finite_seen<float>(p, s, b, h, seen, 4 * col);
                        y.y += not_finite_seen<float>(p, s, b, h, seen, 4 * col + 1);
                        y.z += not_finite_seen<float>(p, s, b, h, seen, 4 * col + 2);
                        y.w += not_finite_seen<float>(p, s, b, h, seen, 4 * col + 3);
                    }
                    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + b * p.os[0] + t * p.os[1] + (h * p.G + g) * p.os[2] +
                                               4 * col) = y;
                }
            }
        if (SPLIT) {
            __syncthreads();
            join_cluster<float>(p, s, b, h, row0 / ROWS, room, any_bad, [&](int r, int four, float4& x, float& m_, float& l_) {
                x = *reinterpret_cast<const float4*>(sQ + r * pitch + 4 * four);
                m_ = sTop[r];
                l_ = sSum[r];
            });
            break;
        }
        if (!whole && threadIdx.x < ROWS) {
            slot[ROWS * p.D + threadIdx.x] = sTop[threadIdx.x];
            slot[ROWS * p.D + ROWS + threadIdx.x] = sSum[threadIdx.x];
            if (threadIdx.x == 0) slot[ROWS * p.D + 2 * ROWS] = any_bad ? 1.f : 0.f;
        }
        first_unit = false;
        __syncthreads();                                                 // (sQ, sS, sTop, sSum)
    }
    copies_wait<0>();
}

// ---- units that several CTAs had ------------------------------------------------------------------------------------------------

// The pieces' sums, in the order of the keys, each multiplied by what its maximum is away from the largest so far.  What says which pieces
// there are, and which rows have none, is read while the kernel before is still at work (it does not write that); behind it a piece's
// maximum and sums are asked for together, several pieces at a time: one way to memory and back.

// The unit that is cut for the first time where CTA `cta`'s tiles begin: its pieces are c0 .. c1 (c0 == c1: there is none).
struct Cut {
    Sequence s;
    int b, h, rt, c0, c1;
    bool second;                                 // the first piece is its CTA's last unit
};
__device__ __forceinline__ Cut cut_at(const Params& p, int cta) {
    Cut u{};
    int none;
    const Division d(total_work(p, 0, none), p.ctas);
    if (cta < 1 || cta >= d.ctas) return u;
    Cursor at;
    at.find(p, d.first(cta), 1);
    const int begin = d.first(cta) - at.tile;
    if (!at.tile || d.cta_of(begin) != cta - 1) return u;
    u.s = at.s;
    u.b = at.b; u.h = at.h; u.rt = at.rt;
    u.c0 = cta - 1;
    u.c1 = d.cta_of(begin + at.s.tiles - 1);
    u.second = d.first(u.c0) < begin;
    return u;
}
// Rows without anything, of all sequences: zeros, by all warps of the grid.  (Up to 2^30 tokens are taken: with a step added they stay
// below 2^31.)
__device__ __forceinline__ int next_zero_row(const Params& p, int i) {
    const int blocks = gridDim.x * gridDim.y * gridDim.z;
    for (; i < p.B * p.T; i += blocks * kWarps) {
        const int b = i / p.T;
        const Sequence s = sequence_of(p, b);
        if (i - b * p.T >= s.count || !s.total) break;
    }
    return i;
}
__device__ __forceinline__ int first_zero_row(const Params& p) {
    return next_zero_row(p, ((blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * kWarps + (threadIdx.x >> 5));
}
template <typename T>
__device__ __forceinline__ void write_zeros(const Params& p, int i) {
    for (; i < p.B * p.T; i = next_zero_row(p, i + gridDim.x * gridDim.y * gridDim.z * kWarps)) {
        const int b = i / p.T;
        T* out = static_cast<T*>(p.out) + b * p.os[0] + (i - b * p.T) * p.os[1];
        for (int h = 0; h < p.Hk * p.G; ++h)
            for (int c = threadIdx.x & 31; c < p.D; c += 32) out[h * p.os[2] + c] = from_f32<T>(0.f);
    }
}
// Sums joined so far: N groups of four channels of one row.
template <int N>
struct Joined {
    float top, sum;
    float4 y[N];
    __device__ __forceinline__ Joined() : top(-INFINITY), sum(0.f) {
#pragma unroll
        for (int v = 0; v < N; ++v) y[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // (a part without keys, m = -inf, has zeros; so has what was joined before any)
    __device__ __forceinline__ void add(float m, float l, const float4 (&x)[N]) {
        const float now = fmaxf(top, m), before = top == now ? 1.f : ex2(top - now), f = m == now ? 1.f : ex2(m - now);
        top = now;
        sum = sum * before + l * f;
#pragma unroll
        for (int v = 0; v < N; ++v) {
            y[v].x = fmaf(x[v].x, f, y[v].x * before); y[v].y = fmaf(x[v].y, f, y[v].y * before);
            y[v].z = fmaf(x[v].z, f, y[v].z * before); y[v].w = fmaf(x[v].w, f, y[v].w * before);
        }
    }
};

// Tiles of 16 rows.  WARPS of a block's four warps share the pieces of a row: all four where units have several pieces each (a block per
// unit and row), else a warp goes through every fourth row of 16 of one unit (a block per boundary between two CTAs' tiles).
constexpr int JOIN_ROWS = 16;
template <typename T, int WARPS>
__global__ void __launch_bounds__(kThreads) join_kernel(const Params p) {
    __shared__ float4 sY[WARPS == 4 ? 4 : 1][2][32];
    __shared__ float sT[4][2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Cut u{};
    if (WARPS == 4) {
        int before;
        const int unit = blockIdx.x, rest = unit % (p.Hk * p.row_tiles);
        u.b = unit / (p.Hk * p.row_tiles);
        u.h = rest / p.row_tiles;
        u.rt = rest - u.h * p.row_tiles;
        u.s = sequence_of(p, u.b);
        const Division d(total_work(p, u.b, before), p.ctas);
        if (u.rt < u.s.row_tiles && u.s.tiles) {
            const int begin = before + (u.h * u.s.row_tiles + u.rt) * u.s.tiles;
            u.c0 = d.cta_of(begin);
            u.c1 = d.cta_of(begin + u.s.tiles - 1);
            u.second = d.first(u.c0) < begin;
        }
    } else {
        u = cut_at(p, blockIdx.x);
    }
    const int zero = first_zero_row(p);
    chain_begin();
    write_zeros<T>(p, zero);
    if (u.c0 == u.c1) return;                    // (written by its CTA, or not this block's)
    const int tail = p.rows_per_tile * p.D;
    const bool wide = p.D > 128;
#pragma unroll 1
    for (int i = 0; i < (WARPS == 4 ? 1 : JOIN_ROWS / kWarps); ++i) {
        const int r = WARPS == 4 ? blockIdx.y : blockIdx.y * JOIN_ROWS + i * kWarps + warp, row = u.rt * p.rows_per_tile + r;
        if (r >= p.rows_per_tile || row >= u.s.count * p.G) return;          // (the whole block, or a warp that meets no other)
        Joined<2> all;
        float bad = 0.f;
        constexpr int BATCH = 4;
#pragma unroll 1
        for (int c = u.c0 + (WARPS == 4 ? warp : 0); c <= u.c1; c += WARPS * BATCH) {
            float m[BATCH], l[BATCH], hit[BATCH];
            float4 x[BATCH][2];
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int at = c + e * WARPS;
                m[e] = -CUDART_INF_F;
                l[e] = hit[e] = 0.f;
                x[e][0] = x[e][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (at > u.c1) continue;
                const float* from = slot_of(p, at, at > u.c0 || !u.second);
                m[e] = from[tail + r];
                l[e] = from[tail + p.rows_per_tile + r];
                hit[e] = from[tail + 2 * p.rows_per_tile];
                if (4 * lane < p.D) x[e][0] = *reinterpret_cast<const float4*>(from + r * p.D + 4 * lane);
                if (wide && 4 * lane + 128 < p.D) x[e][1] = *reinterpret_cast<const float4*>(from + r * p.D + 4 * lane + 128);
            }
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                all.add(m[e], l[e], x[e]);
                bad += hit[e];
            }
        }
        if (WARPS == 4) {
            sY[warp][0][lane] = all.y[0];
            sY[warp][1][lane] = all.y[1];
            if (lane == 0) {
                sT[warp][0] = all.top;
                sT[warp][1] = all.sum;
            }
            bad = __syncthreads_or(bad != 0.f) ? 1.f : 0.f;
            if (warp) return;
            all = Joined<2>();
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float4 x[2] = {sY[w][0][lane], sY[w][1][lane]};
                all.add(sT[w][0], sT[w][1], x);
            }
        }
        const float inv = inverse_of(p, u.s, u.b, row, all.sum);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int col = 4 * (lane + 32 * v);
            if (col < p.D) write_four<T>(p, u.s, u.b, u.h, row, col, all.y[v], inv, bad != 0.f);
        }
    }
}

// Tiles of 128 rows and more: a block per boundary, 128 rows and 16 channels, a thread a row (its neighbours' sums lie beside its own).  Four
// pieces are asked for at once: units of few tiles lie on many CTAs (8 units of 27 tiles, 18 pieces each, 52 us with a piece after the other).
__global__ void __launch_bounds__(kThreads) join_tiles_kernel(const Params p) {
    constexpr int FOURS = 4, BATCH = 4;
    const Cut u = cut_at(p, blockIdx.x);
    const int zero = first_zero_row(p);
    chain_begin();
    write_zeros<__nv_bfloat16>(p, zero);
    const int r = blockIdx.y * 128 + threadIdx.x, row = u.rt * p.rows_per_tile + r;
    if (u.c0 == u.c1 || row >= u.s.count * p.G) return;
    const int tail = p.rows_per_tile * p.D;
    Joined<FOURS> all;
    bool bad = false;
#pragma unroll 1
    for (int c = u.c0; c <= u.c1; c += BATCH) {
        float m[BATCH], l[BATCH], hit[BATCH];
        float4 x[BATCH][FOURS];
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
            m[e] = -CUDART_INF_F;
            l[e] = hit[e] = 0.f;
#pragma unroll
            for (int v = 0; v < FOURS; ++v) x[e][v] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (c + e > u.c1) continue;
            const float* from = slot_of(p, c + e, c + e > u.c0 || !u.second);
            m[e] = from[tail + r];
            l[e] = from[tail + p.rows_per_tile + r];
            hit[e] = from[tail + 2 * p.rows_per_tile + (r >> 7)];            // (a word for every 128 rows)
#pragma unroll
            for (int v = 0; v < FOURS; ++v) {
                const int four = blockIdx.z * FOURS + v;
                if (4 * four < p.D) x[e][v] = reinterpret_cast<const float4*>(from)[four * p.rows_per_tile + r];
            }
        }
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
            all.add(m[e], l[e], x[e]);
            bad |= hit[e] != 0.f;
        }
    }
    const float inv = inverse_of(p, u.s, u.b, row, all.sum);
#pragma unroll
    for (int v = 0; v < FOURS; ++v) {
        const int col = (blockIdx.z * FOURS + v) * 4;
        if (col < p.D) write_four<__nv_bfloat16>(p, u.s, u.b, u.h, row, col, all.y[v], inv, bad);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------

struct Plan {
    bool tiles;                          // on the tensor cores, 128 rows a tile
    int rows_per_tile, tile, stages, ctas_per_sm;
    size_t smem;
};

constexpr int kStepsBuilt[] = {4, 5, 6, 8, 12, 16};
int steps_of(int D) {
    for (int s : kStepsBuilt)
        if (16 * s >= D) return s;
    return 0;
}

Plan plan_of(int dtype, int rows, int D, bool tiles) {
    Plan g{};
    if (tiles) {
        g.tiles = true;
        g.rows_per_tile = rows > 128 ? 256 : 128;
        g.tile = 128;
        g.ctas_per_sm = 1;
        return g;
    }
    g.rows_per_tile = ROWS;
    if (dtype == CONVNN_F32) {
        g.tile = 32;
        g.stages = D <= 64 ? 3 : 2;
        g.smem = 4 * ((size_t)ROWS * (D + 4) + SW * ROWS * SP + ROWS * PP + 3 * ROWS + 4 + (size_t)g.stages * 2 * TILE * (D + 4));
        g.ctas_per_sm = g.smem <= 112 * 1024 ? 2 : 1;
    } else {
        const int DP = 16 * steps_of(D), pitch = ((DP / 8) | 1) * 16;
        g.tile = 64;
        g.stages = DP <= 64 ? 4 : DP <= 96 ? 3 : 2;
        g.smem = (size_t)16 * pitch + 4 * (ROWS * (DP + 8) + 5 * ROWS + 4) + (size_t)kWarps * g.stages * 32 * pitch;
        g.ctas_per_sm = g.smem <= 112 * 1024 ? 2 : 1;
    }
    return g;
}

// More than one tile of 16 rows: keys and values would be read more than once.
bool tiles_wanted(int dtype, int rows, int D) { return dtype == CONVNN_BF16 && rows > ROWS && D <= 128; }

long long slot_floats(const Plan& g, int D) { return (long long)g.rows_per_tile * (D + 2) + 4; }

// What is asked of the driver once on each device: that a kernel's clusters may have sixteen CTAs, and how many clusters of 1, 2, 4, 8, 16 run
// at once, which goes by its shared memory and so by the channels, a multiple of 4 (one more than that; 0: not asked).
struct Clusters {
    std::atomic<int> allowed[16];
    std::atomic<short> fit[16][64][5];
};
// As many CTAs a unit, up to p.split, as leave all clusters room at once; p.split = 0 where the even division is the better one: its second
// kernel takes as long as a CTA's `worth` tiles.
int launch_clusters(void (*kern)(Params), Params& p, unsigned units, int unit_tiles, int worth, int threads, size_t smem, cudaStream_t st,
                    Clusters& known) {
    int device = 0;
    cudaGetDevice(&device);
    const bool remembered = device >= 0 && device < 16;
    if (!remembered || !known.allowed[device].load(std::memory_order_relaxed)) {
        const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return set_error(CONVNN_E_CUDA, "tree_attention: %s", cudaGetErrorString(e));
        if (remembered) known.allowed[device].store(1, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2]{};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1] = chained_attribute(st);
    cfg.blockDim = threads; cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr;
    for (int size = 4;; --size) {
        if ((1 << size) > p.split) continue;
        attr[0].val.clusterDim.x = (unsigned)(p.split = 1 << size);
        cfg.gridDim = units * (unsigned)p.split;
        if (size == 0) break;
        std::atomic<short>* fit = remembered ? &known.fit[device][p.D / 4 - 1][size] : nullptr;
        int clusters = fit ? fit->load(std::memory_order_relaxed) - 1 : -1;
        if (clusters < 0) {
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&clusters, reinterpret_cast<const void*>(kern), &cfg) != cudaSuccess) {   // (none fits)
                cudaGetLastError();
                clusters = 0;
            }
            if (fit) fit->store((short)(clusters + 1), std::memory_order_relaxed);
        }
        if (units <= (unsigned)clusters) break;
    }
    if ((unit_tiles + p.split - 1) / p.split > (long long)units * unit_tiles / p.ctas + worth) {
        p.split = 0;
        return CONVNN_OK;
    }
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kern, p);               // an error stays the thread's last error (CONVNN_CHECK_LAUNCH)
    return CONVNN_OK;
}
// p.split: the most CTAs a unit may have, 0: none; on return what it got, 0: the even division.
template <int DS, int STAGES>
int launch_rows(Params& p, unsigned units, int unit_tiles, size_t smem, cudaStream_t st) {
    if (p.split) {
        const size_t joined = smem + join_bytes(p.D / 4);
        CONVNN_ENSURE_SMEM((rows_kernel<DS, STAGES, true>), joined);
        static Clusters known{};
        const int rc = launch_clusters(rows_kernel<DS, STAGES, true>, p, units, unit_tiles, 6, kThreads, joined, st, known);
        if (rc) return rc;
    }
    if (!p.split) {
        CONVNN_ENSURE_SMEM((rows_kernel<DS, STAGES, false>), smem);
        launch_chained(rows_kernel<DS, STAGES, false>, p.ctas, kThreads, smem, st, p);
    }
    CONVNN_CHECK_LAUNCH("tree_attention");
    return CONVNN_OK;
}
template <int STAGES>
int launch_scalar(Params& p, unsigned units, int unit_tiles, size_t smem, cudaStream_t st) {
    if (p.split) {
        const size_t joined = smem + join_bytes(p.D / 4);
        CONVNN_ENSURE_SMEM((scalar_kernel<STAGES, true>), joined);
        static Clusters known{};
        const int rc = launch_clusters(scalar_kernel<STAGES, true>, p, units, unit_tiles, 2, kScalarThreads, joined, st, known);
        if (rc) return rc;
    }
    if (!p.split) {
        CONVNN_ENSURE_SMEM((scalar_kernel<STAGES, false>), smem);
        launch_chained(scalar_kernel<STAGES, false>, p.ctas, kScalarThreads, smem, st, p);
    }
    CONVNN_CHECK_LAUNCH("tree_attention");
    return CONVNN_OK;
}

}  // namespace

size_t tree_attention_workspace(int dtype, int T, int G, int D) {
    const Plan scalar = plan_of(dtype, T * G, D, false), tiles = plan_of(dtype, T * G, D, true);
    const size_t a = (size_t)scalar.ctas_per_sm * slot_floats(scalar, D), b = (size_t)tiles.ctas_per_sm * slot_floats(tiles, D);
    return (size_t)device_sms() * 2 * 4 * (tiles_wanted(dtype, T * G, D) && b > a ? b : a);
}

int launch_tree_attention(const convnn_tree_attention* a, const convnn_cache* cache, void* workspace, size_t workspace_bytes,
                          cudaStream_t st) {
    const int rows = a->T * (a->Hq / a->Hk);
    const Plan g = plan_of(a->dtype, rows, a->D, tiles_wanted(a->dtype, rows, a->D) && tree_tiles_supported(a, cache));
    Params p{};
    p.q = a->q; p.k = cache->k; p.v = cache->v; p.out = a->out;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a->q_stride[i]; p.os[i] = a->out_stride[i];
        p.ks[i] = cache->k_stride[i]; p.vs[i] = cache->v_stride[i];
    }
    p.table = cache->table; p.table_stride = cache->table_stride;
    p.lengths = a->lengths; p.counts = a->counts;
    p.tree = reinterpret_cast<const long long*>(a->tree);
    p.tree_stride[0] = a->tree_stride[0]; p.tree_stride[1] = a->tree_stride[1];
    p.B = a->B; p.T = a->T; p.Hk = a->Hk; p.G = a->Hq / a->Hk; p.D = a->D;
    p.pages = cache->pages; p.page_size = cache->page_size; p.width = cache->width;
    p.rows_per_tile = g.rows_per_tile; p.tile = g.tile;
    p.row_tiles = (p.T * p.G + g.rows_per_tile - 1) / g.rows_per_tile;
    p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
    p.partial = static_cast<float*>(workspace);
    p.slot = slot_floats(g, p.D);
    p.ctas = device_sms() * g.ctas_per_sm;
    int bits = 0;
    while ((1ll << bits) < p.page_size) ++bits;
    p.slot_shift = 31 + bits;
    p.slot_factor = (uint32_t)(((1ull << p.slot_shift) + p.page_size - 1) / p.page_size);
    const long long units = (long long)p.B * p.Hk * p.row_tiles, keys = (long long)p.width * p.page_size;
    if (units > 0x7fffffffll || (double)units * (double)((keys + p.tile - 1) / p.tile) > 2147483647.0)
        return set_error(CONVNN_E_UNSUPPORTED, "tree_attention: %lld units of up to %lld keys", units, keys);
    if (workspace_bytes < (size_t)p.ctas * 2 * p.slot * 4)
        return set_error(CONVNN_E_WORKSPACE, "tree_attention: workspace of %zu bytes, %zu needed", workspace_bytes,
                         (size_t)p.ctas * 2 * p.slot * 4);
    // A unit to a cluster where all tiles that there may be are few for each CTA that runs at once: as many CTAs as run at once, up to
    // sixteen a unit.  us with clusters and with the even division: 8 units of 65 tiles of 64 keys 11.3 and 17.6, 64 of them 28.5 and 37.0,
    // 128 units of 9 8.9 and 14.8; 2 units of 257 23.2 and 21.4, in float32 (514 tiles of 32) 80.9 and 30.9.
    const long long unit_tiles = (keys + p.tile - 1) / p.tile;
    if (!g.tiles && units * unit_tiles <= 16ll * p.ctas)
        for (p.split = 1; p.split < MOST_PARTS && p.split < unit_tiles && units * p.split * 2 <= p.ctas;) p.split *= 2;
    int rc;
    if (g.tiles) {
        rc = launch_tree_tiles(p, st);
    } else if (a->dtype == CONVNN_F32) {
        rc = g.stages == 3 ? launch_scalar<3>(p, (unsigned)units, (int)unit_tiles, g.smem, st) : launch_scalar<2>(p, (unsigned)units, (int)unit_tiles, g.smem, st);
    } else {
        switch (steps_of(p.D)) {
            case 4: rc = launch_rows<4, 4>(p, (unsigned)units, (int)unit_tiles, g.smem, st); break;
            case 5: rc = launch_rows<5, 3>(p, (unsigned)units, (int)unit_tiles, g.smem, st); break;
            case 6: rc = launch_rows<6, 3>(p, (unsigned)units, (int)unit_tiles, g.smem, st); break;
            case 8: rc = launch_rows<8, 2>(p, (unsigned)units, (int)unit_tiles, g.smem, st); break;
            case 12: rc = launch_rows<12, 2>(p, (unsigned)units, (int)unit_tiles, g.smem, st); break;
            default: rc = launch_rows<16, 2>(p, (unsigned)units, (int)unit_tiles, g.smem, st); break;
        }
    }
    if (rc || p.split) return rc;
    if (g.tiles) {
        launch_chained(join_tiles_kernel, dim3(p.ctas, g.rows_per_tile / 128, (p.D + 15) / 16), kThreads, 0, st, p);
        CONVNN_CHECK_LAUNCH("tree_attention");
        return CONVNN_OK;
    }
    const int joined = rows < ROWS ? rows : ROWS;
    const bool many = units * 4 <= p.ctas;                   // pieces a unit
    const dim3 grid = many ? dim3((unsigned)units, joined) : dim3(p.ctas, (joined + JOIN_ROWS - 1) / JOIN_ROWS);
    if (a->dtype == CONVNN_F32) {
        if (many) launch_chained(join_kernel<float, 4>, grid, kThreads, 0, st, p);
        else launch_chained(join_kernel<float, 1>, grid, kThreads, 0, st, p);
    } else {
        if (many) launch_chained(join_kernel<__nv_bfloat16, 4>, grid, kThreads, 0, st, p);
        else launch_chained(join_kernel<__nv_bfloat16, 1>, grid, kThreads, 0, st, p);
    }
    CONVNN_CHECK_LAUNCH("tree_attention");
    return CONVNN_OK;
}

}  // namespace convnn
