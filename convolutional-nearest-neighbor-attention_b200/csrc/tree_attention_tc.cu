// Attention of drafted tokens over a paged cache on the tensor cores: a tile of 128 query rows of one sequence and key head against
// tiles of 128 keys (tree_attention.cu has the formulas, the division of the work and the join).
//   warp 0     copies: the pages that hold a tile's keys and values, a box per page (or part of one) and 64 channels, 128-byte
//              swizzled; pages that are not there by a coordinate outside the map, which fills zeros
//   warp 1     products.  S = Q K^T (both from shared memory, K-major) and O += P V (P from tensor memory, V as it lies in its pages:
//              channels side by side are rows along N).  Neither the scores nor their weights leave the SM's tensor memory.
//   warps 2-9  softmax, in two groups of four: a thread owns a row, the groups take the unit's tiles in turn, each with a maximum, a
//              sum and an accumulator of its own, so that one group's exponentials run while the other's products do.  A maximum is
//              replaced, and the accumulator multiplied, only when a tile exceeds it by 2^8 (float32 holds what that leaves).
// At the unit's end the two accumulators are added, each group writing half of the channels.
// A weight is rounded to one bfloat16 for its product (a second part would cost half the tensor cores' time); its sum is of the
// unrounded ones.
#include "f32x2.cuh"
#include "paged_attention.cuh"
#include "sm100.cuh"

namespace convnn {

__device__ int g_tree_attention_status = 0;   // error latch of this translation unit

namespace {

using namespace sm100;
using namespace paged;

constexpr int kRows = 128, kKeys = kTileKeys, kTileThreads = 320;
constexpr uint32_t kChunk = 128 * 128;        // 128 rows of 64 channels

struct TileMaps {
    int box, boxes;                           // entries a copy, copies a tile
    float factor, sign;                       // of the scores: log2(e) * |scale|, and what q is multiplied by (1, -1, 0)
};

__device__ __forceinline__ void fail(volatile int* abort_flag, int code) {
    *abort_flag = 1;
    atomicCAS(&g_tree_attention_status, 0, code);
}
__device__ __forceinline__ void tie(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tie16(uint32_t (&r)[16]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
// The two softmax groups.
__device__ __forceinline__ void groups_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// DC columns of 64 channels, STAGES tiles of keys and of values in flight.
template <int DC, int STAGES>
__global__ void __launch_bounds__(kTileThreads, 1)
tiles_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Params p, const TileMaps tm) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr uint32_t kTileBytes = DC * kChunk;
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + kTileBytes;
    uint8_t* sV = sK + STAGES * kTileBytes;
    float2* sScale = reinterpret_cast<float2*>(sV + STAGES * kTileBytes);    // [128]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + kRows);
    uint64_t *k_full = bars, *k_empty = k_full + STAGES, *v_full = k_empty + STAGES, *v_empty = v_full + STAGES;
    uint64_t *s_full = v_empty + STAGES, *p_ready = s_full + 2, *o_done = p_ready + 2, *q_ready = o_done + 2, *drained = q_ready + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* sBad = reinterpret_cast<int*>(tmem_slot + 2);
    volatile int* sStop = reinterpret_cast<volatile int*>(tmem_slot + 3);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, 1);
            mbar_init(v_full + i, 1);
            mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_ready + i, 4);
            mbar_init(o_done + i, 1);
        }
        mbar_init(q_ready, 8);
        mbar_init(drained, 1);
        *abort_flag = 0;
        *sBad = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmK);
        prefetch_tensormap(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    // (channels behind D, which q's rows leave open, stay zeros)
    if (p.D % 16)
      for (uint32_t i = threadIdx.x; i < kTileBytes / 16; i += kTileThreads) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    chain_begin();

    const int steps = (p.D + 15) / 16;                       // of 16 channels
    Cursor at;
    at.start(p, blockIdx.x);
    uint32_t it = 0;                                         // tiles so far

    if (warp == 0) {
        // ---- copies
        const uint32_t k0 = smem_u32(sK), v0 = smem_u32(sV);
        bool ok = true;
        while (at.left > 0 && ok) {
            const int n = at.run();
            for (int j = 0; j < n; ++j, ++it) {
                const uint32_t stage = it % STAGES, ph = (it / STAGES) & 1u;
                const int entry = (at.tile + j) * kKeys + lane * tm.box, slot = p.slot_at(entry), row = entry - slot * p.page_size;
                int page = -1;
                if (lane < tm.boxes && entry < at.s.total) page = p.table[at.b * p.table_stride + slot];
                if ((unsigned)page >= (unsigned)p.pages) page = p.pages;      // outside the map: zeros
                const uint32_t dst = stage * kTileBytes + lane * (tm.box * 128);
                if (!mbar_wait_warp(smem_u32(k_empty + stage), ph ^ 1u, abort_flag)) { fail(abort_flag, 141); ok = false; break; }
                if (lane == 0) mbar_expect_tx(k_full + stage, kTileBytes);
                __syncwarp();
                if (lane < tm.boxes)
                    for (int c = 0; c < DC; ++c)
                        tma_load_4d_a(k0 + dst + c * kChunk, &tmK, smem_u32(k_full + stage), c * 64, row, at.h, page);
                if (!mbar_wait_warp(smem_u32(v_empty + stage), ph ^ 1u, abort_flag)) { fail(abort_flag, 142); ok = false; break; }
                if (lane == 0) mbar_expect_tx(v_full + stage, kTileBytes);
                __syncwarp();
                if (lane < tm.boxes)
                    for (int c = 0; c < DC; ++c)
                        tma_load_4d_a(v0 + dst + c * kChunk, &tmV, smem_u32(v_full + stage), c * 64, row, at.h, page);
            }
            if (ok) at.skip(p, n);
        }
        if (!ok && lane == 0) {
            // what was asked for lands before the block leaves (it: the tile whose keys, and perhaps values, were not)
            int never = 0;
            for (uint32_t f = it >= STAGES ? it - STAGES : 0; f < it; ++f) {
                mbar_wait(k_full + f % STAGES, (f / STAGES) & 1u, &never);
                mbar_wait(v_full + f % STAGES, (f / STAGES) & 1u, &never);
            }
            if (mbar_try_wait(k_empty + it % STAGES, ((it / STAGES) & 1u) ^ 1u)) mbar_wait(k_full + it % STAGES, (it / STAGES) & 1u, &never);
        }
    } else if (warp == 1) {
        // ---- products
        const uint32_t idesc_s = make_idesc_bf16_f32(kRows, kKeys), idesc_o = make_idesc_bf16_f32(kRows, 16 * steps) | kIdescBAlongN;
        const uint64_t kd = kmajor_desc_hi(128), nd = mnmajor_desc_hi(kChunk);
        const uint32_t q0 = smem_u32(sQ), k0 = smem_u32(sK), v0 = smem_u32(sV);
        uint32_t units = 0, made[2] = {0, 0}, scored = 0;
        bool ok = true;
        auto scores = [&](int j) -> bool {                   // tile j of the unit, the it + (j - done)-th of the CTA
            const uint32_t stage = scored % STAGES, ph = (scored / STAGES) & 1u;
            if (!mbar_wait_warp(smem_u32(k_full + stage), ph, abort_flag)) { fail(abort_flag, 143); return false; }
            tc_fence_after_sync();
            if (elect_one()) {
                const uint64_t ad = kd | (uint64_t)((q0 & 0x3FFFFu) >> 4), bd = kd | (uint64_t)(((k0 + stage * kTileBytes) & 0x3FFFFu) >> 4);
                for (int k = 0; k < steps; ++k) {
                    const uint32_t off = (k >> 2) * (kChunk >> 4) + (k & 3) * 2;
                    mma_bf16_ss(tmem + (j & 1) * kKeys, ad + off, bd + off, idesc_s, k != 0);
                }
                mma_commit(k_empty + stage);
                mma_commit(s_full + (j & 1));
            }
            ++scored;
            return true;
        };
        while (at.left > 0 && ok) {
            const int n = at.run();
            if (!mbar_wait_warp(smem_u32(q_ready), units & 1u, abort_flag)) { fail(abort_flag, 144); ok = false; break; }
            ++units;
            tc_fence_after_sync();
            ok = scores(0) && (n < 2 || scores(1));
            for (int j = 0; j < n && ok; ++j, ++it) {
                const uint32_t stage = it % STAGES, ph = (it / STAGES) & 1u, s = j & 1;
                if (!mbar_wait_warp(smem_u32(p_ready + s), made[s] & 1u, abort_flag)) { fail(abort_flag, 145); ok = false; break; }
                ++made[s];
                if (!mbar_wait_warp(smem_u32(v_full + stage), ph, abort_flag)) { fail(abort_flag, 146); ok = false; break; }
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint64_t bd = nd | (uint64_t)(((v0 + stage * kTileBytes) & 0x3FFFFu) >> 4);
                    for (int k = 0; k < kKeys / 16; ++k)
                        mma_bf16_ts(tmem + 2 * kKeys + s * 128, tmem + s * kKeys + k * 8, bd + k * (2048 >> 4), idesc_o, j >= 2 || k != 0);
                    mma_commit(v_empty + stage);
                    mma_commit(o_done + s);
                }
                if (j + 2 < n) ok = scores(j + 2);
            }
            if (ok) at.skip(p, n);
        }
        // none is in flight when the tensor memory is given back, however the loop ended
        int never = 0;
        if (elect_one()) mma_commit(drained);
        mbar_wait_warp(smem_u32(drained), 0, &never);
    } else {
        // ---- softmax
        const int group = (warp - 2) >> 2, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t tS = tmem + group * kKeys + lanes, tO = tmem + 2 * kKeys + group * 128 + lanes, tO0 = tmem + 2 * kKeys + lanes;
        const int chunks = p.D / 8;
        uint32_t seen = 0;                                   // tiles of this group so far
        bool first_unit = true;
        while (at.left > 0) {
            bool ok = true;
            const int n = at.run(), tile0 = at.tile;
            const Sequence s = at.s;
            const int b = at.b, h = at.h, row0 = at.rt * kRows;
            // the unit's rows of q, by all eight warps
            for (int i = threadIdx.x - 64; i < kRows * chunks; i += 256) {
                const int rr = i / chunks, col = i - rr * chunks, t = (row0 + rr) / p.G, g = row0 + rr - t * p.G;
                uint4 v = make_uint4(0, 0, 0, 0);
                if (t < s.count && tm.sign != 0.f)
                    v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + b * p.qs[0] + t * p.qs[1] +
                                                        (h * p.G + g) * p.qs[2] + col * 8);
                if (tm.sign < 0.f) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
                *reinterpret_cast<uint4*>(sQ + (col >> 3) * kChunk + rr * 128 + (((col & 7) ^ (rr & 7)) << 4)) = v;
            }
            fence_proxy_async();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);

            const unsigned long long drafts = s.total - s.length >= 64 ? ~0ull : (1ull << (s.total - s.length)) - 1;
            const unsigned long long mask = seen_by(p, s, b, row0 + r) & drafts;
            const bool busy = row0 + quad * 32 < s.count * p.G;               // (any row of this warp)
            float m = -CUDART_INF_F, l = 0.f;
            bool bad = false;
            for (int j = group; j < n; j += 2, ++seen) {
                const uint32_t tile_at = it + j;
                if (!__all_sync(0xffffffffu, mbar_wait(s_full + group, seen & 1u, abort_flag))) { if (lane == 0) fail(abort_flag, 147); ok = false; break; }
                tc_fence_after_sync();
                const int key0 = (tile0 + j) * kKeys;
                const bool masked = key0 + kKeys > s.length;
                if (busy) {
                    uint32_t x[4][32];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tmem_ld_x32(tS + 32 * c, x[c]);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 4; ++c) tie(x[c]);
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int first = key0 + 32 * c - s.length;       // (a drafted token's index; below 0: cached)
                            uint32_t see = first >= 64 ? 0u : (uint32_t)(mask >> (first < 0 ? 0 : first));
                            if (first <= -32) see = 0xffffffffu;
                            else if (first < 0) see = (uint32_t)(mask << -first) | ((1u << -first) - 1u);
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(see >> e & 1u)) x[c][e] = 0xff800000u;
                        }
                    }
                    float top4[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        top4[c] = __uint_as_float(x[c][0]);
#pragma unroll
                        for (int e = 1; e < 32; ++e) top4[c] = fmaxf(top4[c], __uint_as_float(x[c][e]));
                    }
                    const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
                    const bool grows = (top - m) * tm.factor > 8.f || (m == -CUDART_INF_F && top > m);
                    if (__any_sync(0xffffffffu, grows)) {
                        const float now = grows ? top : m;
                        const float f = grows ? ex2((m - now) * tm.factor) : 1.f;
                        m = now;
                        l *= f;
                        if (j >= 2) {
                            if (!__all_sync(0xffffffffu, mbar_wait(o_done + group, (seen - 1) & 1u, abort_flag))) {
                                if (lane == 0) fail(abort_flag, 148);
                                ok = false;
                                break;
                            }
                            tc_fence_after_sync();
#pragma unroll 1
                            for (int c = 0; c < 16 * steps; c += 16) {
                                uint32_t o[16];
                                tmem_ld_x16(tO + c, o);
                                tmem_ld_wait();
                                tie16(o);
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st_x16(tO + c, o);
                            }
                        }
                    }
                    const float base = m == -CUDART_INF_F ? 0.f : -m * tm.factor;
                    const f32x2 factor2 = pack2(tm.factor, tm.factor), base2 = pack2(base, base);
                    f32x2 sum2[2] = {0ull, 0ull};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float a, d;
                            unpack2(fma2(pack2(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1])), factor2, base2), a, d);
                            a = ex2(a);
                            d = ex2(d);
                            sum2[e & 1] = add2(sum2[e & 1], pack2(a, d));
                            const __nv_bfloat162 hh = __floats2bfloat162_rn(a, d);
                            w[e] = *reinterpret_cast<const uint32_t*>(&hh);
                        }
                        tmem_st_x16(tS + 16 * c, w);
                    }
                    float a, d;
                    unpack2(add2(sum2[0], sum2[1]), a, d);
                    l += a + d;
                    tmem_st_wait();
                }
                if (masked) {
                    // values of entries that are not there: zeros; of drafted tokens that are not finite: zeros for now
                    const uint32_t stage = tile_at % STAGES;
                    if (!__all_sync(0xffffffffu, mbar_wait(v_full + stage, (tile_at / STAGES) & 1u, abort_flag))) { if (lane == 0) fail(abort_flag, 149); ok = false; break; }
                    const int entry = key0 + r;
                    if (entry >= s.length) {
                        for (int col = 0; col < chunks; ++col) {
                            uint4* at16 = reinterpret_cast<uint4*>(sV + stage * kTileBytes + (col >> 3) * kChunk + r * 128 + (((col & 7) ^ (r & 7)) << 4));
                            if (entry >= s.total) {
                                *at16 = make_uint4(0, 0, 0, 0);
                                continue;
                            }
                            const uint4 v = *at16;
                            uint32_t w[4] = {v.x, v.y, v.z, v.w};
                            bool hit = false;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if ((w[e] & 0x7f80u) == 0x7f80u) { w[e] &= 0xffff0000u; hit = true; }
                                if ((w[e] & 0x7f800000u) == 0x7f800000u) { w[e] &= 0xffffu; hit = true; }
                            }
                            if (hit) {
                                *at16 = make_uint4(w[0], w[1], w[2], w[3]);
                                bad = true;
                            }
                        }
                    }
                    fence_proxy_async();
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready + group);
            }
            // ---- the unit's end: both groups' sums.  A warp that gave up comes here too, and all eight leave together (a barrier has no limit)
            if (bad) atomicOr(sBad, 1);
            if (ok && n > group && !__all_sync(0xffffffffu, mbar_wait(o_done + group, (seen - 1) & 1u, abort_flag)) && lane == 0)
                fail(abort_flag, 148);
            if (group == 1) sScale[r] = make_float2(m, l);
            tc_fence_before_sync();
            groups_sync();
            tc_fence_after_sync();
            if (threadIdx.x == 64) *sStop = *abort_flag;
            const bool any_bad = *reinterpret_cast<volatile int*>(sBad) != 0;
            const bool whole = tile0 == 0 && n == s.tiles;
            float* slot = slot_of(p, blockIdx.x, first_unit);
            if (group == 0) {
                const float2 other = sScale[r];
                const float top = fmaxf(m, other.x);
                float f0 = m == -CUDART_INF_F ? 0.f : ex2((m - top) * tm.factor);
                float f1 = other.x == -CUDART_INF_F ? 0.f : ex2((other.x - top) * tm.factor);
                const float sum = l * f0 + other.y * f1;
                if (whole) {
                    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                    f0 *= inv;
                    f1 *= inv;
                } else {
                    float* tail = slot + (long long)kRows * p.D;
                    tail[r] = top * tm.factor;
                    tail[kRows + r] = sum;
                    if (r == 0) tail[2 * kRows] = any_bad ? 1.f : 0.f;
                }
                sScale[r] = make_float2(f0, f1);
            }
            groups_sync();
            if (*sStop) break;
            if (threadIdx.x == 64) *sBad = 0;
            if (busy) {
                const float2 f = sScale[r];
                const int t = (row0 + r) / p.G, g = row0 + r - t * p.G;
                const bool there = t < s.count;
                const int half = (steps + 1) / 2;
#pragma unroll 1
                for (int c = group ? half : 0; c < (group ? steps : half); ++c) {
                    uint32_t o[16], o1[16];
                    __syncwarp();
                    tmem_ld_x16(tO0 + 16 * c, o);
                    if (n > 1) tmem_ld_x16(tO0 + 128 + 16 * c, o1);
                    tmem_ld_wait();
                    tie16(o);
                    if (n > 1) tie16(o1);
                    float y[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        y[e] = __uint_as_float(o[e]) * f.x;
                        if (n > 1) y[e] = fmaf(__uint_as_float(o1[e]), f.y, y[e]);
                    }
                    if (!there) continue;
                    if (whole) {
                        if (any_bad)
                            for (int e = 0; e < 16; ++e)
                                if (16 * c + e < p.D) y[e] += not_finite_seen<__nv_bfloat16>(p, s, b, h, mask, 16 * c + e);
                        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + b * p.os[0] + t * p.os[1] + (h * p.G + g) * p.os[2] + 16 * c;
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            if (16 * c + 8 * u >= p.D) continue;
                            __nv_bfloat162 w[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = __floats2bfloat162_rn(y[8 * u + 2 * e], y[8 * u + 2 * e + 1]);
                            *reinterpret_cast<uint4*>(out + 8 * u) = *reinterpret_cast<uint4*>(w);
                        }
                    } else {
                        float* dst = slot + (long long)r * p.D + 16 * c;
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (16 * c + 4 * u < p.D)
                                *reinterpret_cast<float4*>(dst + 4 * u) = make_float4(y[4 * u], y[4 * u + 1], y[4 * u + 2], y[4 * u + 3]);
                    }
                }
            }
            first_unit = false;
            it += n;
            at.skip(p, n);
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

template <int DC, int STAGES>
int launch_tiles(const CUtensorMap& k, const CUtensorMap& v, const Params& p, const TileMaps& tm, cudaStream_t st) {
    const size_t smem = 1024 + (size_t)(1 + 2 * STAGES) * DC * kChunk + kRows * sizeof(float2) + 8 * (4 * STAGES + 8) + 16;
    CONVNN_ENSURE_SMEM((tiles_kernel<DC, STAGES>), smem);
    launch_chained(tiles_kernel<DC, STAGES>, p.ctas, kTileThreads, smem, st, k, v, p, tm);
    CONVNN_CHECK_LAUNCH("tree_attention");
    return CONVNN_OK;
}

bool map_of(CUtensorMap* m, const void* base, const Params& p, const long long* stride, int box) {
    const uint64_t dims[4] = {(uint64_t)p.D, (uint64_t)p.page_size, (uint64_t)p.Hk, (uint64_t)p.pages};
    // (page, head, row) -> (row, head, page); the stride of a single row, head or page is not looked at, but has to be one
    uint64_t bytes[3];
    for (int i = 0; i < 3; ++i) bytes[i] = dims[i + 1] == 1 ? 16 : (uint64_t)stride[2 - i] * 2;
    const uint32_t shape[4] = {64, (uint32_t)box, 1, 1};
    return encode_tensor_map_bf16(m, base, 4, dims, bytes, shape, 128);
}

}  // namespace

bool tree_tiles_supported(const convnn_tree_attention* a, const convnn_cache* c) {
    for (int i = 0; i < 3; ++i)                              // what a tensor map takes
        if (c->k_stride[i] >= (1ll << 38) || c->v_stride[i] >= (1ll << 38)) return false;
    auto apart = [](const int64_t* s, int n, int i) { return n == 1 || s[i] > 0; };
    return a->D <= 128 && c->page_size % 16 == 0 && apart(c->k_stride, c->pages, 0) && apart(c->v_stride, c->pages, 0) &&
           apart(c->k_stride, a->Hk, 1) && apart(c->v_stride, a->Hk, 1) && c->k_stride[2] > 0 && c->v_stride[2] > 0;
}

int launch_tree_tiles(const Params& p, cudaStream_t st) {
    TileMaps tm{};
    tm.box = 16;
    while (tm.box < kKeys && p.page_size % (2 * tm.box) == 0) tm.box *= 2;
    tm.boxes = kKeys / tm.box;
    tm.factor = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
    tm.sign = p.scale_log2 > 0.f ? 1.f : p.scale_log2 < 0.f ? -1.f : 0.f;
    CUtensorMap k, v;
    if (!map_of(&k, p.k, p, p.ks, tm.box) || !map_of(&v, p.v, p, p.vs, tm.box)) return CONVNN_E_CUDA;
    return p.D <= 64 ? launch_tiles<1, 6>(k, v, p, tm, st) : launch_tiles<2, 3>(k, v, p, tm, st);
}

int read_tree_attention_status(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_tree_attention_status, sizeof(int));
    if (e != cudaSuccess) return set_error(CONVNN_E_CUDA, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(e));
    *out = v;
    return CONVNN_OK;
}

}  // namespace convnn
