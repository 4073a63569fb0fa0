// Attention of drafted tokens over a paged cache on the tensor cores: a tile of 128 query rows of one sequence and key head against
// tiles of 128 keys (tree_attention.cu has the formulas, the division of the work and the join).
// A unit's work is two streams, each with scores, weights and an accumulator of its own in tensor memory, so that one's exponentials run
// while the other's products do: with up to 128 rows the even and the odd tiles of keys, whose accumulators are added at the unit's end,
// with more two tiles of rows, which share every tile of keys and values.
//   warp 0     copies: the pages that hold a tile's keys and values, a box per page (or part of one) and 64 channels, 128-byte
//              swizzled; pages that are not there by a coordinate outside the map, which fills zeros
//   warp 1     products.  S = Q K^T (both from shared memory, K-major) and O += P V (P from tensor memory, V as it lies in its pages:
//              channels side by side are rows along N).  Neither the scores nor their weights leave the SM's tensor memory.
//   warps 4-11 softmax, a group of four for each stream: a thread owns a row, with a maximum and a sum.  The maximum is replaced, and
//              the accumulator multiplied, only when a tile exceeds it by 2^8 (float32 holds what that leaves).
// A weight is rounded to one bfloat16 for its product (a second part would cost half the tensor cores' time); its sum is of the
// unrounded ones.  Off by 2^-8 of itself at most, a weight adds to a result of many independent values about what the result's own rounding
// is off: 0.0023 of it (root of the mean square) where 16 rows a tile, whose weights are two bfloat16, are off by 0.0017.
// 16 sequences of 32 to 64 drafted tokens over 4096 to 16384 entries, 32 query and 8 key heads of 128: 208 us for the first hundred calls (238
// after seconds of them, when the clock has fallen to 1717 MHz at 990 W; the other figures here are of hundreds too), of which the two products
// are 77 at the tensor cores' nominal rate.  What bounds it is the way round: scores, 2000 cycles of softmax, weights, 1200 cycles of products; a
// stream's next scores wait for its last weights (they lie where those were), and a period of both streams is 3990 cycles where the tensor
// cores need 2050 and the exponentials as many.  How it came here: one tile of rows, two streams of keys 325 us (the second tile of rows reads all
// keys again); two tiles of rows sharing them, registers moved 243; the next unit's queries before the last one's sums, sums side by side 222; one
// wait a step 218; pieces joined by a thread a row 208.  Tried and slower: a quarter of the exponentials as polynomials with the product
// in halves 229 (the exponential unit is not what is waited for: without any exponential 240 of 243); one room of scores for both streams,
// weights apart, so that the next scores are there when the last weights are done: 232, and with the weights kept in registers until
// their room is free 244 to 286 (216 registers do not hold them); steps of 64 keys with two rooms of scores a stream 240 (half the registers, nothing
// spilled, but twice the hand-overs, and a product of 64 columns reads its 128 rows from shared memory as one of 128 does).
#include "f32x2.cuh"
#include "paged_attention.cuh"
#include "sm100.cuh"

namespace convnn {

__device__ int g_tree_attention_status = 0;   // error latch of this translation unit

namespace {

using namespace sm100;
using namespace paged;

constexpr int kRows = 128, kKeys = kTileKeys, kTileThreads = 384;
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
// A wait of a converged warp for as many barriers as its lanes name (0: none), which costs what one does.
__device__ __forceinline__ bool mbar_wait_lanes(uint32_t bar, uint32_t parity, volatile int* abort) {
    bool done = bar == 0 || mbar_try_wait_a(bar, parity);
    if (__all_sync(0xffffffffu, done)) return true;
    const unsigned long long t0 = global_timer_ns();
    for (uint32_t i = 0; i < kStartPollLimit; ++i) {
        if (!done) done = mbar_try_wait_a(bar, parity);
        if (__all_sync(0xffffffffu, done)) return true;
        if ((i & 255u) == 255u && __any_sync(0xffffffffu, *abort || global_timer_ns() - t0 > kWaitBudgetNs)) return false;
    }
    return false;
}
// The softmax warps: with TWO each group for itself.
template <bool TWO> __device__ __forceinline__ void groups_sync(int group) {
    if (TWO) asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");
    else asm volatile("bar.sync 1, 256;" ::: "memory");
}

// Registers move from the warps that copy and multiply to those that hold a row of scores: 56 + 2 * 216 of the 3 * 168 a thread that the
// block starts with.
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// DC columns of 64 channels, KS tiles of keys and VS of values in flight; TWO: tiles of rows, else tiles of keys as the two streams.
template <int DC, int KS, int VS, bool TWO>
__global__ void __launch_bounds__(kTileThreads, 1)
tiles_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Params p, const TileMaps tm) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    constexpr uint32_t kTileBytes = DC * kChunk;
    uint8_t* sQ = smem;
    uint8_t* sK = sQ + (TWO ? 2 : 1) * kTileBytes;
    uint8_t* sV = sK + KS * kTileBytes;
    float2* sScale = reinterpret_cast<float2*>(sV + VS * kTileBytes);        // [128]
    uint64_t* bars = reinterpret_cast<uint64_t*>(sScale + kRows);
    uint64_t *k_full = bars, *k_empty = k_full + KS, *v_full = k_empty + KS, *v_empty = v_full + VS;
    uint64_t *s_full = v_empty + VS, *p_ready = s_full + 2, *o_done = p_ready + 2, *q_ready = o_done + 2, *drained = q_ready + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* sStop = reinterpret_cast<volatile int*>(tmem_slot + 2);    // [2]: a group's
    int* sBad = reinterpret_cast<int*>(tmem_slot + 4);                       // [8]: a unit's, in turn

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < KS; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, 1);
        }
        for (int i = 0; i < VS; ++i) {
            mbar_init(v_full + i, 1);
            mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_ready + i, 4);
            mbar_init(o_done + i, 1);
        }
        mbar_init(q_ready, TWO ? 4 : 8);
        mbar_init(q_ready + 1, 4);
        mbar_init(drained, 1);
        *abort_flag = 0;
        for (int i = 0; i < 8; ++i) sBad[i] = 0;
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
        for (uint32_t i = threadIdx.x; i < (TWO ? 2 : 1) * kTileBytes / 16; i += kTileThreads) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    chain_begin();

    const int steps = (p.D + 15) / 16;                       // of 16 channels
    Cursor at;
    at.start(p, blockIdx.x);
    uint32_t it = 0;                                         // tiles of keys so far

    if (warp < 4) {
      registers_down<56>();
      if (warp == 0) {
        // ---- copies
        const uint32_t k0 = smem_u32(sK), v0 = smem_u32(sV);
        uint32_t keys = 0;                                   // tiles of keys asked for (of values: it)
        bool ok = true;
        while (at.left > 0 && ok) {
            const int n = at.run();
            for (int j = 0; j < n; ++j, ++it) {
                const uint32_t ks = it % KS, vs = it % VS;
                const int entry = (at.tile + j) * kKeys + lane * tm.box, slot = p.slot_at(entry), row = entry - slot * p.page_size;
                int page = -1;
                if (lane < tm.boxes && entry < at.s.total) page = p.table[at.b * p.table_stride + slot];
                if ((unsigned)page >= (unsigned)p.pages) page = p.pages;      // outside the map: zeros
                const uint32_t off = lane * (tm.box * 128);
                if (!mbar_wait_warp(smem_u32(k_empty + ks), ((it / KS) & 1u) ^ 1u, abort_flag)) { fail(abort_flag, 141); ok = false; break; }
                if (lane == 0) mbar_expect_tx(k_full + ks, kTileBytes);
                __syncwarp();
                if (lane < tm.boxes)
                    for (int c = 0; c < DC; ++c)
                        tma_load_4d_a(k0 + ks * kTileBytes + off + c * kChunk, &tmK, smem_u32(k_full + ks), c * 64, row, at.h, page);
                keys = it + 1;
                if (!mbar_wait_warp(smem_u32(v_empty + vs), ((it / VS) & 1u) ^ 1u, abort_flag)) { fail(abort_flag, 142); ok = false; break; }
                if (lane == 0) mbar_expect_tx(v_full + vs, kTileBytes);
                __syncwarp();
                if (lane < tm.boxes)
                    for (int c = 0; c < DC; ++c)
                        tma_load_4d_a(v0 + vs * kTileBytes + off + c * kChunk, &tmV, smem_u32(v_full + vs), c * 64, row, at.h, page);
            }
            if (ok) at.skip(p, n);
        }
        if (!ok && lane == 0) {                              // what was asked for lands before the block leaves
            int never = 0;
            for (uint32_t f = keys > KS ? keys - KS : 0; f < keys; ++f) mbar_wait(k_full + f % KS, (f / KS) & 1u, &never);
            for (uint32_t f = it > VS ? it - VS : 0; f < it; ++f) mbar_wait(v_full + f % VS, (f / VS) & 1u, &never);
        }
      } else if (warp == 1) {
        // ---- products
        const uint32_t idesc_s = make_idesc_bf16_f32(kRows, kKeys), idesc_o = make_idesc_bf16_f32(kRows, 16 * steps) | kIdescBAlongN;
        const uint64_t kd = kmajor_desc_hi(128), nd = mnmajor_desc_hi(kChunk);
        const uint32_t q0 = smem_u32(sQ), k0 = smem_u32(sK), v0 = smem_u32(sV);
        uint32_t units = 0, made[2] = {0, 0};
        bool ok = true;
        // Step i of a unit: stream i & 1 with tile i (TWO: i / 2) of its keys.  The warp waits once a step, for the weights and values of
        // one product and the keys of the next scores.
        auto tile_of = [&](int i) { return it + (uint32_t)(TWO ? i >> 1 : i); };
        auto scores = [&](int i) {                           // (one lane)
            const uint32_t stage = tile_of(i) % KS, s = i & 1;
            const uint64_t ad = kd | (uint64_t)(((q0 + (TWO ? s * kTileBytes : 0)) & 0x3FFFFu) >> 4);
            const uint64_t bd = kd | (uint64_t)(((k0 + stage * kTileBytes) & 0x3FFFFu) >> 4);
            const uint32_t d = tmem + s * kKeys;
            if (steps == 4 * DC) {
#pragma unroll
                for (int k = 0; k < 4 * DC; ++k) {
                    const uint32_t off = (k >> 2) * (kChunk >> 4) + (k & 3) * 2;
                    mma_bf16_ss(d, ad + off, bd + off, idesc_s, k != 0);
                }
            } else {
                for (int k = 0; k < steps; ++k) {
                    const uint32_t off = (k >> 2) * (kChunk >> 4) + (k & 3) * 2;
                    mma_bf16_ss(d, ad + off, bd + off, idesc_s, k != 0);
                }
            }
            if (!TWO || s) mma_commit(k_empty + stage);
            mma_commit(s_full + s);
        };
        while (at.left > 0 && ok) {
            const int n = at.run(), last = TWO ? 2 * n : n;
            for (int i = 0; i < 2 && i < last && ok; ++i) {
                uint32_t bar = 0, parity = 0;
                if (lane == 0) { bar = smem_u32(k_full + tile_of(i) % KS); parity = (tile_of(i) / KS) & 1u; }
                if (lane == 1 && (TWO || i == 0)) { bar = smem_u32(q_ready + i); parity = units & 1u; }
                if (!mbar_wait_lanes(bar, parity, abort_flag)) { fail(abort_flag, 143); ok = false; break; }
                tc_fence_after_sync();
                if (elect_one()) scores(i);
            }
            for (int i = 0; i < last && ok; ++i) {
                const uint32_t stage = tile_of(i) % VS, s = i & 1;
                uint32_t bar = 0, parity = 0;
                if (lane == 0) { bar = smem_u32(p_ready + s); parity = made[s] & 1u; }
                if (lane == 1) { bar = smem_u32(v_full + stage); parity = (tile_of(i) / VS) & 1u; }
                if (lane == 2 && i + 2 < last) { bar = smem_u32(k_full + tile_of(i + 2) % KS); parity = (tile_of(i + 2) / KS) & 1u; }
                if (!mbar_wait_lanes(bar, parity, abort_flag)) { fail(abort_flag, 145); ok = false; break; }
                ++made[s];
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint64_t bd = nd | (uint64_t)(((v0 + stage * kTileBytes) & 0x3FFFFu) >> 4);
                    const uint32_t d = tmem + 2 * kKeys + s * 128, a = tmem + s * kKeys;
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k) mma_bf16_ts(d, a + k * 8, bd + k * (2048 >> 4), idesc_o, i >= 2 || k != 0);
                    if (!TWO || s) mma_commit(v_empty + stage);
                    mma_commit(o_done + s);
                    if (i + 2 < last) scores(i + 2);
                }
            }
            it += n;
            ++units;
            if (ok) at.skip(p, n);
        }
        // none is in flight when the tensor memory is given back, however the loop ended
        int never = 0;
        if (elect_one()) mma_commit(drained);
        mbar_wait_warp(smem_u32(drained), 0, &never);
      }
    } else {
        // ---- softmax
        registers_up<216>();
        const int group = (warp - 4) >> 2, quad = warp & 3, r = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t tS = tmem + group * kKeys + lanes, tO = tmem + 2 * kKeys + group * 128 + lanes, tO0 = tmem + 2 * kKeys + lanes;
        const int chunks = p.D / 8;
        // Rows of q of the unit at c, this warp's share of them: TWO, 32 of its group's tile; else 16 of the one tile.
        auto load_rows = [&](const Cursor& c) {
            constexpr int CPR = DC * 8, ITEMS = (TWO ? 32 : 16) * CPR / 32, BATCH = ITEMS < 8 ? ITEMS : 8;
            const int row_first = TWO ? group * kRows + quad * 32 : (warp - 4) * 16, tile_row = c.rt * (TWO ? 2 : 1) * kRows;
#pragma unroll 1
            for (int i0 = 0; i0 < ITEMS; i0 += BATCH) {
                uint4 v[BATCH];
#pragma unroll
                for (int e = 0; e < BATCH; ++e) {
                    const int item = (i0 + e) * 32 + lane, col = item % CPR, row = tile_row + row_first + item / CPR, t = row / p.G;
                    v[e] = make_uint4(0, 0, 0, 0);
                    if (t < c.s.count && col < chunks && tm.sign != 0.f)
                        v[e] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + c.b * p.qs[0] + t * p.qs[1] +
                                                               (c.h * p.G + row - t * p.G) * p.qs[2] + col * 8);
                }
#pragma unroll
                for (int e = 0; e < BATCH; ++e) {
                    const int item = (i0 + e) * 32 + lane, col = item % CPR, rr = row_first + item / CPR;
                    if (tm.sign < 0.f) { v[e].x ^= 0x80008000u; v[e].y ^= 0x80008000u; v[e].z ^= 0x80008000u; v[e].w ^= 0x80008000u; }
                    if (col < chunks)
                        *reinterpret_cast<uint4*>(sQ + (rr >> 7) * kTileBytes + (col >> 3) * kChunk + (rr & 127) * 128 +
                                                  (((col & 7) ^ (rr & 7)) << 4)) = v[e];
                }
            }
            fence_proxy_async();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready + (TWO ? group : 0));
        };
        uint32_t seen = 0, units = 0;                        // tiles of this group, units so far
        bool first_unit = true;
        if (TWO && at.left > 0) load_rows(at);
        while (at.left > 0) {
            bool ok = true;
            const int n = at.run(), tile0 = at.tile;
            const Sequence s = at.s;
            const int b = at.b, h = at.h, unit0 = at.rt * (TWO ? 2 : 1) * kRows, row0 = unit0 + (TWO ? group * kRows : 0);
            const int last = TWO ? 2 * n : n;
            // (with TWO a group may still write what the unit before the last one was when the other one begins this unit)
            int* unit_bad = sBad + (units & 7);
            if (threadIdx.x == 128) sBad[(units + 4) & 7] = 0;
            if (!TWO) load_rows(at);

            const unsigned long long drafts = s.total - s.length >= 64 ? ~0ull : (1ull << (s.total - s.length)) - 1;
            const unsigned long long mask = seen_by(p, s, b, row0 + r) & drafts;
            const bool busy = row0 + quad * 32 < s.count * p.G;               // (any row of this warp)
            float m = -CUDART_INF_F, l = 0.f;
            for (int i = group; i < last; i += 2, ++seen) {
                const int j = TWO ? i >> 1 : i;
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
                        if (i >= 2) {
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
                    const uint32_t stage = tile_at % VS;
                    if (!__all_sync(0xffffffffu, mbar_wait(v_full + stage, (tile_at / VS) & 1u, abort_flag))) { if (lane == 0) fail(abort_flag, 149); ok = false; break; }
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
                            if (hit) {                       // (first the word of it: with TWO the other group may come second)
                                atomicOr(unit_bad, 1);
                                __threadfence_block();
                                *at16 = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                    }
                    fence_proxy_async();
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready + group);
            }
            // ---- the unit's end.  A warp that gave up comes here too, and the warps of a barrier, which has no limit, leave together
            if (TWO && ok && at.left > n) {                  // the stream's scores are done, and the next unit's may begin
                Cursor ahead = at;
                ahead.skip(p, n);
                load_rows(ahead);
            }
            if (ok && last > group && !__all_sync(0xffffffffu, mbar_wait(o_done + group, (seen - 1) & 1u, abort_flag)) && lane == 0)
                fail(abort_flag, 148);
            if (!TWO && group == 1) sScale[r] = make_float2(m, l);
            tc_fence_before_sync();
            groups_sync<TWO>(group);
            tc_fence_after_sync();
            if (threadIdx.x == 128 || (TWO && threadIdx.x == 256)) sStop[group] = *abort_flag;
            const bool any_bad = *reinterpret_cast<volatile int*>(unit_bad) != 0;
            const bool whole = tile0 == 0 && n == s.tiles;
            float* slot = slot_of(p, blockIdx.x, first_unit);
            float2 f = make_float2(1.f, 0.f);                // what this stream's and, of the same rows, the other's sums are multiplied by
            if (TWO || group == 0) {
                const float2 other = TWO ? make_float2(-CUDART_INF_F, 0.f) : sScale[r];
                const float top = fmaxf(m, other.x);
                f.x = m == -CUDART_INF_F ? 0.f : ex2((m - top) * tm.factor);
                f.y = other.x == -CUDART_INF_F ? 0.f : ex2((other.x - top) * tm.factor);
                const float sum = l * f.x + other.y * f.y;
                if (whole) {
                    const float inv = inverse_of(p, s, b, row0 + r, sum);
                    f.x *= inv;
                    f.y *= inv;
                } else {
                    float* tail = slot + (long long)p.rows_per_tile * p.D;
                    tail[row0 - unit0 + r] = top * tm.factor;
                    tail[p.rows_per_tile + row0 - unit0 + r] = sum;
                    if (r == 0) tail[2 * p.rows_per_tile + (TWO ? group : 0)] = any_bad ? 1.f : 0.f;
                }
                if (!TWO) sScale[r] = f;
            }
            groups_sync<TWO>(group);
            if (sStop[TWO ? group : 0]) break;
            if (busy) {
                if (!TWO) f = sScale[r];
                const int t = (row0 + r) / p.G, g = row0 + r - t * p.G;
                const bool there = t < s.count;
                const int half = (steps + 1) / 2;            // (TWO: each group writes its own rows, else half of the channels of all)
#pragma unroll 1
                for (int c = !TWO && group ? half : 0; c < (TWO || group ? steps : half); ++c) {
                    uint32_t o[16], o1[16];
                    __syncwarp();
                    tmem_ld_x16((TWO ? tO : tO0) + 16 * c, o);
                    if (!TWO && n > 1) tmem_ld_x16(tO0 + 128 + 16 * c, o1);
                    tmem_ld_wait();
                    tie16(o);
                    if (!TWO && n > 1) tie16(o1);
                    float y[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        y[e] = __uint_as_float(o[e]) * f.x;
                        if (!TWO && n > 1) y[e] = fmaf(__uint_as_float(o1[e]), f.y, y[e]);
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
                        // (four channels of a warp's rows side by side)
                        float4* dst = reinterpret_cast<float4*>(slot) + (long long)(4 * c) * p.rows_per_tile + row0 - unit0 + r;
#pragma unroll
                        for (int u = 0; u < 4; ++u)
                            if (16 * c + 4 * u < p.D)
                                dst[u * p.rows_per_tile] = make_float4(y[4 * u], y[4 * u + 1], y[4 * u + 2], y[4 * u + 3]);
                    }
                }
            }
            first_unit = false;
            ++units;
            it += n;
            at.skip(p, n);
            if (!TWO) {                                      // both accumulators are read by both groups
                tc_fence_before_sync();
                groups_sync<TWO>(group);
                tc_fence_after_sync();
            }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

template <int DC, int KS, int VS, bool TWO>
int launch_tiles(const CUtensorMap& k, const CUtensorMap& v, const Params& p, const TileMaps& tm, cudaStream_t st) {
    const size_t smem = 1024 + (size_t)((TWO ? 2 : 1) + KS + VS) * DC * kChunk + kRows * sizeof(float2) + 8 * (2 * KS + 2 * VS + 9) + 48;
    CONVNN_ENSURE_SMEM((tiles_kernel<DC, KS, VS, TWO>), smem);
    launch_chained(tiles_kernel<DC, KS, VS, TWO>, p.ctas, kTileThreads, smem, st, k, v, p, tm);
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
    if (p.rows_per_tile > kRows)
        return p.D <= 64 ? launch_tiles<1, 6, 5, true>(k, v, p, tm, st) : launch_tiles<2, 3, 2, true>(k, v, p, tm, st);
    return p.D <= 64 ? launch_tiles<1, 6, 6, false>(k, v, p, tm, st) : launch_tiles<2, 3, 3, false>(k, v, p, tm, st);
}

int read_tree_attention_status(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_tree_attention_status, sizeof(int));
    if (e != cudaSuccess) return set_error(CONVNN_E_CUDA, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(e));
    *out = v;
    return CONVNN_OK;
}

}  // namespace convnn
