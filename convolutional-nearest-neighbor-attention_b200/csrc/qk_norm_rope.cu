// Norm of every query and key head, rotation by its token's position, and on request the new keys and values into a paged cache, in
// one pass.
//   n = x * (mean(x^2) + eps)^-1/2 * weight          over the D channels of one head, in float32; x itself without a weight
//   (n_a, n_b) -> (n_a cos_i - n_b sin_i, n_b cos_i + n_a sin_i)   on the pairs (i, i + R/2), or neighbours (2i, 2i + 1), i < R/2
// rounded once, to the storage type.  Values are copied as they are.
// A group of lanes owns a head: each lane two vectors of V channels, those of a pair where pairs lie R/2 apart, so that the rotation
// needs no exchange and the norm's sum log2(lanes) of them.  A group keeps its U heads, all queries', all keys' or all values', and goes
// from token to token with their weight in registers; cosines and sines serve the U heads, whose values are requested before the first is
// used.  Groups that share a token are neighbours: a warp reads its heads as one stretch.
// Memory is what bounds it, as far as its latency is hidden: 131072 tokens of 12 + 12 heads of 64, 810 MB, 145 us (5.6 TB/s, 85 % of a plain
// copy's rate); 8 x 4096 tokens of 32 + 8 + 8 heads of 128 into a cache, 822 MB, 143 us.  A group per token that goes through its heads, with
// the weights of both kinds: 262 and 232 us (one CTA an SM, few loads in flight).  Four heads at once on two CTAs an SM are the best of what was
// tried: three heads on three CTAs 229 us, two on four 278, four on three (85 registers) 237, all heads of a token four at a time 171,
// six on three CTAs of 128 threads 156, streaming loads 149, eight times as many CTAs in turn 153.
#include <math_constants.h>

#include "common.cuh"

namespace convnn {
namespace {

constexpr int kThreads = 256;

struct HeadsParams {
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;                         // k_out, v_out: rows of the cache's pages where there is a table
    long long qs[3], ks[3], vs[3], qo[3], ko[3], vo[3];  // (batch, token, head); of the cache: (page, row, head)
    const void *wq, *wk;
    const float* rope;
    const int32_t *positions, *table, *lengths, *counts;
    long long rope_stride, pos_stride[2], table_stride;
    int rope_rows, pages, page_size, width;
    unsigned tokens, parts, abreast;                     // B * T; groups that share a token's heads; tokens at a time
    int parts_q, parts_k;
    int T, Hq, Hk, D, half, interleaved;                 // half = R / 2
    float eps, inv_d;
};

template <typename T, int V> struct Vec;
template <> struct Vec<__nv_bfloat16, 8> { using type = uint4; };
template <> struct Vec<__nv_bfloat16, 4> { using type = uint2; };
template <> struct Vec<__nv_bfloat16, 1> { using type = unsigned short; };
template <> struct Vec<float, 4> { using type = uint4; };
template <> struct Vec<float, 1> { using type = unsigned; };

template <typename T, int V>
__device__ __forceinline__ void widen(float (&x)[V], const typename Vec<T, V>::type& raw) {
    if constexpr (sizeof(T) == 4) {
        const float* f = reinterpret_cast<const float*>(&raw);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = f[e];
    } else if constexpr (V == 1) {
        x[0] = __uint_as_float((unsigned)raw << 16);
    } else {
        const unsigned* w = reinterpret_cast<const unsigned*>(&raw);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
}
template <typename T, int V>
__device__ __forceinline__ typename Vec<T, V>::type narrow(const float (&x)[V]) {
    typename Vec<T, V>::type raw;
    if constexpr (sizeof(T) == 4) {
        float* f = reinterpret_cast<float*>(&raw);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = x[e];
    } else if constexpr (V == 1) {
        raw = __bfloat16_as_ushort(__float2bfloat16_rn(x[0]));
    } else {
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) h[e] = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
    }
    return raw;
}

// LPH lanes a head, N pairs of vectors a lane (several only where V = 1), U heads at once.
template <typename T, int V, int LPH, int N, int U>
__global__ void __launch_bounds__(kThreads, 2) heads_kernel(const HeadsParams p) {
    using Raw = typename Vec<T, V>::type;
    chain_begin();
    const unsigned unit = blockIdx.x * (unsigned)(kThreads / LPH) + threadIdx.x / LPH, first = unit / p.parts;
    if (first >= p.abreast) return;                      // (a whole group, and no exchange leaves its group)
    const int part = (int)(unit - first * p.parts), lane = threadIdx.x % LPH;
    const unsigned group_mask = LPH == 32 ? 0xffffffffu : ((1u << (LPH % 32)) - 1u) << ((threadIdx.x & 31u) / LPH * LPH);

    // the group's heads
    const bool is_q = part < p.parts_q, is_v = part >= p.parts_q + p.parts_k;
    const int h0 = (is_q ? part : part - p.parts_q - (is_v ? p.parts_k : 0)) * U, count = min(U, (is_q ? p.Hq : p.Hk) - h0);
    const long long *ss = is_q ? p.qs : is_v ? p.vs : p.ks, *ds = is_q ? p.qo : is_v ? p.vo : p.ko;
    const long long s0 = ss[0], s1 = ss[1], s2 = ss[2], d0 = ds[0], d1 = ds[1], d2 = ds[2];
    const T* from = static_cast<const T*>(is_q ? p.q : is_v ? p.v : p.k) + h0 * s2;
    T* to = static_cast<T*>(is_q ? p.q_out : is_v ? p.v_out : p.k_out) + h0 * d2;
    const T* weight = static_cast<const T*>(is_q ? p.wq : is_v ? nullptr : p.wk);
    const bool normed = weight != nullptr, turn = !is_v && p.half, paged = p.table != nullptr && !is_q;

    // the lane's channels: two vectors each, and their place in the table of cosines and sines
    int c0[N], c1[N], place[N];
    Raw w0[N], w1[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int pair = lane + n * LPH;                 // of vectors
        const int turned = p.half / V;                   // pairs of vectors that are rotated
        place[n] = -1;
        if (p.interleaved) {
            c0[n] = 2 * V * pair;
            c1[n] = c0[n] + V;
            if (pair < turned) place[n] = V * pair;
        } else if (pair < turned) {
            c0[n] = V * pair;
            c1[n] = c0[n] + p.half;
            place[n] = c0[n];
        } else {
            c0[n] = 2 * p.half + 2 * V * (pair - turned);
            c1[n] = c0[n] + V;
        }
        w0[n] = w1[n] = Raw{};
        if (normed && c0[n] < p.D) w0[n] = *reinterpret_cast<const Raw*>(weight + c0[n]);
        if (normed && c1[n] < p.D) w1[n] = *reinterpret_cast<const Raw*>(weight + c1[n]);
    }

#pragma unroll 1
    for (unsigned token = first; token < p.tokens; token += p.abreast) {
        const int b = (int)(token / (unsigned)p.T), t = (int)(token - (unsigned)b * (unsigned)p.T);
        const T* src = from + b * s0 + t * s1;
        Raw x0[U][N], x1[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                x0[u][n] = x1[u][n] = Raw{};
                if (u < count && c0[n] < p.D) x0[u][n] = *reinterpret_cast<const Raw*>(src + u * s2 + c0[n]);
                if (u < count && c1[n] < p.D) x1[u][n] = *reinterpret_cast<const Raw*>(src + u * s2 + c1[n]);
            }
        // where the token is, and where it goes
        long long position = t;
        bool live = true, stored = true;
        T* dst = to + b * d0 + t * d1;
        if (p.table) {
            live = !p.counts || t < p.counts[b];
            const unsigned entry = (unsigned)max(p.lengths[b], 0) + (unsigned)t, slot = entry / (unsigned)p.page_size;   // (below 2^32)
            position = entry;
            if (paged) {
                int page = -1;
                if (live && slot < (unsigned)p.width) page = p.table[b * p.table_stride + slot];
                stored = (unsigned)page < (unsigned)p.pages;                 // (a page that is not there keeps nothing)
                dst = to + page * d0 + (long long)(entry - slot * p.page_size) * d1;
            }
        }
        float cs[N][V], sn[N][V];
        if (turn) {
            if (p.positions) position = p.positions[b * p.pos_stride[0] + t * p.pos_stride[1]];
            const bool there = (unsigned long long)position < (unsigned long long)p.rope_rows;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const float* row = p.rope + position * p.rope_stride + place[n];
                if (place[n] >= 0 && there) {
                    if constexpr (V % 4 == 0) {
#pragma unroll
                        for (int e = 0; e < V; e += 4) {
                            *reinterpret_cast<float4*>(&cs[n][e]) = *reinterpret_cast<const float4*>(row + e);
                            *reinterpret_cast<float4*>(&sn[n][e]) = *reinterpret_cast<const float4*>(row + p.half + e);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            cs[n][e] = row[e];
                            sn[n][e] = row[p.half + e];
                        }
                    }
                } else {                                 // not rotated; or no such position, which shows
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        cs[n][e] = place[n] >= 0 ? CUDART_NAN_F : 1.f;
                        sn[n][e] = place[n] >= 0 ? CUDART_NAN_F : 0.f;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= count) break;                   // (the same for the whole group)
            if (normed || turn) {
                float a[N][V], c[N][V];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    widen<T, V>(a[n], x0[u][n]);
                    widen<T, V>(c[n], x1[u][n]);
                }
                if (normed) {
                    float sum = 0.f;
#pragma unroll
                    for (int n = 0; n < N; ++n)
#pragma unroll
                        for (int e = 0; e < V; ++e) sum = fmaf(a[n][e], a[n][e], fmaf(c[n][e], c[n][e], sum));
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(group_mask, sum, o);
                    const float r = rsqrtf(fmaf(sum, p.inv_d, p.eps));
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        float g0[V], g1[V];
                        widen<T, V>(g0, w0[n]);
                        widen<T, V>(g1, w1[n]);
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            a[n][e] *= r * g0[e];
                            c[n][e] *= r * g1[e];
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    if (turn) {
                        if (!p.interleaved || V == 1) {
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float y = a[n][e] * cs[n][e] - c[n][e] * sn[n][e];
                                c[n][e] = c[n][e] * cs[n][e] + a[n][e] * sn[n][e];
                                a[n][e] = y;
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < V; e += 2) {
                                const int i = e / 2, j = V / 2 + e / 2, e1 = (e + 1) % V;
                                const float y = a[n][e] * cs[n][i] - a[n][e1] * sn[n][i];
                                a[n][e1] = a[n][e1] * cs[n][i] + a[n][e] * sn[n][i];
                                a[n][e] = y;
                                const float z = c[n][e] * cs[n][j] - c[n][e1] * sn[n][j];
                                c[n][e1] = c[n][e1] * cs[n][j] + c[n][e] * sn[n][j];
                                c[n][e] = z;
                            }
                        }
                    }
                    x0[u][n] = narrow<T, V>(a[n]);
                    x1[u][n] = narrow<T, V>(c[n]);
                }
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (is_q && !live) x0[u][n] = x1[u][n] = Raw{};
                if (stored && c0[n] < p.D) *reinterpret_cast<Raw*>(dst + u * d2 + c0[n]) = x0[u][n];
                if (stored && c1[n] < p.D) *reinterpret_cast<Raw*>(dst + u * d2 + c1[n]) = x1[u][n];
            }
        }
    }
}

template <typename T, int V, int LPH, int N, int U>
int launch_group(HeadsParams& p, cudaStream_t st) {
    p.parts_q = (p.Hq + U - 1) / U;
    p.parts_k = (p.Hk + U - 1) / U;
    p.parts = (unsigned)(p.parts_q + p.parts_k * (p.v ? 2 : 1));
    // as many groups as are resident at once, two CTAs an SM: each has its set-up behind it after one token
    const long long resident = (long long)device_sms() * 2 * (kThreads / LPH);
    const long long abreast = resident / p.parts < 1 ? 1 : resident / p.parts;
    p.abreast = abreast < p.tokens ? (unsigned)abreast : p.tokens;
    const unsigned grid = (unsigned)(((long long)p.abreast * p.parts + kThreads / LPH - 1) / (kThreads / LPH));
    launch_chained(heads_kernel<T, V, LPH, N, U>, grid, kThreads, 0, st, p);
    CONVNN_CHECK_LAUNCH("qk_norm_rope");
    return CONVNN_OK;
}

template <typename T, int V>
int launch_vectors(HeadsParams& p, cudaStream_t st) {
    const int pairs = (p.D / V + 1) / 2;
    if (pairs <= 4) return launch_group<T, V, 4, 1, 4>(p, st);
    if (pairs <= 8) return launch_group<T, V, 8, 1, 4>(p, st);
    if (pairs <= 16) return launch_group<T, V, 16, 1, 4>(p, st);
    return launch_group<T, V, 32, 1, 4>(p, st);
}

template <typename T>
int launch_of(HeadsParams& p, cudaStream_t st) {
    // V channels at once where every row, weight and table row starts on a boundary of V values and the pairs' halves are whole vectors
    auto fits = [&](int V) {
        const int bytes = V * (int)sizeof(T);
        if (p.half % V || (p.D - 2 * p.half) % (2 * V) || (p.half && (p.rope_stride % 4 || !aligned16(p.rope)))) return false;
        auto on = [&](const void* a, const long long* s) {
            if (!a) return true;
            for (int i = 0; i < 3; ++i)
                if (s[i] % V) return false;
            return reinterpret_cast<uintptr_t>(a) % bytes == 0;
        };
        const long long none[3] = {0, 0, 0};
        return on(p.q, p.qs) && on(p.k, p.ks) && on(p.v, p.vs) && on(p.q_out, p.qo) && on(p.k_out, p.ko) && on(p.v_out, p.vo) &&
               on(p.wq, none) && on(p.wk, none);
    };
    if constexpr (sizeof(T) == 2) {
        if (fits(8)) return launch_vectors<T, 8>(p, st);
    }
    if (fits(4)) return launch_vectors<T, 4>(p, st);
    return launch_group<T, 1, 32, 4, 2>(p, st);          // a channel at a time
}

}  // namespace

int launch_heads(const convnn_heads* h, const convnn_cache* cache, const int32_t* lengths, const int32_t* counts, cudaStream_t st) {
    HeadsParams p{};
    p.q = h->q; p.k = h->k; p.v = cache ? h->v : nullptr;
    p.q_out = h->q_out; p.k_out = cache ? cache->k : h->k_out; p.v_out = cache ? cache->v : nullptr;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = h->q_stride[i]; p.ks[i] = h->k_stride[i]; p.vs[i] = h->v_stride[i];
        p.qo[i] = h->q_out_stride[i]; p.ko[i] = h->k_out_stride[i];
    }
    if (cache) {                                         // (a cache's strides are given as page, head, row)
        p.ko[0] = cache->k_stride[0]; p.ko[1] = cache->k_stride[2]; p.ko[2] = cache->k_stride[1];
        p.vo[0] = cache->v_stride[0]; p.vo[1] = cache->v_stride[2]; p.vo[2] = cache->v_stride[1];
        p.table = cache->table ? cache->table : lengths;   // (not read where a sequence has no pages)
        p.table_stride = cache->table_stride;
        p.pages = cache->pages; p.page_size = cache->page_size; p.width = cache->width;
        p.lengths = lengths; p.counts = counts;
    }
    p.wq = h->q_weight; p.wk = h->k_weight;
    p.rope = h->rope; p.rope_stride = h->rope_stride; p.rope_rows = h->rope_rows;
    p.positions = h->positions;
    p.pos_stride[0] = h->position_stride[0]; p.pos_stride[1] = h->position_stride[1];
    p.T = h->T; p.tokens = (unsigned)h->B * (unsigned)h->T;
    p.Hq = h->q ? h->Hq : 0; p.Hk = h->k ? h->Hk : 0;
    p.D = h->D; p.half = h->rope ? h->rotary / 2 : 0; p.interleaved = h->interleaved;
    p.eps = h->eps; p.inv_d = 1.0f / (float)h->D;
    return h->dtype == CONVNN_F32 ? launch_of<float>(p, st) : launch_of<__nv_bfloat16>(p, st);
}

}  // namespace convnn
