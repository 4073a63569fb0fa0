// What the kernels of attention over a paged cache share: the call's parameters, the work's division among CTAs and the places of what
// they hand on to one another.
//
// A unit is a tile of query rows (row = token * group + head of the group) of one sequence and key head; its keys come in tiles.  Tiles of
// all units, in order, are divided evenly among the CTAs, whatever the sequences' lengths: they are on the device, and the host never
// learns them.  A unit whose tiles belong to several CTAs is joined from their unnormalised sums by a second kernel, which also writes the
// rows that no unit has (tokens behind a sequence's count, nothing to attend to).  The order of every sum is the division's, so that
// results do not change from run to run.
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace convnn {
namespace paged {

constexpr int kTileKeys = 128;                   // keys of a tile on the tensor cores

struct Params {
    const void *q, *k, *v;
    void* out;
    long long qs[3], os[3];                      // batch, token, head
    long long ks[3], vs[3];                      // page, head, row
    const int32_t *table, *lengths, *counts;
    const long long* tree;                       // (B, T) masks, nullptr: a chain
    long long table_stride, tree_stride[2];
    int B, T, Hk, G, D, pages, page_size, width;
    int row_tiles, rows_per_tile, tile;          // of T * G rows; keys per tile
    float scale_log2;                            // scale * log2(e)
    float* partial;                              // [2 * CTAs][rows_per_tile * (D + 2) + 4]: sums, maxima, sums of weights, what was not finite
    long long slot;                              // floats of one of them
    int ctas;
    int split;                                   // CTAs of a cluster that share a unit, each an even part of its tiles; 0: division over all

    // entry / page_size of an entry below 2^31: the product with 2^slot_shift / page_size, rounded up to 32 bits, is off by less than
    // entry * page_size < 2^slot_shift
    uint32_t slot_factor;
    int slot_shift;
    __device__ __forceinline__ int slot_at(int entry) const { return (int)(((unsigned long long)(unsigned)entry * slot_factor) >> slot_shift); }
};

// One sequence.
struct Sequence {
    int length, count, total;                    // cached entries, drafted tokens, both (as far as the table goes)
    int tiles, row_tiles;                        // of keys; of rows that are there
    __device__ __forceinline__ int work() const { return tiles * row_tiles; }
};
__device__ __forceinline__ Sequence sequence_of(const Params& p, int b) {
    Sequence s;
    const int room = p.width * p.page_size;      // (at most 2^30)
    s.length = min(max(p.lengths[b], 0), room);
    s.count = p.counts ? min(max(p.counts[b], 0), p.T) : p.T;
    s.total = s.count ? min(s.length + s.count, room) : 0;
    s.tiles = (s.total + p.tile - 1) / p.tile;
    s.row_tiles = (s.count * p.G + p.rows_per_tile - 1) / p.rows_per_tile;
    return s;
}
// Whole warp: tiles of all units (fewer than 2^31), and of the sequences before b.
__device__ __forceinline__ int total_work(const Params& p, int b, int& before) {
    const int lane = threadIdx.x & 31;
    int all = 0, first = 0;
    for (int i = lane; i < p.B; i += 32) {
        const int w = sequence_of(p, i).work() * p.Hk;
        all += w;
        if (i < b) first += w;
    }
    before = (int)__reduce_add_sync(0xffffffffu, (unsigned)first);
    return (int)__reduce_add_sync(0xffffffffu, (unsigned)all);
}
// How the tiles are divided: `ctas` CTAs get some, the first `more` of them one more than the others.
struct Division {
    int ctas, each, more;
    __device__ __forceinline__ Division(int work, int most) {
        ctas = min(work, most);
        each = ctas ? work / ctas : 0;
        more = work - each * ctas;
    }
    __device__ __forceinline__ int first(int cta) const { return cta * each + min(cta, more); }
    __device__ __forceinline__ int cta_of(int at) const {
        const int rich = more * (each + 1);
        return at < rich ? at / (each + 1) : more + (at - rich) / each;
    }
};

// A CTA's way through its tiles.
struct Cursor {
    Sequence s;
    int b, h, rt, tile;
    int left;                                    // tiles that are still to come, this one included

    // Whole warp; the same in all lanes.
    __device__ __forceinline__ void start(const Params& p, int cta) {
        int none;
        const Division d(total_work(p, 0, none), p.ctas);
        b = h = rt = tile = left = 0;
        if (cta < d.ctas) find(p, d.first(cta), d.first(cta + 1) - d.first(cta));
    }
    // A unit of its own for every `split` CTAs, a part of its tiles each; whatever is not there has none.
    __device__ __forceinline__ void start_part(const Params& p, int cta) {
        const int unit = cta / p.split, part = cta - unit * p.split, rest = unit % (p.Hk * p.row_tiles);
        b = unit / (p.Hk * p.row_tiles);
        h = rest / p.row_tiles;
        rt = rest - h * p.row_tiles;
        s = sequence_of(p, b);
        tile = s.tiles * part / p.split;
        left = rt < s.row_tiles ? s.tiles * (part + 1) / p.split - tile : 0;
    }
    // `count` tiles from `begin` on.
    __device__ __forceinline__ void find(const Params& p, int begin, int count) {
        const int lane = threadIdx.x & 31;
        left = count;
        int before = 0;
        for (int b0 = 0;; b0 += 32) {
            int w = 0;
            if (b0 + lane < p.B) w = sequence_of(p, b0 + lane).work() * p.Hk;
            int sum = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned found = __ballot_sync(0xffffffffu, before + sum > begin);
            if (found) {
                const int at = __ffs(found) - 1;
                b = b0 + at;
                before += __shfl_sync(0xffffffffu, sum - w, at);
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        s = sequence_of(p, b);
        const int rest = begin - before;
        h = rest / s.work();
        const int in_head = rest - h * s.work();
        rt = in_head / s.tiles;
        tile = in_head - rt * s.tiles;
    }
    __device__ __forceinline__ void next(const Params& p) {
        if (--left == 0) return;
        if (++tile < s.tiles) return;
        tile = 0;
        if (++rt < s.row_tiles) return;
        rt = 0;
        if (++h < p.Hk) return;
        h = 0;
        do s = sequence_of(p, ++b);
        while (s.work() == 0);
    }
    // Tiles of the unit that belong to this CTA, and the next unit.
    __device__ __forceinline__ int run() const { return min(left, s.tiles - tile); }
    __device__ __forceinline__ void skip(const Params& p, int n) {
        tile += n - 1;
        left -= n - 1;
        next(p);
    }
    __device__ __forceinline__ bool last_of_unit() const { return left == 1 || tile + 1 == s.tiles; }
};

// Mask of the drafted tokens that row r sees; rows that are not there see none.
__device__ __forceinline__ unsigned long long seen_by(const Params& p, const Sequence& s, int b, int row) {
    const int t = row / p.G;
    if (t >= s.count) return 0;
    if (!p.tree) return ~0ull >> (63 - t);
    return (unsigned long long)p.tree[b * p.tree_stride[0] + t * p.tree_stride[1]];
}

// One over a row's sum of weights, the largest of which is 1.  There is none where a row is not there or sees nothing, whose result is zeros, and
// where all that it sees has a score of minus infinity, which has no softmax: NaN.
__device__ __forceinline__ float inverse_of(const Params& p, const Sequence& s, int b, int row, float sum) {
    if (sum != 0.f) return 1.0f / sum;
    if (row >= s.count * p.G) return 0.f;
    const int drafted = s.total - s.length;
    const unsigned long long there = drafted >= 64 ? ~0ull : (1ull << drafted) - 1;
    return s.length > 0 || (seen_by(p, s, b, row) & there) ? CUDART_NAN_F : 0.f;
}

// Values that are not finite do not stay in a product with zero: those of drafted tokens, which some rows see and others do not, are
// taken out before it (a zero in their place) and added to the rows that see them here, at the end.
template <typename T>
__device__ __forceinline__ float not_finite_seen(const Params& p, const Sequence& s, int b, int h, unsigned long long mask, int c) {
    float add = 0.f;
    for (int j = 0; j < s.total - s.length; ++j) {
        const int entry = s.length + j, slot = p.slot_at(entry);
        const int page = p.table[b * p.table_stride + slot];
        if (!(mask >> j & 1) || (unsigned)page >= (unsigned)p.pages) continue;
        const float v = to_f32(static_cast<const T*>(p.v)[page * p.vs[0] + h * p.vs[1] + (entry - slot * p.page_size) * p.vs[2] + c]);
        if (!isfinite(v)) add += v;
    }
    return add;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The partial sums of a CTA's unit: slot 0 if the CTA's first tile is in it, else 1.
__device__ __forceinline__ float* slot_of(const Params& p, int cta, bool first) { return p.partial + (2ll * cta + !first) * p.slot; }

}  // namespace paged

// 128 rows a tile on the tensor cores (tree_attention_tc.cu): bfloat16, up to 128 channels, pages of a multiple of 16 entries.
bool tree_tiles_supported(const convnn_tree_attention* a, const convnn_cache* cache);
int launch_tree_tiles(const paged::Params& p, cudaStream_t st);
}  // namespace convnn
