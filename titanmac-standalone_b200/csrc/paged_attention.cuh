// Attention over paged keys (tmw_paged_attention, tmw_paged_attention_scaled; tmw_paged_tree_attention where its own kernel does not
// go): the line of tiles, the cores, the join.
//
// For every (sequence, key head) the query heads that read it see the persistent keys and the tokens lo .. pos of the sequence;
// with s_j = q k_j scale, o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), m a running maximum: one pass, each key and value read
// once for all heads of the group.  A step does two to a few multiply-adds per number read: HBM bounds it, or, for a
// handful of keys, launch and latency.
//
// The lengths are on the device and may differ by any factor, so the host cannot cut the work up.  The keys of an item - a
// sequence and the heads of one key head, at most kMaxRows of them - come in tiles of 32 or 16, the tiles of all items in one line, and
// every warp of the grid takes an equal piece of the line, whatever the lengths.  A warp has its own ring of tiles in shared
// memory (cp.async), its own running maximum and sums, and meets no barrier on its way: an item that lies in its piece is stored
// from its registers.  Of an item that was cut, the warps of a CTA join their parts through shared memory when all of them are
// done; what was cut between CTAs goes to scratch memory, and a second kernel, launched under the first, joins it in the order of
// the CTAs.
//
// bf16, 553,000 tokens of 12 sequences, 32 heads of 128 on 4: 191 us, 5.9 TB/s; 48 sequences of 1 to 16384 tokens, 32 heads on 8, fp16:
// 119 us, 5.7 TB/s.  (Warps of a CTA on neighbouring tiles, joined at every item's end: 192 and 202 when this took 187 and 118.)
#pragma once

#include <math_constants.h>

#include <type_traits>

#include "paged.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.cuh"

namespace tmw {
namespace {

constexpr int kMaxRows = 16;

struct PagedAttention {
    PageMap map;
    const void *q, *k_pages, *v_pages, *k_pers, *v_pers;
    void* o;
    const float *k_scales, *v_scales, *k_pers_scales, *v_pers_scales;  // of pages in 8 bits
    long long qs[3], os[3];  // {batch, head, node}
    const int32_t* pos;      // with drafted nodes: tokens in front of them
    const int32_t *counts, *positions;  // of the nodes
    const int64_t* seen;
    int nodes;
    int batch, np, window;
    int pers_tiles;         // of the persistent keys
    bool whole_runs;        // sixteen tokens from a multiple of sixteen on lie in one page
    int run;                // as many from a multiple of that on do, 16, 8 or none
    bool bf16;              // of two types with 16 bits
    bool q_pairs, o_pairs;  // queries can be read, outputs stored two at a time
    bool q_wide, o_wide;    // sixteen bytes at a time
    int group;              // query heads of a key head
    int rows, parts;        // query heads of an item at most; items of a key head
    int items;              // of a sequence
    float scale;            // times log2(e)
    int row_bytes;
    float* partial;  // [CTA][2][rows][head_dim]: of the item that a CTA begins in, of the one that begins in it
    float2* sums;    // [CTA][2][rows]: maximum, sum
    float* firsts;   // [CTA][warp][rows][head_dim]: what a warp has of the item that its piece begins in
    int4* joins;     // [CTA]: the item that begins in it and ends in another one - sequence (-1: none), item, last CTA
    int* status;
    long long room[3];
};
// What a launch takes of the host goes by its arguments' size, in steps that repeat every 64 bytes (driver 580.159; this kernel's launch and
// its join's, us: 232 bytes 4.3, 240 - 272 4.7, 280 - 288 4.0, 296 4.4, 304 - 336 4.7, 344 - 352 4.0).
static_assert(sizeof(PagedAttention) % 64 == 24 || sizeof(PagedAttention) % 64 == 32, "a size that launches quickly");

// Tiles, of KT keys, of sequence b's items; lo, pos: its first and last token seen (lo > pos: none); count: its drafted nodes, the last
// tokens.  0 with bad: no such position.  TREE: with drafted nodes instead of one new token.
template <int KT, bool TREE>
__device__ __forceinline__ int tiles_of(const PagedAttention& p, int b, int& lo, int& pos, int& count, bool& bad) {
    pos = __ldg(p.pos + b);
    lo = 0;
    count = 1;
    if constexpr (TREE) {
        const int start = pos;
        count = p.counts != nullptr ? __ldg(p.counts + b) : p.nodes;
        bad = start < -1 || (start >= 0 && (count < 0 || count > p.nodes || (long long)start + count > p.map.capacity));
        if (bad || start < 0 || count == 0) return 0;
        pos = start + count - 1;
        if (p.window >= 0 && start > p.window) lo = start - p.window;
        return p.pers_tiles + pos / KT - lo / KT + 1;
    }
    bad = pos < -1 || pos >= p.map.capacity;
    if (bad) return 0;
    if (pos < 0) return p.pers_tiles;
    if (p.window >= 0 && pos > p.window) lo = pos - p.window;
    return p.pers_tiles + pos / KT - lo / KT + 1;
}

// A place in the line.  An item takes COST more units of it than it has tiles, ahead of them: loading the queries and
// storing the output hold a warp up for about that long, and pieces of equal length are to take equal time.
// items of a key head's query rows: of a sequence with so many nodes
template <bool TREE>
__device__ __forceinline__ int parts_of(const PagedAttention& p, int count) {
    return TREE ? (count * p.group + p.rows - 1) / p.rows : p.parts;
}
template <int KT, bool TREE, int COST>
struct Cursor {
    int b, item;  // sequence, item of it
    int head;     // the item's key head
    int t, n;     // unit of the item; units of an item
    int lo, pos, count;
    __device__ __forceinline__ void sequence(const PagedAttention& p) {
        bool bad;
        n = tiles_of<KT, TREE>(p, b, lo, pos, count, bad);
        if (n > 0) n += COST;
    }
    __device__ __forceinline__ int parts(const PagedAttention& p) const { return parts_of<TREE>(p, count); }
    __device__ __forceinline__ int tile() const { return t - COST; }
    // the next item's first unit; not past the end of the line
    __device__ __forceinline__ void next_item(const PagedAttention& p) {
        t = 0;
        const int of_head = parts(p);
        if (++item < (TREE ? p.map.kv_heads * of_head : p.items)) {
            head = of_head == 1 ? item : item / of_head;
            return;
        }
        item = head = 0;
        do {
            ++b;
            sequence(p);
        } while (n == 0);
    }
};

__device__ __forceinline__ long long scan(long long x) {  // sums up to each lane
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    return x;
}

// The piece of the line of the CTA's `warp` of `most`: units [first, end), of pieces of `per` units, `warps` of which go to a CTA; and the
// place where it begins.
struct Share {
    long long first, end, per;
    int warps;
};
template <int KT, bool TREE, int COST>
__device__ __forceinline__ Share find_share(const PagedAttention& p, Cursor<KT, TREE, COST>& at, int warp, int most) {
    const int lane = threadIdx.x & 31;
    auto units = [&](int b) -> long long {
        if (b >= p.batch) return 0;
        int lo, pos, count;
        bool bad;
        const int n = tiles_of<KT, TREE>(p, b, lo, pos, count, bad);
        const int items = TREE ? p.map.kv_heads * parts_of<TREE>(p, count) : p.items;
        return n > 0 ? (long long)(n + COST) * items : 0;
    };
    // each lane sums up a run of sequences
    const int run = (p.batch + 31) / 32;
    long long mine = 0;
#pragma unroll 8
    for (int i = 0; i < run; ++i) mine += units(lane * run + i);
    const long long upto = scan(mine), total = __shfl_sync(0xffffffffu, upto, 31);
    Share s;
    s.warps = most;
    s.per = (total + (long long)gridDim.x * most - 1) / ((long long)gridDim.x * most);
    if (s.per <= COST) {  // a tile at least, and with less than that for every warp all SMs rather than all warps of some
        s.per = COST + 1;
        s.warps = (int)((total + gridDim.x * s.per - 1) / (gridDim.x * s.per));
        s.warps = max(min(s.warps, most), 1);
    }
    s.first = s.per * (blockIdx.x * (long long)s.warps + warp);
    s.end = warp >= s.warps ? s.first : s.first + s.per < total ? s.first + s.per : total;
    if (s.first >= s.end) return s;
    // the run that holds the first unit, and the sequence in it
    const int owner = __ffs(__ballot_sync(0xffffffffu, upto > s.first)) - 1;
    long long before = __shfl_sync(0xffffffffu, upto - mine, owner);
    for (int i = 0;; i += 32) {
        const int b = owner * run + i + lane;
        const long long own = i + lane < run ? units(b) : 0, sum = scan(own) + before;
        const uint32_t there = __ballot_sync(0xffffffffu, sum > s.first);
        if (there != 0) {
            const int l = __ffs(there) - 1;
            at.b = owner * run + i + l;
            before = __shfl_sync(0xffffffffu, sum - own, l);
            break;
        }
        before = __shfl_sync(0xffffffffu, sum, 31);
    }
    at.sequence(p);
    const long long inside = s.first - before;
    at.item = (int)(inside / at.n);
    at.t = (int)(inside - (long long)at.item * at.n);
    at.head = at.item / at.parts(p);
    return s;
}

// The query rows of an item: heads first .. of a key head or, with drafted nodes, rows first .. of the (node, head) pairs.
struct Rows {
    int b, head, first, n;  // head: the key head
};
template <bool TREE>
__device__ __forceinline__ Rows rows_of(const PagedAttention& p, int b, int head, int part, int count) {
    const int first = part * p.rows;
    return {b, head, first, min(p.rows, (TREE ? count * p.group : p.group) - first)};
}
// where row r of them is, through {batch, head, node} strides
template <bool TREE>
__device__ __forceinline__ long long row_at(const PagedAttention& p, const long long (&strides)[3], const Rows& rows, int r) {
    const long long at = rows.b * strides[0];
    if constexpr (!TREE) return at + (rows.head * p.group + rows.first + r) * strides[1];
    const int node = (rows.first + r) / p.group, g = rows.first + r - node * p.group;
    return at + (rows.head * p.group + g) * strides[1] + node * strides[2];
}
// the node's first token seen, and which nodes it sees
__device__ __forceinline__ int first_seen(const PagedAttention& p, int b, int start, int node) {
    if (p.window < 0) return 0;
    return max(max(__ldg(p.positions + (long long)b * p.nodes + node), start) - p.window, 0);
}
__device__ __forceinline__ uint64_t nodes_seen(const PagedAttention& p, int b, int count, int node) {
    return (uint64_t)__ldg(p.seen + (long long)b * p.nodes + node) & (~0ull >> (64 - count));
}

// 1 / l, what a sum of weights turns into (the largest score's weight is 1 or more: no sum at all is that of scores of -inf)
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? CUDART_NAN_F : 1.0f / l; }
// the same of a row of an item; a node may see nothing, its output is zero
template <bool TREE>
__device__ __forceinline__ float inverse_of(const PagedAttention& p, const Rows& rows, int r, float l) {
    if (TREE && l == 0.f && p.np == 0) {
        const int start = __ldg(p.pos + rows.b), count = p.counts != nullptr ? __ldg(p.counts + rows.b) : p.nodes;
        const int node = (rows.first + r) / p.group;
        if (first_seen(p, rows.b, start, node) >= start && nodes_seen(p, rows.b, count, node) == 0) return 0.f;
    }
    return inverse(l);
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}

// The same where tiles come by TMA: of the pages and the persistent keys as rows of 16-bit pairs.
struct alignas(64) PagedAttentionBulk : PagedAttention {
    CUtensorMap k_map, v_map, k_pers_map, v_pers_map;
};

// A warp's ring: tiles of keys, as many of values, and which of their rows are seen and which have no page; the first key's token (-1:
// persistent ones); with pages in 8 bits the rows' scales, of the keys and of the values.
struct Ring {
    unsigned char* tiles;
    uint2* marks;
    int* places;
    float* scales;
    uint32_t arrived;  // with TMA: a barrier for each stage
};
template <typename P>
constexpr bool kScaled = sizeof(P) == 1;

// Brings a warp's tiles into its ring, one after the other.  Rows that do not count become zeros: whatever stands in a page behind
// a sequence's end, infinities and NaN among them, reaches no product.  A lane looks its row's page up a tile ahead of the copies
// that need it.  Where pages are made of sixteens, so are the tiles' runs of memory; else every row is found by itself.
template <typename P, int KT, bool TREE, int COST, typename Layout>
struct Loader {
    static constexpr bool kBulk = false;
    const PagedAttention& p;
    const Ring& ring;
    const Layout& lay;
    Cursor<KT, TREE, COST> at;
    int j0, first, last;  // of the tile: its first key; rows first .. last are seen
    int slot, page;       // of this lane's row

    __device__ __forceinline__ bool persistent() const { return at.tile() < p.pers_tiles; }
    __device__ __forceinline__ int row_of_lane() const { return threadIdx.x & (KT - 1) & 31; }
    __device__ __forceinline__ void look() {
        const bool pers = persistent();
        const int r = row_of_lane();
        j0 = (pers ? at.tile() : at.lo / KT + at.tile() - p.pers_tiles) * KT;
        first = pers ? 0 : max(at.lo - j0, 0);
        last = min(pers ? p.np - 1 - j0 : at.pos - j0, KT - 1);
        if (!pers && r >= first && r <= last) {
            const uint32_t column = p.map.page.div((uint32_t)(j0 + r));
            slot = j0 + r - (int)(column * p.map.page.d);
            page = __ldg(p.map.table + at.b * p.map.table_stride + column);
        }
    }
    __device__ __forceinline__ void issue(int stage) {
        const int lane = threadIdx.x & 31, r = row_of_lane();
        const bool pers = persistent(), mine = r >= first && r <= last;
        const unsigned char *k, *v;
        long long row = -1;  // where this lane's row is, in elements
        if (pers) {
            k = static_cast<const unsigned char*>(p.k_pers);
            v = static_cast<const unsigned char*>(p.v_pers);
            if (mine) row = ((long long)at.head * p.np + j0 + r) * p.map.head_dim;
        } else {
            k = static_cast<const unsigned char*>(p.k_pages);
            v = static_cast<const unsigned char*>(p.v_pages);
            if (mine && (uint32_t)page < (uint32_t)p.map.pages)
                row = (((long long)page * p.map.kv_heads + at.head) * p.map.page.d + slot) * p.map.head_dim;
        }
        const uint32_t seen = (2u << last) - (1u << first), lost = __ballot_sync(0xffffffffu, mine && row < 0) & (0xffffffffu >> (32 - KT));
        if (lane == 0) {
            ring.marks[stage] = make_uint2(seen, lost);
            if (TREE) ring.places[stage] = pers ? -1 : j0;
        }
        if constexpr (kScaled<P>) {
            if (lane < KT) {
                const long long token = pers ? (long long)at.head * p.np + j0 + r : ((long long)page * p.map.kv_heads + at.head) * p.map.page.d + slot;
                const bool there = mine && row >= 0;
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring.scales + (stage * 2 * KT + lane));
                copy4(dst, there ? (pers ? p.k_pers_scales : p.k_scales) + token : p.k_scales, there);
                copy4(dst + KT * 4, there ? (pers ? p.v_pers_scales : p.v_scales) + token : p.k_scales, there);
            }
        }
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring.tiles) + stage * 2 * KT * lay.pitch();
        const int chunks = lay.chunks();
        // a lane's chunks, every 32nd one: chunk c of row rr (by steps: chunks is not always a constant)
        struct Chunk {
            int rr, c;
        };
        const Chunk start{lane / chunks, lane % chunks};
        auto after = [&](Chunk x) {
            x.rr += 32 / chunks;
            x.c += 32 % chunks;
            if (x.c >= chunks) x.c -= chunks, ++x.rr;
            return x;
        };
        if (pers || p.whole_runs) {
#pragma unroll
            for (int h = 0; h < KT / 16; ++h) {
                const int from = min(max(first, h * 16), KT - 1);  // a row that has the run's page, if any has
                const long long off = (__shfl_sync(0xffffffffu, row, from) - (from - h * 16) * p.map.head_dim) * (long long)sizeof(P) + lane * 16;
                const unsigned char *kr = k + off, *vr = v + off;
                const int n = 16 * chunks;
                const uint32_t want = seen >> (h * 16) & 0xffffu & ~(lost >> (h * 16));
                Chunk x = start;
                if (want == 0xffffu) {
#pragma unroll
                    for (int i0 = 0; i0 < n; i0 += 32, x = after(x)) {
                        if (n % 32 != 0 && x.rr >= 16) break;
                        const uint32_t dst = to + lay.offset(h * 16 + x.rr, x.c);
                        copy16(dst, kr + i0 * 16, true);
                        copy16(dst + KT * lay.pitch(), vr + i0 * 16, true);
                    }
                } else {
#pragma unroll 4
                    for (int i0 = 0; i0 < n; i0 += 32, x = after(x)) {
                        if (n % 32 != 0 && x.rr >= 16) break;
                        const uint32_t dst = to + lay.offset(h * 16 + x.rr, x.c);
                        const bool there = want >> x.rr & 1;  // (no byte is read where not: any address will do)
                        copy16(dst, there ? static_cast<const void*>(kr + i0 * 16) : p.sums, there);
                        copy16(dst + KT * lay.pitch(), there ? static_cast<const void*>(vr + i0 * 16) : p.sums, there);
                    }
                }
            }
        } else {
            Chunk x = start;
            for (int i0 = 0; i0 < KT * chunks; i0 += 32, x = after(x)) {
                const long long at_row = __shfl_sync(0xffffffffu, row, x.rr & (KT - 1));
                if (x.rr >= KT) continue;
                const bool there = at_row >= 0;
                const long long off = at_row * (long long)sizeof(P) + x.c * 16;
                const uint32_t dst = to + lay.offset(x.rr, x.c);
                copy16(dst, there ? static_cast<const void*>(k + off) : p.sums, there);
                copy16(dst + KT * lay.pitch(), there ? static_cast<const void*>(v + off) : p.sums, there);
            }
        }
    }
};

// The same by TMA, a run of rows at a time: pages made of sixteens, or of eights, hold as many neighbouring tokens as one run of memory, and the
// hardware puts the chunks of a row where the layout has them.  Where the next 32 runs are every lane finds out for one of them,
// so a tile costs a handful of instructions of one lane and two shuffles instead of an address and a copy for every sixteen bytes
// (heads of 64, int8: 311 instructions to a tile of 32 keys with every tile's rows looked up for itself).  What is not seen in a run is
// brought too: a core has to see to it that it does no harm.
template <typename P, int KT, bool TREE, int COST, typename Layout>
struct BulkLoader {
    static constexpr bool kBulk = true;
    static_assert(KT == 32, "marks are a word");
    const PagedAttentionBulk& p;
    const Ring& ring;
    const Layout& lay;
    Cursor<KT, TREE, COST> at;
    int planned = 1 << 30, page = -1;  // tile of the item whose first run is lane 0's; this lane's page
    int row = -1;                      // this lane's run among the rows of the pool (of the persistent keys); -1: not wanted, -2: nowhere
    uint32_t there = 0;                // lanes whose runs are to be brought

    __device__ __forceinline__ int key_of_run(int tile, bool pers) const {
        return (pers ? tile : at.lo / KT + tile - p.pers_tiles) * KT;
    }
    // Looks the pages of the runs from the next tile on up, if that has no plan yet.
    __device__ __forceinline__ void look() {
        const int tile = at.tile();
        if (tile >= planned && tile < planned + p.run) return;  // (32 runs are those of p.run tiles)
        planned = tile;
        const int lane = threadIdx.x & 31, r = lane * p.run, mine = tile + r / KT;
        const bool pers = mine < p.pers_tiles;
        const int j = key_of_run(mine, pers) + r % KT;
        page = -1;
        row = -1;
        if (mine < at.n - COST && j <= (pers ? p.np - 1 : at.pos) && j + p.run > (pers ? 0 : at.lo)) {
            row = j;
            if (!pers) {
                const uint32_t column = p.map.page.div((uint32_t)j);
                row = j - (int)(column * p.map.page.d);
                page = __ldg(p.map.table + at.b * p.map.table_stride + column);
            }
        }
        there = 0;
    }
    // A whole plan's rows, once their pages have come.
    __device__ __forceinline__ void find() {
        const int lane = threadIdx.x & 31, mine = planned + lane * p.run / KT;
        if (row >= 0) {
            if (mine < p.pers_tiles) row += at.head * p.np;
            else row = (uint32_t)page < (uint32_t)p.map.pages ? (page * p.map.kv_heads + at.head) * (int)p.map.page.d + row : -2;
        }
        there = __ballot_sync(0xffffffffu, row >= 0);
    }
    __device__ __forceinline__ void issue(int stage) {
        const int tile = at.tile();
        const bool pers = tile < p.pers_tiles;
        if (tile == planned) find();
        const int runs = KT / p.run, first_run = (tile - planned) * runs;
        const int j0 = key_of_run(tile, pers), first = pers ? 0 : max(at.lo - j0, 0), last = min((pers ? p.np - 1 : at.pos) - j0, KT - 1);
        const uint32_t bar = ring.arrived + stage * 8;
        constexpr int kBoxes = Layout::kBoxes, kHalf = KT * Layout::kBoxBytes;
        const int box = p.run * Layout::kBoxBytes, here = __popc(there >> first_run & ((1u << runs) - 1));
        const uint32_t seen = (2u << last) - (1u << first);
        uint32_t lost = 0;
        int run[KT / 8];
#pragma unroll
        for (int i = 0; i < KT / 8; ++i) {
            run[i] = -1;
            if (i >= 2 && runs == 2) continue;
            run[i] = __shfl_sync(0xffffffffu, row, first_run + i);
            if (run[i] == -2) lost |= ((1u << p.run) - 1) << i * p.run;
        }
        if (kScaled<P> && pers) {  // scales that need not begin on sixteen bytes
            const int r = threadIdx.x & 31;
            const bool mine = r <= last;
            const int of = at.head * p.np + j0 + r;
            ring.scales[stage * 2 * KT + r] = mine ? __ldg(p.k_pers_scales + of) : 0.f;
            ring.scales[stage * 2 * KT + KT + r] = mine ? __ldg(p.v_pers_scales + of) : 0.f;
            ptx::fence_proxy_async_smem();  // (before the copies of a later tile write there)
            __syncwarp();
        }
        if (ptx::elect_one()) {  // (all of it in one such branch: what one lane alone runs needs no loop over the lanes' operands)
            ring.marks[stage] = make_uint2(seen, lost & seen);
            if (TREE) ring.places[stage] = pers ? -1 : j0;
            const uint32_t keys = (uint32_t)__cvta_generic_to_shared(ring.tiles) + stage * 2 * KT * Layout::pitch();
            const uint32_t scales = (uint32_t)__cvta_generic_to_shared(ring.scales) + stage * 2 * KT * 4;
            const CUtensorMap *k = pers ? &p.k_pers_map : &p.k_map, *v = pers ? &p.v_pers_map : &p.v_map;
            const int scale_bytes = kScaled<P> && !pers ? p.run * 4 : 0;
            ptx::mbar_expect_tx(bar, here * 2 * (kBoxes * box + scale_bytes));
#pragma unroll
            for (int i = 0; i < KT / 8; ++i) {
                if (run[i] < 0) continue;
#pragma unroll
                for (int c = 0; c < kBoxes; ++c) {
                    ptx::tma_load_2d(keys + c * kHalf + i * box, k, bar, c * Layout::kBoxBytes / 2, run[i]);
                    ptx::tma_load_2d(keys + KT * Layout::pitch() + c * kHalf + i * box, v, bar, c * Layout::kBoxBytes / 2, run[i]);
                }
                if (kScaled<P> && !pers) {
                    ptx::bulk_load(scales + i * scale_bytes, p.k_scales + run[i], scale_bytes, bar);
                    ptx::bulk_load(scales + KT * 4 + i * scale_bytes, p.v_scales + run[i], scale_bytes, bar);
                }
            }
        }
    }
};

// queries and outputs of either 16-bit type, which p.bf16 tells apart
struct Any16 {
    uint16_t bits;
};
template <typename T>
__device__ __forceinline__ void put(const PagedAttention& p, T* to, float x) {
    if constexpr (std::is_same<T, Any16>::value) {
        to->bits = p.bf16 ? __bfloat16_as_ushort(from_f32<__nv_bfloat16>(x)) : __half_as_ushort(from_f32<__half>(x));
    } else {
        *to = from_f32<T>(x);
    }
}
template <typename T>
__device__ __forceinline__ float get(const PagedAttention& p, const T* from) {
    if constexpr (std::is_same<T, Any16>::value) {
        return p.bf16 ? __uint_as_float((uint32_t)from->bits << 16) : __half2float(__ushort_as_half(from->bits));
    } else {
        return to_f32<T>(*from);
    }
}

// ---- the core on CUDA cores: every type, head_dim a multiple of 8 --------------------------------------------------------
// Lane l has key l % 16 of a tile and one half of the head's dimensions of its scores; then the four dimensions from 4 l on (and
// from 128 + 4 l, with QUADS 2) of the outputs.  kRows query heads, their numbers as fp32 in shared memory.
template <typename T>
struct SimtLayout {
    int bytes;  // of a row; 16 more keep the rows of 8 lanes off each other's banks
    __host__ __device__ __forceinline__ int pitch() const { return bytes + 16; }
    __device__ __forceinline__ int chunks() const { return bytes / 16; }
    __device__ __forceinline__ int offset(int r, int c) const { return r * pitch() + c * 16; }
};

template <typename T>
__device__ __forceinline__ float4 load4(const unsigned char* at);
template <>
__device__ __forceinline__ float4 load4<float>(const unsigned char* at) { return *reinterpret_cast<const float4*>(at); }
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const unsigned char* at) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}
template <>
__device__ __forceinline__ float4 load4<__half>(const unsigned char* at) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

template <>
__device__ __forceinline__ float4 load4<int8_t>(const unsigned char* at) {
    const char4 w = *reinterpret_cast<const char4*>(at);
    return make_float4(w.x, w.y, w.z, w.w);
}
template <>
__device__ __forceinline__ float4 load4<E4m3>(const unsigned char* at) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(at);
    const float2 a = __half22float2(from_e4m3(w)), b = __half22float2(from_e4m3(w >> 16));
    return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ void add_product(float4& acc, float w, const float4& x) {
    acc.x = fmaf(w, x.x, acc.x);
    acc.y = fmaf(w, x.y, acc.y);
    acc.z = fmaf(w, x.z, acc.z);
    acc.w = fmaf(w, x.w, acc.w);
}

// T: of queries and outputs, P: of keys and values.
template <typename T, typename P, int ROWS, int QUADS, bool TREE = false>
struct SimtCore {
    static constexpr int kRows = ROWS, KT = 16;
    using Layout = SimtLayout<P>;
    static constexpr int kItemCost = 1;
    using Load = Loader<P, KT, TREE, kItemCost, Layout>;
    using Args = PagedAttention;
    const PagedAttention& p;
    float* q;        // [kRows][head_dim], of the CTA's warp
    float* weights;  // [KT][kRows]
    float m[kRows], l[kRows];
    // with drafted nodes
    int start, low[kRows];      // tokens in front of them; first of these that a row sees
    uint64_t nodes[kRows];      // those that it sees
    float4 o[kRows][QUADS];

    // shared memory of a warp besides its ring
    static __host__ __device__ int extra(int head_dim) { return (kRows * head_dim + KT * kRows) * (int)sizeof(float); }

    __device__ SimtCore(const PagedAttention& p, unsigned char* mine) : p(p), q(reinterpret_cast<float*>(mine)) {
        weights = q + kRows * p.map.head_dim;
    }
    __device__ __forceinline__ void load_queries(const Rows& of, int count) {
        const int lane = threadIdx.x & 31, dim = p.map.head_dim;
        if constexpr (TREE) start = __ldg(p.pos + of.b);
        __syncwarp();
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const T* from = static_cast<const T*>(p.q) + row_at<TREE>(p, p.qs, of, r);
            for (int i = lane; i < dim; i += 32) q[r * dim + i] = r < of.n ? get(p, from + i) : 0.f;
            if constexpr (TREE) {
                const int node = (of.first + r) / p.group;
                low[r] = r < of.n ? first_seen(p, of.b, start, node) : 0;
                nodes[r] = r < of.n ? nodes_seen(p, of.b, count, node) : 0;
            }
        }
        __syncwarp();
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            m[r] = -CUDART_INF_F;
            l[r] = 0.f;
#pragma unroll
            for (int h = 0; h < QUADS; ++h) o[r][h] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ void tile(const Ring& ring, int stage, uint2 marks, const Layout& lay) {
        const unsigned char* tile = ring.tiles + stage * 2 * KT * lay.pitch();
        const int lane = threadIdx.x & 31, key = lane & (KT - 1), dim = p.map.head_dim, half = dim / 2;
        const unsigned char* row = tile + key * lay.pitch();
        float s[kRows] = {};
#pragma unroll 4
        for (int i = (lane >> 4) * half; i < (lane >> 4) * half + half; i += 4) {
            const float4 k4 = load4<P>(row + i * sizeof(P));
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float4 q4 = *reinterpret_cast<const float4*>(q + r * dim + i);
                s[r] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[r]))));
            }
        }
        const bool there = marks.x >> key & 1, lost = marks.y >> key & 1;
        float k_scale = p.scale, v_scale = 1.f;
        if constexpr (kScaled<P>) {
            k_scale *= ring.scales[stage * 2 * KT + key];
            v_scale = ring.scales[stage * 2 * KT + KT + key];
        }
        int token = -1;
        if constexpr (TREE) token = ring.places[stage] < 0 ? -1 : ring.places[stage] + key;
        float w[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            bool seen = there;
            if constexpr (TREE)
                if (token >= 0) seen = there && (token < start ? token >= low[r] : (nodes[r] >> ((token - start) & 63) & 1) != 0);
            const bool bad = TREE ? lost && seen : lost;
            float x = (s[r] + __shfl_xor_sync(0xffffffffu, s[r], 16)) * k_scale;
            x = bad ? CUDART_NAN_F : seen ? x : -CUDART_INF_F;
            float top = x;
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float now = fmaxf(m[r], top), base = now == -CUDART_INF_F ? 0.f : now;
            const float keep = m[r] == -CUDART_INF_F ? 1.f : exp2f(m[r] - base);  // (nothing to keep, or NaN)
            m[r] = now;
            w[r] = seen ? exp2f(x - base) : 0.f;
            l[r] = l[r] * keep + w[r];
#pragma unroll
            for (int h = 0; h < QUADS; ++h) {
                o[r][h].x *= keep; o[r][h].y *= keep; o[r][h].z *= keep; o[r][h].w *= keep;
            }
        }
        if (lane < KT) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) weights[key * kRows + r] = kScaled<P> && w[r] != 0.f ? w[r] * v_scale : w[r];
        }
        __syncwarp();
        const unsigned char* values = tile + KT * lay.pitch();
#pragma unroll
        for (int h = 0; h < QUADS; ++h) {
            const int i = h * 128 + lane * 4;
            if (i >= dim) break;
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const float4 v4 = load4<P>(values + j * lay.pitch() + i * sizeof(P));
                float wj[kRows];
#pragma unroll
                for (int r = 0; r < kRows; r += 4) {
                    if constexpr (kRows >= 4) *reinterpret_cast<float4*>(wj + r) = *reinterpret_cast<const float4*>(weights + j * kRows + r);
                    else wj[r] = weights[j * kRows + r];
                }
#pragma unroll
                for (int r = 0; r < kRows; ++r)  // (what a node does not see may be infinite)
                    if (!TREE || wj[r] != 0.f) add_product(o[r][h], wj[r], v4);
            }
        }
        __syncwarp();
    }
    // use(row, its maximum, its sum, first dimension, up to four numbers of the output), from every lane that has some
    template <typename F>
    __device__ __forceinline__ void results(const Rows& rows, F&& use) {
        const int lane = threadIdx.x & 31, dim = p.map.head_dim;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            float t = l[r];
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
            if (r >= rows.n) continue;
#pragma unroll
            for (int h = 0; h < QUADS; ++h) {
                const float x[4] = {o[r][h].x, o[r][h].y, o[r][h].z, o[r][h].w};
                if (h * 128 + lane * 4 < dim) use(r, m[r], t, h * 128 + lane * 4, x);
            }
        }
    }
    __device__ __forceinline__ void store(const Rows& rows) {
        results(rows, [&](int r, float, float sum, int d, const float (&x)[4]) {
            const float scale = inverse_of<TREE>(p, rows, r, sum);
            T* at = static_cast<T*>(p.o) + row_at<TREE>(p, p.os, rows, r) + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) put(p, at + e, x[e] * scale);
        });
    }
};

// Four codes as fp16 numbers, two to a register: the first and third, the second and fourth.  (int8 as subnormal numbers, a byte with its
// sign bit turned over as it stands: two instructions less, but then 128 too much, and sums that begin at what takes it off wait for the
// weights' own sum: 8 x 40000 tokens of 32 heads on 4 of 128 86 us instead of 80.)
template <typename P>
__device__ __forceinline__ void to_pairs(uint32_t w, uint32_t& even, uint32_t& odd);
template <>
__device__ __forceinline__ void to_pairs<int8_t>(uint32_t w, uint32_t& even, uint32_t& odd) {
    w ^= 0x80808080u;  // 0 .. 255 under the exponent of 1024, less 1024 + 128
    const uint32_t bias = 0x64806480u;
    const auto less = [&](uint32_t x) {
        const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
        return *reinterpret_cast<const uint32_t*>(&d);
    };
    even = less(__byte_perm(w, 0x64646464u, 0x4240));
    odd = less(__byte_perm(w, 0x64646464u, 0x4341));
}
template <>
__device__ __forceinline__ void to_pairs<E4m3>(uint32_t w, uint32_t& even, uint32_t& odd) {
    w = __byte_perm(w, w, 0x3120);
    const __half2 a = from_e4m3(w), b = from_e4m3(w >> 16);
    even = *reinterpret_cast<const uint32_t*>(&a);
    odd = *reinterpret_cast<const uint32_t*>(&b);
}

// ---- the core on tensor cores: 16-bit types, head_dim 16, 32, 64, 80, 96, 128, 192 or 256 -------------------------------------------------
// mma.sync with the keys, then the dimensions of the values, as the sixteen rows of a tile and eight query heads as its columns
// (tcgen05's 64 or 128 rows would wait for as many keys per step, and the step is bound by HBM long before the tensor cores): the
// scores are K Q^T, their exponentials, turned over eight by eight (movmatrix), are the operand of V^T W^T.  A weight goes in as several
// 16-bit numbers that add up to it: three in bf16, all 24 bits; two in fp16, 22 bits, what the exponential itself has.  One alone
// would put up to 2^-8 of itself on the output, two in bf16 2^-16, which shows where values cancel.  In fp16 they are raised by
// 2^12, as far as the largest allows, so that those below 2^-14 of it keep their bits.  The products cut their sums off instead of
// rounding them, so a tile's begin at zero and are added to the outputs by themselves (all in one chain, a warp's 900 tiles brought
// its part 2^-12 nearer to zero), one chain for each sixteen keys (one for all 32: 12.4 us for 700 tokens instead of 10.9).  Up to
// eight heads: the tile's upper eight rows are zeros and have no registers.
template <int DH>
struct MmaLayout {
    int bytes;
    static constexpr bool kTurned = DH / 8 % 4 == 0;
    __host__ __device__ static constexpr int pitch() { return DH * 2 + (kTurned ? 0 : 16); }
    __host__ __device__ static constexpr int chunks() { return DH / 8; }
    // eight rows' same chunk stands on different banks: by its place in the row, or by rows of an odd number of chunks
    __device__ __forceinline__ static int offset(int r, int c) {
        const int turn = !kTurned ? 0 : chunks() % 8 == 0 ? r & 7 : r >> 1 & 3;
        return r * pitch() + ((c ^ turn) << 4);
    }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// the same cut off instead of rounded
template <typename T>
__device__ __forceinline__ uint32_t cut2(float a, float b);
template <>
__device__ __forceinline__ uint32_t cut2<__nv_bfloat16>(float a, float b) {
    uint32_t w;
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}
template <>
__device__ __forceinline__ uint32_t cut2<__half>(float a, float b) {
    uint32_t w;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// Two weights as so many 16-bit numbers each: a weight cut off, what that lacks, cut off too but for the last one.  Of a weight that
// is not zero none is below the smallest number that a product takes (2^-126; 2^-24 under the raise, 2^-36 of the largest weight), so
// that all of them take an infinite value to the same infinity; of one that is zero all are.
constexpr int kMostTerms = 3;
template <typename T>
constexpr int kTerms = std::is_same<T, __half>::value ? 2 : 3;
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t (&terms)[kMostTerms]);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float a, float b, uint32_t (&terms)[kMostTerms]) {
    const auto as_pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
    const auto bits = [](__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); };
    terms[0] = cut2<__nv_bfloat16>(a, b);
    const __nv_bfloat162 least = __hmin2(as_pair(terms[0]), as_pair(0x00800080u));
    const float2 first = unpack2<__nv_bfloat16>(terms[0]);
    a -= first.x, b -= first.y;
    terms[1] = bits(__hmax2(as_pair(cut2<__nv_bfloat16>(a, b)), least));
    const float2 second = unpack2<__nv_bfloat16>(terms[1]);
    terms[2] = bits(__hmax2(as_pair(pack2<__nv_bfloat16>(a - second.x, b - second.y)), least));
}
template <>
__device__ __forceinline__ void split2<__half>(float a, float b, uint32_t (&terms)[kMostTerms]) {
    const auto as_pair = [](uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
    const auto bits = [](__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); };
    // (whether a weight is zero, from its upper sixteen bits: those of a positive number are in order in every format)
    const __half2 least = __hmin2(as_pair(cut2<__nv_bfloat16>(a, b)), as_pair(0x00010001u));
    terms[0] = bits(__hmax2_nan(as_pair(cut2<__half>(a, b)), least));
    const float2 first = unpack2<__half>(terms[0]);
    terms[1] = bits(__hmax2(as_pair(pack2<__half>(a - first.x, b - first.y)), least));
}

// an 8 x 8 matrix of 16-bit numbers, two of a row to a lane, with rows and columns exchanged
__device__ __forceinline__ uint32_t turned(uint32_t w) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
    return r;
}

// EIGHTS: of query heads; lane l has heads l % 4 * 2 and the next one of each eight
template <typename T, int DH, int EIGHTS>
struct MmaCore {
    static constexpr int kRows = kMaxRows, KT = DH > 128 ? 16 : 32;
    static constexpr float kRaise = std::is_same<T, __half>::value ? 12.f : 0.f;
    using Layout = MmaLayout<DH>;
    static constexpr int kItemCost = 1;
    using Load = Loader<T, KT, false, kItemCost, Layout>;
    using Args = PagedAttention;
    const PagedAttention& p;
    uint32_t q[EIGHTS][DH / 16][2];
    float m[EIGHTS][2], l[EIGHTS][2];  // l: of this lane's keys
    float o[EIGHTS][DH / 16][4];       // dimension 16 k + lane / 4 of both heads, 16 k + 8 + lane / 4 of both

    static __host__ __device__ int extra(int) { return 0; }

    __device__ MmaCore(const PagedAttention& p, unsigned char*) : p(p) {}
    __device__ __forceinline__ void load_queries(const Rows& of, int) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            const int r = h * 8 + lane / 4;
            const T* from = static_cast<const T*>(p.q) + row_at<false>(p, p.qs, of, r) + lane % 4 * 2;
#pragma unroll
            for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t w = 0;
                    if (r < of.n) {
                        const T* at = from + k * 16 + i * 8;
                        if (p.q_pairs) w = *reinterpret_cast<const uint32_t*>(at);
                        else w = *reinterpret_cast<const uint16_t*>(at) | (uint32_t)*reinterpret_cast<const uint16_t*>(at + 1) << 16;
                    }
                    q[h][k][i] = w;
                }
        }
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            m[h][0] = m[h][1] = -CUDART_INF_F;
            l[h][0] = l[h][1] = 0.f;
#pragma unroll
            for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[h][k][i] = 0.f;
        }
    }
    __device__ __forceinline__ void tile(const Ring& ring, int stage, uint2 marks, const Layout& lay) {
        const unsigned char* tile = ring.tiles + stage * 2 * KT * lay.pitch();
        const int lane = threadIdx.x & 31;
        const uint32_t keys = (uint32_t)__cvta_generic_to_shared(tile), values = keys + KT * Layout::pitch();
        float s[EIGHTS][KT / 16][4];  // of each sixteen: keys lane / 4 and 8 + lane / 4, both heads each
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[h][g][i] = 0.f;
#pragma unroll
        for (int k = 0; k < DH / 16; ++k)
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) {
                uint32_t a[4];
                ldmatrix4(a, keys + lay.offset(g * 16 + (lane & 15), k * 2 + (lane >> 4)));
#pragma unroll
                for (int h = 0; h < EIGHTS; ++h) mma_16816<T>(s[h][g], a[0], a[1], a[2], a[3], q[h][k][0], q[h][k][1]);
            }
        uint32_t weights[EIGHTS][KT / 16][2][kMostTerms];
        float keep[EIGHTS][2];
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            float base[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = -CUDART_INF_F;
#pragma unroll
                for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = g * 16 + i * 8 + lane / 4;
                        float& x = s[h][g][i * 2 + e];
                        x *= p.scale;
                        if (marks.x != 0xffffffffu >> (32 - KT) || marks.y != 0)
                            x = marks.y >> key & 1 ? CUDART_NAN_F : marks.x >> key & 1 ? x : -CUDART_INF_F;
                        top = fmaxf(top, x);
                    }
#pragma unroll
                for (int d = 4; d < 32; d *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float now = fmaxf(m[h][e], top);
                base[e] = now == -CUDART_INF_F ? 0.f : now;
                keep[h][e] = m[h][e] == -CUDART_INF_F ? 1.f : ex2_ftz(m[h][e] - base[e]);  // (nothing to keep, or NaN)
                m[h][e] = now;
                l[h][e] *= keep[h][e];
            }
#pragma unroll
            for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float w[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[e] = ex2_ftz(s[h][g][i * 2 + e] - base[e] + kRaise);
                        l[h][e] += w[e];
                    }
                    split2<T>(w[0], w[1], weights[h][g][i]);
#pragma unroll
                    for (int t = 0; t < kTerms<T>; ++t) weights[h][g][i][t] = turned(weights[h][g][i][t]);
                }
        }
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
            float sum[KT / 16][EIGHTS][4];  // of this tile
            uint32_t a[KT / 16][4];
#pragma unroll
            for (int g = 0; g < KT / 16; ++g) {
                ldmatrix4_trans(a[g], values + lay.offset(g * 16 + (lane >> 4) * 8 + (lane & 7), k * 2 + (lane >> 3 & 1)));
#pragma unroll
                for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[g][h][i] = 0.f;
            }
#pragma unroll
            for (int t = 0; t < kTerms<T>; ++t)
#pragma unroll
                for (int g = 0; g < KT / 16; ++g)
#pragma unroll
                    for (int h = 0; h < EIGHTS; ++h)
                        mma_16816<T>(sum[g][h], a[g][0], a[g][1], a[g][2], a[g][3], weights[h][g][0][t], weights[h][g][1][t]);
#pragma unroll
            for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = sum[0][h][i];
#pragma unroll
                    for (int g = 1; g < KT / 16; ++g) x += sum[g][h][i];
                    o[h][k][i] = fmaf(o[h][k][i], keep[h][i & 1], x);
                }
        }
    }
    template <typename F>
    __device__ __forceinline__ void results(const Rows& rows, F&& use) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = h * 8 + lane % 4 * 2 + e;
                float t = l[h][e];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) t += __shfl_xor_sync(0xffffffffu, t, d);
                if (r >= rows.n) continue;
#pragma unroll
                for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float x[1] = {o[h][k][i * 2 + e]};
                        use(r, m[h][e], t, k * 16 + i * 8 + lane / 4, x);
                    }
            }
    }
    // rounded, and turned over eight by eight so that a lane has two neighbouring dimensions of one head
    __device__ __forceinline__ void store(const Rows& rows) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < EIGHTS; ++h) {
            float scale[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float t = l[h][e];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) t += __shfl_xor_sync(0xffffffffu, t, d);
                scale[e] = inverse(t);
            }
            const int r = h * 8 + lane / 4;
            T* at = static_cast<T*>(p.o) + row_at<false>(p, p.os, rows, r) + lane % 4 * 2;
#pragma unroll
            for (int k = 0; k < DH / 16; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t w = turned(pack2<T>(o[h][k][i * 2] * scale[0], o[h][k][i * 2 + 1] * scale[1]));
                    if (r >= rows.n) continue;
                    if (p.o_pairs) {
                        *reinterpret_cast<uint32_t*>(at + k * 16 + i * 8) = w;
                    } else {
                        reinterpret_cast<uint16_t*>(at)[k * 16 + i * 8] = (uint16_t)w;
                        reinterpret_cast<uint16_t*>(at)[k * 16 + i * 8 + 1] = (uint16_t)(w >> 16);
                    }
                }
        }
    }
};

// ---- the line of tiles ------------------------------------------------------------------------------------------------------

// weight of a part whose maximum is m under the common one (base: that, or 0 where it is -inf): a part of hidden scores alone
// holds zeros, or NaN that has to stay
__device__ __forceinline__ float part_weight(float m, float base) { return m == -CUDART_INF_F ? 1.f : exp2f(m - base); }

// A warp's part of an item that was cut: of the one that its piece begins in (0), of the one that begins in it (1).
struct Part {
    int there;
    Rows rows;
    int item, starts, ends;
    long long item_end;
};

template <typename T, typename P, bool TREE, typename Core, int W, int S>  // up to W warps
__global__ void __launch_bounds__(W * 32) paged_attention_kernel(const __grid_constant__ typename Core::Args p) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    constexpr int KT = Core::KT, COST = Core::kItemCost;
    constexpr bool kBulk = Core::Load::kBulk;
    __shared__ alignas(8) uint64_t arrived[W][kBulk ? S : 1];
    __shared__ int given_up;
    // (what TMA writes turns its chunks by the address: tiles on 1024 bytes)
    unsigned char* smem = kBulk ? dynamic + (1024 - (uint32_t)__cvta_generic_to_shared(dynamic)) % 1024 : dynamic;
    __shared__ uint2 marks[W][S];
    __shared__ int places[W][TREE ? S : 1];
    __shared__ Part parts[2 * W];
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x / 32, dim = p.map.head_dim;
    const typename Core::Layout lay{p.row_bytes};
    const int tile_bytes = S * 2 * KT * lay.pitch(), ring_bytes = tile_bytes + (kScaled<P> ? S * 2 * KT * (int)sizeof(float) : 0);
    const int extra = Core::extra(dim);
    // a warp's tiles and scales; or the tiles of all of them, then all scales
    const int step = kBulk ? tile_bytes : ring_bytes + extra;
    unsigned char* mine = smem + warp * step;
    unsigned char* scales = kBulk ? smem + warps * tile_bytes + warp * (ring_bytes - tile_bytes) : mine + tile_bytes;
    const Ring ring{mine, marks[warp], places[warp], reinterpret_cast<float*>(scales), (uint32_t)__cvta_generic_to_shared(arrived[warp])};
    float2* part_sums = reinterpret_cast<float2*>(smem + warps * (ring_bytes + extra));  // [2 * warps][rows]
    // a warp's first part [rows][head_dim] goes through memory; its second one, made when all its tiles are done, where they were
    auto part_out = [&](int w, int which) {
        return which == 0 ? p.firsts + (blockIdx.x * warps + w) * (long long)p.rows * dim
                          : reinterpret_cast<float*>(smem + w * step);
    };

    if (tid == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (lane < 2) parts[2 * warp + lane].there = 0;
    if constexpr (kBulk) {
        if (tid == 0) given_up = 0;
        if (lane < S) ptx::mbar_init(ring.arrived + lane * 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        ptx::fence_proxy_async_smem();
        __syncthreads();
    }
    __syncwarp();

    Cursor<KT, TREE, COST> at;
    const Share share = find_share<KT, TREE, COST>(p, at, warp, warps);
    if (share.first < share.end) {
        typename Core::Load ahead{p, ring, lay, at};  // of the tile to load next, unit `load` of the line
        long long load = share.first;
        int stage_in = 0, stage_out = 0;
        uint32_t phase = 0;  // a bit for each stage
        auto look = [&]() {
            if (load < share.end && ahead.at.t < COST) {
                load += COST - ahead.at.t;
                ahead.at.t = COST;
            }
            if (load < share.end) ahead.look();
        };
        auto fetch = [&]() {
            if (load < share.end) {
                ahead.issue(stage_in);
                if (++load < share.end && ++ahead.at.t == ahead.at.n) {
                    ahead.at.next_item(p);
                    if constexpr (kBulk) ahead.planned = 1 << 30;
                }
                look();
            }
            if constexpr (!kBulk) asm volatile("cp.async.commit_group;" ::: "memory");
            stage_in = stage_in + 1 == S ? 0 : stage_in + 1;
        };
        look();
#pragma unroll
        for (int s = 0; s < S - 1; ++s) fetch();

        Core core(p, mine + ring_bytes);
        auto queries = [&](const Cursor<KT, TREE, COST>& c) {
            const Rows rows = rows_of<TREE>(p, c.b, c.head, c.item - c.head * c.parts(p), c.count);
            core.load_queries(rows, c.count);
            return rows;
        };
        long long begin = share.first;
        bool bad_page = false;
        Rows rows = queries(at);
        while (begin < share.end) {
            const long long item_end = begin + (at.n - at.t), end = item_end < share.end ? item_end : share.end;
            const int tiles = (int)(end - begin) - max(COST - at.t, 0);
            core.reset();
            for (int i = 0; i < tiles; ++i) {
                if constexpr (!kBulk) asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
                if constexpr (kBulk) {
                    ptx::mbar_wait(ring.arrived + stage_out * 8, phase >> stage_out & 1, &given_up, p.status);
                    phase ^= 1u << stage_out;
                }
                __syncwarp();
                fetch();
                const uint2 mark = ring.marks[stage_out];
                bad_page |= mark.y != 0;
                core.tile(ring, stage_out, mark, lay);
                stage_out = stage_out + 1 == S ? 0 : stage_out + 1;
            }
            const Cursor<KT, TREE, COST> done = at;
            const Rows done_rows = rows;
            if (item_end < share.end) {  // the next item's queries load while this one's results are stored
                at.next_item(p);
                rows = queries(at);
            }
            begin = end;
            if (tiles <= 0) continue;
            const bool starts = done.t <= COST, ends = end == item_end;
            if (starts && ends) {
                core.store(done_rows);
            } else {
                const int which = starts ? 1 : 0;
                __syncwarp();
                float* to = part_out(warp, which);
                float2* sums = part_sums + (2 * warp + which) * p.rows;
                core.results(done_rows, [&](int r, float top, float sum, int d, const auto& x) {
                    constexpr int N = sizeof(x) / sizeof(float);
                    if (d == 0) sums[r] = make_float2(top, sum);
#pragma unroll
                    for (int e = 0; e < N; ++e) to[r * dim + d + e] = x[e];
                });
                if (lane == 0) parts[2 * warp + which] = {1, done_rows, done.item, starts, ends, item_end};
            }
        }
        if (bad_page && lane == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
    }
    __syncthreads();

    // The CTA's parts of one item are neighbours: one that begins here, or that the CTA begins in, and those that go on with it.
    // Each item's numbers, four to a thread, begin with the thread behind the last one's.
    const uint32_t there = __ballot_sync(0xffffffffu, lane < 2 * warps && parts[lane].there);
    int turn = 0;
    for (uint32_t todo = there & (0xaaaaaaaau | 1u); todo != 0; todo &= todo - 1) {
        const int i = __ffs(todo) - 1;
        const uint32_t rest = todo & (todo - 1), members = there & ~((1u << i) - 1) & (rest != 0 ? (rest & (0u - rest)) - 1 : 0xffffffffu);
        const Part part = parts[i];
        const bool starts = part.starts, ends = parts[31 - __clz(members)].ends;
        const Rows rows = part.rows;
        const long long slot = (blockIdx.x * 2 + (starts ? 1 : 0)) * (long long)p.rows;
        const int units = rows.n * dim / 4;
        int x = tid - turn;
        if (x < 0) x += blockDim.x;
        for (; x < units; x += blockDim.x) {
            const int r = x * 4 / dim;
            float m = -CUDART_INF_F, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t j = members; j != 0; j &= j - 1) m = fmaxf(m, part_sums[(__ffs(j) - 1) * p.rows + r].x);
            const float base = m == -CUDART_INF_F ? 0.f : m;
#pragma unroll 4
            for (uint32_t j = members; j != 0; j &= j - 1) {
                const int at = __ffs(j) - 1;
                const float2 sum = part_sums[at * p.rows + r];
                const float w = part_weight(sum.x, base);
                l = fmaf(w, sum.y, l);
                add_product(o, w, reinterpret_cast<const float4*>(part_out(at >> 1, at & 1))[x]);
            }
            if (starts && ends) {
                T* to = static_cast<T*>(p.o) + row_at<TREE>(p, p.os, rows, r) + (x * 4 - r * dim);
                const float scale = inverse_of<TREE>(p, rows, r, l);
                put(p, to + 0, o.x * scale);
                put(p, to + 1, o.y * scale);
                put(p, to + 2, o.z * scale);
                put(p, to + 3, o.w * scale);
            } else {
                reinterpret_cast<float4*>(p.partial + slot * dim)[x] = o;
                if (x * 4 == r * dim) p.sums[slot + r] = make_float2(m, l);
            }
        }
        turn = (turn + units) % blockDim.x;
        if (starts && !ends && tid == 0)
            p.joins[blockIdx.x] = make_int4(rows.b, part.item, (int)((part.item_end - 1) / (share.per * share.warps)), 0);
    }

    // sequences without a key to see, or without a place
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        int lo, pos, count;
        bool bad;
        if (tiles_of<KT, TREE>(p, b, lo, pos, count, bad) > 0) continue;
        if (bad && tid == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        const int heads = p.group * p.map.kv_heads;
        if (TREE && !bad) continue;  // no nodes
        const int n = TREE ? (count < 0 || count > p.nodes ? p.nodes : count) : 1;
        for (int i = tid; i < n * heads * dim; i += blockDim.x) {
            const int d = i % dim, row = i / dim, node = TREE ? row / heads : 0, h = row - node * heads;
            T* to = static_cast<T*>(p.o) + b * p.os[0] + h * p.os[1] + d;
            if (TREE) to += node * p.os[2];
            put(p, to, bad ? CUDART_NAN_F : 0.f);
        }
    }
}

// The parts of an item that was cut: CTA (c, .) joins 128 dimensions of a row of the one that begins in CTA c.  Its warps take every
// kJoinWarps-th part each, a lane four dimensions, kJoinAhead parts on their way at once.  The first two parts, mostly all there are,
// load before it is known whether there is an item (one sequence of 65536 tokens in 148 parts: 20.7 us the two kernels, with one part
// at a time 22.7; 700 tokens: 10.9, 12.4).
constexpr int kJoinWarps = 8, kJoinAhead = 6;
template <typename T, bool TREE>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_join_kernel(const __grid_constant__ PagedAttention p) {
    __shared__ float2 warp_sums[kJoinWarps];
    __shared__ float4 outs[kJoinWarps][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dim = p.map.head_dim;
    const int r = blockIdx.y % p.rows, d = blockIdx.y / p.rows * 128 + lane * 4;
    auto slot = [&](int i) { return (2LL * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * p.rows + r; };
    float2 ml[kJoinAhead];
    float4 part[kJoinAhead];
    auto load = [&](int i, float2& sums, float4& out) {
        sums = __ldcg(p.sums + slot(i));
        if (d < dim) out = __ldcg(reinterpret_cast<const float4*>(p.partial + slot(i) * dim + d));
    };
    pdl_wait();
    const int4 join = __ldcg(p.joins + blockIdx.x);
    if (warp < 2) load(warp, ml[0], part[0]);  // (there is a CTA behind this one: never past the scratch memory)
    if (join.x < 0) return;
    const int count = TREE ? (p.counts != nullptr ? __ldg(p.counts + join.x) : p.nodes) : 1, parts = parts_of<TREE>(p, count);
    const Rows rows = rows_of<TREE>(p, join.x, join.y / parts, join.y % parts, count);
    if (r >= rows.n) return;
    const int n = join.z - (int)blockIdx.x + 1;
    float m = -CUDART_INF_F, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = warp; i0 < n; i0 += kJoinWarps * kJoinAhead) {
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            const int i = i0 + j * kJoinWarps;
            if (i >= 2 && i < n) load(i, ml[j], part[j]);
        }
#pragma unroll
        for (int j = 0; j < kJoinAhead; ++j) {
            if (i0 + j * kJoinWarps >= n) break;
            const float now = fmaxf(m, ml[j].x), base = now == -CUDART_INF_F ? 0.f : now, keep = part_weight(m, base),
                        w = part_weight(ml[j].x, base);
            m = now;
            l = fmaf(w, ml[j].y, l * keep);
            o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
            if (d < dim) add_product(o, w, part[j]);
        }
    }
    if (lane == 0) warp_sums[warp] = make_float2(m, l);
    outs[warp][lane] = o;
    __syncthreads();
    if (warp != 0 || d >= dim) return;
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) m = fmaxf(m, warp_sums[w].x);
    const float base = m == -CUDART_INF_F ? 0.f : m;
    float sum = 0.f;
    float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) {
        const float x = part_weight(warp_sums[w].x, base);
        sum = fmaf(x, warp_sums[w].y, sum);
        add_product(out, x, outs[w][lane]);
    }
    const float scale = inverse_of<TREE>(p, rows, r, sum);
    T* to = static_cast<T*>(p.o) + row_at<TREE>(p, p.os, rows, r) + d;
    put(p, to + 0, out.x * scale);
    put(p, to + 1, out.y * scale);
    put(p, to + 2, out.z * scale);
    put(p, to + 3, out.w * scale);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

// Shared memory of a CTA, one to an SM: with much more, what is left of the SM's memory as L1 is too little for the copies on their
// way, and they come from L2 twice (32 heads on 4, 553,000 tokens, rings of three tiles in 226 KB: 231 us when this took 189).  Head
// size 64 has eleven warps here; with twelve its 256 windows of 512 take the same 68.5 us.
constexpr int kMostShared = 193 * 1024 + 512;
// What TMA brings does not go through L1.
constexpr int kMostSharedBulk = 216 * 1024;

// Keys and values as TMA's swizzles leave their rows: boxes of 128, 64 or 32 bytes, one behind the other for all 32 rows, the sixteen-byte
// chunks of a row turned so that eight rows' same chunk stands on different banks.
template <int ROWB>
struct BoxLayout {
    int bytes;
    static constexpr int kBoxBytes = ROWB % 128 == 0 ? 128 : ROWB % 64 == 0 ? 64 : 32, kBoxes = ROWB / kBoxBytes, kInBox = kBoxBytes / 16;
    __host__ __device__ static constexpr int pitch() { return ROWB; }
    __host__ __device__ static constexpr int chunks() { return ROWB / 16; }
    __device__ __forceinline__ static int turn(int r) { return kInBox == 8 ? r & 7 : kInBox == 4 ? r >> 1 & 3 : r >> 2 & 1; }
    __device__ __forceinline__ static int offset(int r, int c) {
        return c / kInBox * 32 * kBoxBytes + r * kBoxBytes + ((c % kInBox ^ turn(r)) << 4);
    }
};

// the maps of what TMA reads, rows of pairs of bytes; none of what does not exist
template <typename Layout>
bool make_maps(const tmw_paged_attention_desc& d, PagedAttentionBulk& p) {
    const CUtensorMapSwizzle turns = Layout::kBoxBytes == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                     : Layout::kBoxBytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                               : CU_TENSOR_MAP_SWIZZLE_32B;
    const auto make = [&](CUtensorMap* map, const void* base, int rows) {
        return rows == 0 || make_map_2d(map, base, TMW_F16, rows, Layout::pitch() / 2, Layout::pitch() / 2, p.run, Layout::kBoxBytes / 2, turns);
    };
    const int rows = d.at.pages * d.at.kv_heads * d.at.page_size, pers = d.at.kv_heads * d.n_persistent;
    return make(&p.k_map, d.at.k_pages, rows) && make(&p.v_map, d.at.v_pages, rows) && make(&p.k_pers_map, d.k_pers, pers) &&
           make(&p.v_pers_map, d.v_pers, pers);
}
// whether pages can come by TMA: runs of eight neighbours at least, rows numbered in 32 bits, scales that begin on sixteen bytes
inline bool can_bulk(const tmw_paged_attention_desc& d, const tmw_page_scales& s) {
    return d.at.page_size % 8 == 0 && (reinterpret_cast<uintptr_t>(s.k_scales) | reinterpret_cast<uintptr_t>(s.v_scales)) % 16 == 0 &&
           (long long)d.at.pages * d.at.kv_heads * d.at.page_size <= 0x7fffffffLL - 32 &&
           (long long)d.at.kv_heads * d.n_persistent <= 0x7fffffffLL - 32;
}

struct Plan {
    int rows, parts, warps, grid, smem;
    size_t sums_at, partial_at, firsts_at, bytes;
};

template <typename T, typename P, bool TREE, typename Core, int W, int S>
struct Kernel {
    using CoreOf = Core;
    static constexpr int KT = Core::KT;
    // nodes: drafted ones of a sequence, 1 without
    static Plan plan(const tmw_paged_attention_desc& d, int row_bytes, int nodes) {
        Plan n;
        const int group = d.heads / d.at.kv_heads * nodes;
        n.parts = (group + Core::kRows - 1) / Core::kRows;
        n.rows = (group + n.parts - 1) / n.parts;
        const int tile = S * 2 * KT * (typename Core::Layout{row_bytes}.pitch() + (kScaled<P> ? (int)sizeof(float) : 0));
        const int warp = tile + Core::extra(d.at.head_dim) + 2 * n.rows * (int)sizeof(float2);
        constexpr int most = Core::Load::kBulk ? kMostSharedBulk - 1024 : kMostShared;
        n.warps = most / warp < W ? most / warp : W;
        n.smem = n.warps * warp + (Core::Load::kBulk ? 1024 : 0);
        // no more CTAs than the longest sequences could have work for
        const long long capacity = (long long)d.at.columns * d.at.page_size;
        const long long keys = d.window >= 0 && d.window + (long long)nodes < capacity ? d.window + (long long)nodes : capacity;
        const long long tiles = ((d.n_persistent + KT - 1) / KT + keys / KT + 2) * (long long)d.at.kv_heads * n.parts * d.at.batch;
        n.grid = (int)(tiles < sm_count() ? tiles : sm_count());
        const size_t out = (size_t)n.rows * d.at.head_dim * sizeof(float);
        n.sums_at = (size_t)n.grid * sizeof(int4);
        n.partial_at = (n.sums_at + (size_t)n.grid * 2 * n.rows * sizeof(float2) + 15) & ~(size_t)15;
        n.firsts_at = n.partial_at + n.grid * 2 * out;
        n.bytes = n.firsts_at + (size_t)n.grid * n.warps * out;
        return n;
    }
    static int launch(typename Core::Args& p, const Plan& n, unsigned char* scratch, cudaStream_t stream) {
        p.rows = n.rows;
        p.parts = n.parts;
        p.items = p.map.kv_heads * n.parts;
        p.pers_tiles = (p.np + KT - 1) / KT;
        p.joins = reinterpret_cast<int4*>(scratch);
        p.sums = reinterpret_cast<float2*>(scratch + n.sums_at);
        p.partial = reinterpret_cast<float*>(scratch + n.partial_at);
        p.firsts = reinterpret_cast<float*>(scratch + n.firsts_at);
        auto kern = paged_attention_kernel<T, P, TREE, Core, W, S>;
        const int rc = allow_shared_memory(reinterpret_cast<const void*>(kern), n.smem);
        if (rc != TMW_OK) return rc;
        kern<<<n.grid, n.warps * 32, n.smem, stream>>>(p);
        TMW_CUDA_TRY(cudaGetLastError());
        if (n.grid > 1)
            TMW_CUDA_TRY(launch_ex(paged_join_kernel<T, TREE>, dim3((unsigned)n.grid - 1, (unsigned)(n.rows * ((p.map.head_dim + 127) / 128))),
                                   dim3(kJoinWarps * 32), 0, stream, true, 1, static_cast<const PagedAttention&>(p)));
        return TMW_OK;
    }
};

// as many query heads at once as a group has, up to four, or eight where a lane has four dimensions of each
template <typename T, typename P, bool TREE, typename F>
int with_simt(const tmw_paged_attention_desc& d, int nodes, F&& use) {
    const int group = d.heads / d.at.kv_heads * nodes;
    if (d.at.head_dim > 128) return group == 1 ? use(Kernel<T, P, TREE, SimtCore<T, P, 1, 2, TREE>, 12, 2>()) : use(Kernel<T, P, TREE, SimtCore<T, P, 4, 2, TREE>, 12, 2>());
    if (group == 1) return use(Kernel<T, P, TREE, SimtCore<T, P, 1, 1, TREE>, 12, 2>());
    return group <= 4 ? use(Kernel<T, P, TREE, SimtCore<T, P, 4, 1, TREE>, 12, 2>()) : use(Kernel<T, P, TREE, SimtCore<T, P, 8, 1, TREE>, 12, 2>());
}
inline int validate(const tmw_paged_attention_desc* d, bool& used) {
    if (d == nullptr) return TMW_ERR_INVALID_ARGUMENT;
    if (d->heads < 0 || d->n_persistent < 0 || d->window < -1 || !(d->scale >= 0.f)) return TMW_ERR_INVALID_ARGUMENT;
    used = d->at.batch > 0 && d->heads > 0;
    const int rc = validate_pages(d->at, used);
    if (rc != TMW_OK) return rc;
    if (d->heads % d->at.kv_heads != 0) {
        set_error_text("tmw_paged_attention: heads must be a multiple of kv_heads");
        return TMW_ERR_INVALID_ARGUMENT;
    }
    if (d->heads > 65535 || d->n_persistent > (1 << 24)) return TMW_ERR_TOO_LARGE;
    return TMW_OK;
}

// The kernels' arguments of a description that says there is something to do.
inline int arguments(const tmw_paged_attention_desc& d, const tmw_page_scales& scales, const void* scratch, PagedAttention& p) {
    const size_t size = dtype_size(d.at.dtype);
    if (d.o == d.q) {
        set_error_text("tmw_paged_attention: o must not be q (other CTAs may still read it)");
        return TMW_ERR_INVALID_ARGUMENT;
    }
    if (d.q == nullptr || d.o == nullptr || d.pos == nullptr || scratch == nullptr ||
        (d.n_persistent > 0 && (d.k_pers == nullptr || d.v_pers == nullptr)))
        return TMW_ERR_INVALID_ARGUMENT;
    const int rc = validate_scales(d.at, scales, true, d.n_persistent > 0);
    if (rc != TMW_OK) return rc;
    for (int i = 0; i < 2; ++i)
        if (d.q_stride[i] < 0 || d.o_stride[i] < 0) return TMW_ERR_INVALID_ARGUMENT;
    if (!rows_apart(d.o_stride, {d.at.batch, d.heads})) {
        set_error_text("tmw_paged_attention: every output must have a place of its own");
        return TMW_ERR_INVALID_ARGUMENT;
    }
    const auto bits = [](const void* x) { return reinterpret_cast<uintptr_t>(x); };
    if ((bits(d.k_pers) | bits(d.v_pers) | bits(scratch)) % 16 != 0 || (bits(d.q) | bits(d.o)) % size != 0)
        return TMW_ERR_INVALID_ARGUMENT;

    p = {};
    p.map = PageMap(d.at);
    p.q = d.q; p.o = d.o;
    p.k_pages = d.at.k_pages; p.v_pages = d.at.v_pages;
    p.k_pers = d.k_pers; p.v_pers = d.v_pers;
    p.k_scales = scales.k_scales; p.v_scales = scales.v_scales;
    p.k_pers_scales = scales.k_pers_scales; p.v_pers_scales = scales.v_pers_scales;
    for (int i = 0; i < 2; ++i) {
        p.qs[i] = d.q_stride[i];
        p.os[i] = d.o_stride[i];
    }
    p.pos = d.pos;
    p.batch = d.at.batch; p.np = d.n_persistent; p.window = d.window;
    p.bf16 = d.at.dtype == TMW_BF16;
    p.whole_runs = d.at.page_size % 16 == 0;
    p.run = d.at.page_size % 16 == 0 ? 16 : d.at.page_size % 8 == 0 ? 8 : 0;
    p.group = d.heads / d.at.kv_heads;
    p.scale = (d.scale > 0.f ? d.scale : 1.0f / sqrtf((float)d.at.head_dim)) * 1.4426950408889634f;
    p.row_bytes = d.at.head_dim * (scales.format == 0 ? (int)size : 1);
    p.q_pairs = bits(d.q) % 4 == 0 && (d.q_stride[0] | d.q_stride[1]) % 2 == 0;
    p.o_pairs = bits(d.o) % 4 == 0 && (d.o_stride[0] | d.o_stride[1]) % 2 == 0;
    p.q_wide = bits(d.q) % 16 == 0 && (d.q_stride[0] | d.q_stride[1]) * (long long)size % 16 == 0;
    p.o_wide = bits(d.o) % 16 == 0 && (d.o_stride[0] | d.o_stride[1]) * (long long)size % 16 == 0;
    p.status = device_status_word();
    return p.status == nullptr ? TMW_ERR_CUDA : TMW_OK;
}

}  // namespace
}  // namespace tmw
