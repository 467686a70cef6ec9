// Attention of a tree's drafted tokens, many rows to a key head, over pages of 16-bit numbers or of codes (tcgen05; head_dim 64 or 128).
//
// Up to 128 (node, head) rows of a key head are one tile of tcgen05.mma, so that 64 keys cost the tensor core the same for 33 rows as for
// 128, a fifth of what mma.sync takes for them (9 cycles of a scheduler for each 16 x 8 x 16).  A CTA, one to an SM, is one worker of the
// line of tiles (paged_attention.cuh), here of 64 keys, and its warps have fixed roles:
//   warp  0, 3  bring K, bring V by TMA, a run of up to 64 neighbouring tokens at a time; every lane looks the page of one run up, for
//               4 to 32 tiles in one go (one warp for both, tile by tile, needed 2050 cycles for each: 183 us instead of 149)
//   warp  1, 2  issue the products for the scores, and those with the values (one elected thread each: a product costs its thread some
//               thirty cycles, and a commit hundreds)
//   warps 4-11  softmax, a thread to a row; queries into shared memory, outputs out of tensor memory
// A tile's chain - products, hand-over, exponentials, hand-over, products - is several times as long as its parts, so two streams of
// softmax warps take the tiles by turns, each with a running maximum, a sum and an output of its own, and two buffers of scores: S = Q K^T
// of four tiles is under way while P goes over its S as two 16-bit numbers a weight (64 columns for 64 fp32 ones) and O += P V.
// The streams are joined when the part ends, or has had kTcMost tiles.  (As two CTAs to an SM, with two tiles of each of K and V: 16 ragged sequences of 32 heads on 8, 32 nodes, 160 us.)
// The running maximum follows only a score that is 2^4 above it: O is brought up in tensor memory then.  Tiles that some row does not
// see in full, at a window's begin and among the nodes, have the rows' bits applied to the scores, and their values made harmless: rows
// that nobody sees are zeros, and what is infinite or no number is added row by row to those that see it.
//
// Pages of 8 bits: TMA brings codes, and eight more warps (12-19, four for the keys, four for the values) turn them into fp16 tiles of
// the same form, once for all rows, and every key's scales into the numbers that the softmax warps use (see the attention of one token):
// scores times the key's scale, weights times the value's in two parts.
//
// 16 sequences of up to 16384, 33 nodes, 32 heads on 8 of 128, fp16, 576 MB: 153 us with the join; 118 tiles of 64 keys to a CTA, 2100 cycles
// each, 1410 for their bytes.  6 of up to 65536, 12 nodes, 32 heads on 4 of 128, int8, 307 MB: 218 us; 122 tiles, 3500 cycles each.  Issue slots are
// 38 % busy either way: two softmax warps to a scheduler, each a row's 64 keys in one dependent chain.
//
// All waits are bounded (tc_ptx.cuh); the tensor memory is given back on every way.
#include "paged_tree.cuh"

namespace tmw {
namespace {

using namespace ptx;

// kTcCost: what an item costs besides its tiles (2 | 4 | 6 | 9: the ragged sequences 149 | 135 | 127 | 124 us)
constexpr int kTcKeys = 64, kTcRows = 128, kTcCost = 9;
// Tensor memory's sums are cut off, not rounded: a product of sixteen keys loses 2^-24 of the sum on the average, 400,000 keys of one part 1.5e-3
// of it.  After so many tiles, 512 products in either stream (3e-5), a part's outputs leave tensor memory and are added up with rounding
// (148 sequences of 100,000 tokens that lie in L2, 40 nodes, fp16: 1125 us without, 1183 so; shorter parts the same).
constexpr int kTcMost = 128;
constexpr int kTcAhead = 4;  // tiles whose scores are under way: buffers of scores, and tiles in the ring of keys

template <typename P, int DH>
struct TcLayout {
    static constexpr bool k8 = kScaled<P>;
    // sub-tiles of 64 columns; tiles in the rings
    static constexpr int kSubs = DH / 64, kKStages = k8 ? 2 : kTcAhead, kVStages = k8 ? 4 : DH == 64 ? 12 : 7;
    // (who waits for the values of four tiles ago must not find the barrier a turn further)
    static_assert(kVStages >= kTcAhead, "a phase is asked for before the next but one");
    static constexpr int kQSub = kTcRows * 128, kSub = kTcKeys * 128, kTile = kSub * kSubs;
    static constexpr int kK = kQSub * kSubs, kV = kK + kKStages * kTile;
    // codes: rings of four tiles, with scales of keys and values; then what becomes of the scales, of eight tiles
    static constexpr int kRawTile = kTcKeys * DH, kRawK = kV + kVStages * kTile, kRawV = kRawK + (k8 ? 4 * kRawTile : 0);
    static constexpr int kScales = kRawV + (k8 ? 4 * kRawTile : 0), kParts = kScales + (k8 ? 4 * 2 * kTcKeys * 4 : 0);
    static constexpr int kBytes = kParts + (k8 ? 8 * 2 * kTcKeys * 8 : 0);
    static constexpr int kThreads = k8 ? 640 : 384;
};
// registers of the codes' form: twenty warps have 96 each at launch
constexpr int kRegsService = 56, kRegsSoftmax = 152;
static_assert(32 * (12 * kRegsService + 8 * kRegsSoftmax) <= 640 * 96, "setmaxnreg: what the softmax warps ask for the others release");
// of a tile: its first key's token (-1: persistent ones), its keys that exist, its runs that have no page
struct TileInfo {
    int place, first, last, lost;
};

// A CTA's parts of items, one after the other, as every role walks over them.
struct Walk {
    Cursor<kTcKeys, true, kTcCost> at, now;  // the next part's first unit; the present part's
    long long begin, end, item_end;
    int first_tile, tiles;
    bool starts, ends;
    __device__ __forceinline__ bool next(const PagedAttention& p, long long limit) {
        while (begin < limit) {
            now = at;
            item_end = begin + (at.n - at.t);
            end = item_end < limit ? item_end : limit;
            first_tile = max(at.t - kTcCost, 0);
            tiles = (int)(end - begin) - max(kTcCost - at.t, 0);
            starts = at.t <= kTcCost;
            ends = end == item_end;
            begin = end;
            if (item_end < limit) at.next_item(p);
            if (tiles > 0) return true;
        }
        return false;
    }
};

// sixteen codes as fp16 numbers, in their order
template <typename P>
__device__ __forceinline__ void to_halves(const uint4& codes, uint4 (&out)[2]) {
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<P, E4m3>::value) {
            const __half2 a = from_e4m3(w[i]), b = from_e4m3(w[i] >> 16);
            x[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
            x[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
        } else {  // 0 .. 255 under the exponent of 1024, less 1024 + 128
            const uint32_t u = w[i] ^ 0x80808080u, bias = 0x64806480u;
            const auto less = [&](uint32_t v) {
                const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&bias));
                return *reinterpret_cast<const uint32_t*>(&d);
            };
            x[2 * i] = less(__byte_perm(u, 0x64646464u, 0x4140));
            x[2 * i + 1] = less(__byte_perm(u, 0x64646464u, 0x4342));
        }
    }
    out[0] = make_uint4(x[0], x[1], x[2], x[3]);
    out[1] = make_uint4(x[4], x[5], x[6], x[7]);
}

template <typename P, int DH>
__global__ void __launch_bounds__(TcLayout<P, DH>::kThreads, 1) paged_tree_tc_kernel(const __grid_constant__ PagedAttentionBulk p) {
    using L = TcLayout<P, DH>;
    constexpr bool k8 = L::k8, BF16 = std::is_same<P, __nv_bfloat16>::value;
    constexpr bool kMayBeWild = !std::is_same<P, int8_t>::value;  // infinities and NaN among the values
    using M = std::conditional_t<BF16, __nv_bfloat16, __half>;
    constexpr int KT = kTcKeys, KS = L::kKStages, VS = L::kVStages;
    constexpr float kRaise = BF16 ? 0.f : k8 ? 10.f : 11.f;  // (a weight is at most 2^4, of codes 2^5, times that)
    constexpr uint32_t kO = 4 * KT, kColumns = 512;  // two buffers of scores for each stream, then their outputs
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ alignas(8) uint64_t bars[1 + 3 * kTcAhead + 2 * VS + (k8 ? 24 : 0)];
    __shared__ TileInfo infos[16];  // of the last tiles
    __shared__ float2 stream_sums[2][kTcRows];
    __shared__ uint32_t tmem_slot;
    __shared__ int given_up, wild[2], first_adds[2], lows[8];
    unsigned char* smem = dynamic + (1024 - smem_u32(dynamic)) % 1024;
    const uint32_t base = smem_u32(smem);
    const uint32_t bar0 = smem_u32(bars);
    // Of tile t, counted over all parts: stream t & 1, buffer of scores t & 3, places of its keys t % KS and of its values t % VS (of its codes
    // t & 3); a barrier's phase is the turn's.  Keys are let go with their scores, scores and weights with the products with the values (v_free).
    const uint32_t q_ready = bar0, k_full = bar0 + 8, s_full = k_full + 32, p_ready = s_full + 32, v_full = p_ready + 32, v_free = v_full + 8 * VS;
    const uint32_t raw_k_full = v_free + 8 * VS, raw_k_free = raw_k_full + 32, raw_v_full = raw_k_free + 32, raw_v_free = raw_v_full + 32;  // codes
    const uint32_t parts_full = raw_v_free + 32;  // of tile t, t & 7
    const auto turn = [](int t) { return (uint32_t)(t >> 2) & 1; };
    const auto v_turn = [](int t) { return (uint32_t)(t / VS) & 1; };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        mbar_init(q_ready, 8);
        for (int i = 0; i < kTcAhead; ++i) mbar_init(k_full + 8 * i, k8 ? 4 : 1), mbar_init(s_full + 8 * i, 1), mbar_init(p_ready + 8 * i, 4);
        for (int i = 0; i < VS; ++i) mbar_init(v_full + 8 * i, k8 ? 4 : 1), mbar_init(v_free + 8 * i, 1);
        if (k8)
            for (int i = 0; i < 4; ++i)
                mbar_init(raw_k_full + 8 * i, 1), mbar_init(raw_k_free + 8 * i, 4), mbar_init(raw_v_full + 8 * i, 1), mbar_init(raw_v_free + 8 * i, 4),
                    mbar_init(parts_full + 16 * i, 4), mbar_init(parts_full + 16 * i + 8, 4);
        wild[0] = wild[1] = first_adds[0] = first_adds[1] = 0;
        given_up = 0;
        p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), kColumns);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_trigger();

    Walk walk;
    const Share share = find_share<KT, true, kTcCost>(p, walk.at, 0, 1);
    walk.begin = share.first;
    const long long limit = share.first < share.end ? share.end : share.first;
    if (warp < 4) {
        if constexpr (k8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsService) : "memory");
        if (warp == 0 || warp == 3) {
            // ---- the keys; the values ----
            const bool values = warp == 3;
            const int runs = KT / p.run;
            int t = 0;
            while (walk.next(p, limit)) {
                const auto& at = walk.now;
                int planned = 0, row = -1, page = -1;  // the first tile of the plan; this lane's run: -1 not wanted, -2 nowhere
                uint32_t there = 0, lost = 0;          // lanes
                auto look = [&](int tile) {
                    planned = tile;
                    tile += lane / runs;
                    const bool pers = tile < p.pers_tiles;
                    const int j = (pers ? tile : at.lo / KT + tile - p.pers_tiles) * KT + lane % runs * p.run;
                    row = -1;
                    if (tile < at.n - kTcCost && j <= (pers ? p.np - 1 : at.pos) && j + p.run > (pers ? 0 : at.lo)) {
                        row = j;
                        if (!pers) {
                            const uint32_t column = p.map.page.div((uint32_t)j);
                            row -= (int)(column * p.map.page.d);
                            page = __ldg(p.map.table + at.b * p.map.table_stride + column);
                        }
                    }
                };
                look(walk.first_tile);
                for (int i = 0; i < walk.tiles; ++i, ++t) {
                    const int tile = walk.first_tile + i;
                    if (tile == planned) {  // the pages have come
                        if (row >= 0) {
                            if (tile + lane / runs < p.pers_tiles) row += at.head * p.np;
                            else row = (uint32_t)page < (uint32_t)p.map.pages ? (page * p.map.kv_heads + at.head) * (int)p.map.page.d + row : -2;
                        }
                        there = __ballot_sync(0xffffffffu, row >= 0);
                        lost = __ballot_sync(0xffffffffu, row == -2);
                    }
                    const bool pers = tile < p.pers_tiles;
                    const int from = (tile - planned) * runs, mask = (1 << runs) - 1;
                    const int slot = values && !k8 ? t % VS : t & 3;
                    uint32_t full, to;
                    if constexpr (k8) {
                        full = (values ? raw_v_full : raw_k_full) + 8 * slot;
                        to = base + (values ? L::kRawV : L::kRawK) + slot * L::kRawTile;
                        if (t >= 4) mbar_wait((values ? raw_v_free : raw_k_free) + 8 * slot, turn(t - 4), &given_up, p.status);
                    } else {
                        full = values ? v_full + 8 * slot : k_full + 8 * slot;
                        to = base + (values ? L::kV : L::kK) + slot * L::kTile;  // (KS is four here)
                        if (values) {
                            if (t >= VS) mbar_wait(v_free + 8 * slot, v_turn(t - VS), &given_up, p.status);
                        } else if (t >= kTcAhead) {
                            mbar_wait(s_full + 8 * slot, turn(t - kTcAhead), &given_up, p.status);
                        }
                    }
                    const CUtensorMap* map = values ? (pers ? &p.v_pers_map : &p.v_map) : (pers ? &p.k_pers_map : &p.k_map);
                    const bool with_scales = k8 && !values;
                    float* scales = reinterpret_cast<float*>(smem + L::kScales) + slot * 2 * KT;
                    if (with_scales && pers) {  // (they need not begin on sixteen bytes)
                        const int j0 = tile * KT;
#pragma unroll
                        for (int h = 0; h < KT; h += 32) {
                            const bool mine = j0 + h + lane < p.np;
                            scales[h + lane] = mine ? __ldg(p.k_pers_scales + at.head * p.np + j0 + h + lane) : 0.f;
                            scales[KT + h + lane] = mine ? __ldg(p.v_pers_scales + at.head * p.np + j0 + h + lane) : 0.f;
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    const int scale_bytes = with_scales && !pers ? p.run * 4 : 0;
                    if (elect_one()) {
                        if (values) {
                            const int j0 = (pers ? tile : at.lo / KT + tile - p.pers_tiles) * KT;
                            infos[t & 15] = {pers ? -1 : j0, pers ? 0 : max(at.lo - j0, 0), min((pers ? p.np - 1 : at.pos) - j0, KT - 1), (int)(lost >> from) & mask};
                        }
                        mbar_expect_tx(full, __popc(there >> from & mask) * (p.run * DH * (int)sizeof(P) + 2 * scale_bytes));
                    }
                    __syncwarp();
                    for (uint32_t todo = there >> from & mask; todo != 0; todo &= todo - 1) {
                        const int r = __ffs(todo) - 1, first = __shfl_sync(0xffffffffu, row, from + r);
                        if (elect_one()) {
                            if constexpr (k8) {
                                tma_load_2d(to + r * p.run * DH, map, full, 0, first);
                                if (scale_bytes != 0) {
                                    bulk_load(smem_u32(scales) + r * scale_bytes, p.k_scales + first, scale_bytes, full);
                                    bulk_load(smem_u32(scales + KT) + r * scale_bytes, p.v_scales + first, scale_bytes, full);
                                }
                            } else {
#pragma unroll
                                for (int s = 0; s < L::kSubs; ++s) tma_load_2d(to + s * L::kSub + r * p.run * 128, map, full, s * 64, first);
                            }
                        }
                    }
                    if (values && (lost >> from & mask) != 0 && lane == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
                    if (from + runs == 32 && i + 1 < walk.tiles) look(tile + 1);
                }
            }
        } else if (warp == 1 && elect_one()) {
            // ---- the scores ----
            constexpr uint32_t fmt = BF16 ? 1u : 0u, idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((KT >> 3) << 17) | ((kTcRows >> 4) << 24);
            int t = 0;
            uint32_t q_phase = 0;
            while (walk.next(p, limit)) {
                mbar_wait(q_ready, q_phase, &given_up, p.status);
                q_phase ^= 1;
                for (int i = 0; i < walk.tiles; ++i, ++t) {
                    mbar_wait(k_full + 8 * (t & 3), turn(t), &given_up, p.status);
                    if (t >= kTcAhead) mbar_wait(v_free + 8 * ((t - kTcAhead) % VS), v_turn(t - kTcAhead), &given_up, p.status);
                    tc_fence_after();
                    const uint64_t q = kmajor_desc(base), keys = kmajor_desc(base + L::kK + t % KS * L::kTile);
#pragma unroll
                    for (int k = 0; k < DH / 16; ++k)
                        mma_ss(tmem + (t & 3) * KT, q + k / 4 * (L::kQSub >> 4) + k % 4 * 2, keys + k / 4 * (L::kSub >> 4) + k % 4 * 2, idesc, k > 0 ? 1u : 0u);
                    tc_commit(s_full + 8 * (t & 3));
                }
            }
        } else if (warp == 2 && elect_one()) {
            // ---- the products with the values ----
            const uint32_t idesc = idesc_b_mnmajor(BF16 ? 1u : 0u, DH);
            int t = 0;
            while (walk.next(p, limit)) {
                for (int i = 0; i < walk.tiles; ++i, ++t) {
                    const int v = t % VS;
                    mbar_wait(v_full + 8 * v, v_turn(t), &given_up, p.status);
                    mbar_wait(p_ready + 8 * (t & 3), turn(t), &given_up, p.status);
                    tc_fence_after();
                    const uint32_t weights = tmem + (t & 3) * KT, to = tmem + kO + (t & 1) * DH;
                    const uint64_t values = mnmajor_desc(base + L::kV + v * L::kTile, L::kSub);
                    const uint32_t onto = i % kTcMost > 1 || *(volatile int*)&first_adds[t & 1] ? 1u : 0u;  // (else it begins its stream's O)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int k = 0; k < KT / 16; ++k)
                            mma_ts(to, weights + half * 32 + k * 8, values + k * 128, idesc, half + k > 0 ? 1u : onto);
                    tc_commit(v_free + 8 * v);
                }
            }
        }
    } else if (k8 && warp >= 12) {
        if constexpr (k8) {
            // ---- codes into fp16 tiles: four warps the keys, with the scales of both, four warps the values ----
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsService) : "memory");
            const int mine = tid & 127;
            auto convert = [&](const unsigned char* from, uint32_t to, uint64_t exists) {
                constexpr int kPieces = KT * DH / 16 / 128, kOfRow = DH / 16;
                uint4 codes[kPieces];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) codes[i] = reinterpret_cast<const uint4*>(from)[i * 128 + mine];
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    const int row = (i * 128 + mine) / kOfRow, c = (i * 128 + mine) % kOfRow * 2;
                    uint4 x[2];
                    to_halves<P>(codes[i], x);
                    if ((exists >> row & 1) == 0) x[0] = x[1] = make_uint4(0, 0, 0, 0);  // (may be no number)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<uint4*>(smem + to + c / 8 * L::kSub + row * 128 + (((c + h) % 8 ^ (row & 7)) << 4)) = x[h];
                }
                fence_proxy_async_smem();
                __syncwarp();
            };
            int t = 0;
            while (walk.next(p, limit)) {
                for (int i = 0; i < walk.tiles; ++i, ++t) {
                    if (warp < 16) {
                        mbar_wait(raw_k_full + 8 * (t & 3), turn(t), &given_up, p.status);
                        if (t >= KS) mbar_wait(s_full + 8 * ((t - KS) & 3), turn(t - KS), &given_up, p.status);
                        convert(smem + L::kRawK + (t & 3) * L::kRawTile, L::kK + t % KS * L::kTile, ~0ull);
                        if (lane == 0) mbar_arrive(k_full + 8 * (t & 3));
                        const float* scales = reinterpret_cast<const float*>(smem + L::kScales) + (t & 3) * 2 * KT;
                        const float vs = scales[KT + (mine & 63)];
                        const int bits = __float_as_int(fmaxf(vs, 0x1p-100f));
                        // of two keys: their own scales and the exponents of their values', then what the exponents leave and their inverses
                        float* parts = reinterpret_cast<float*>(smem + L::kParts) + (t & 7) * 4 * KT + (mine & 63) / 2 * 4 + (mine & 1);
                        if (mine < KT) {
                            parts[0] = scales[mine];
                            parts[2] = __int_as_float(0x4b000000 | (bits >> 23)) - (8388608.f + 127.f) + (vs - vs);
                        } else {
                            parts[2 * KT] = __int_as_float((bits & 0x007fffff) | 0x3f800000);
                            parts[2 * KT + 2] = __int_as_float(0x7f000000 - min(bits & 0x7f800000, 0x7e800000));
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(parts_full + 8 * (t & 7)), mbar_arrive(raw_k_free + 8 * (t & 3));
                    } else {
                        const int slot = t % VS;
                        mbar_wait(raw_v_full + 8 * (t & 3), turn(t), &given_up, p.status);
                        if (t >= VS) mbar_wait(v_free + 8 * slot, v_turn(t - VS), &given_up, p.status);
                        const TileInfo& info = infos[t & 15];
                        uint64_t exists = ~0ull >> (63 - info.last) & ~0ull << info.first;
                        for (uint32_t todo = info.lost; todo != 0; todo &= todo - 1)
                            exists &= ~((p.run == 64 ? ~0ull : (1ull << p.run) - 1) << (__ffs(todo) - 1) * p.run);
                        convert(smem + L::kRawV + (t & 3) * L::kRawTile, L::kV + slot * L::kTile, exists);
                        if (lane == 0) mbar_arrive(v_full + 8 * slot), mbar_arrive(raw_v_free + 8 * (t & 3));
                    }
                }
            }
        }
    } else {
        // ---- softmax: a thread to a row ----
        if constexpr (k8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax) : "memory");
        const int g = (warp - 4) >> 2, row = tid & 127;
        const uint32_t lane_at = (uint32_t)((warp & 3) * 32) << 16, o_at = tmem + lane_at + kO + g * DH;
        int t0 = 0;  // the part's first tile
        while (walk.next(p, limit)) {
            const auto& at = walk.now;
            const Rows rows = rows_of<true>(p, at.b, at.head, at.item - at.head * at.parts(p), at.count);
            const int start = __ldg(p.pos + at.b);
            const bool there = row < rows.n, warp_there = (warp & 3) * 32 < rows.n;
            int low = 0;
            uint64_t nodes = 0;
            float q_scale = p.scale;
            {   // the row's queries, as TMA would leave them
                const uint16_t* from = static_cast<const uint16_t*>(p.q);
                if (there) {
                    const int node = (rows.first + row) / p.group;
                    low = first_seen(p, at.b, start, node);
                    nodes = nodes_seen(p, at.b, at.count, node);
                    from += row_at<true>(p, p.qs, rows, row);
                }
                const auto eight = [&](int c) {
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (there && p.q_wide) {
                        w = *reinterpret_cast<const uint4*>(from + c * 8);
                    } else if (there) {
                        uint32_t x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = from[c * 8 + 2 * e] | (uint32_t)from[c * 8 + 2 * e + 1] << 16;
                        w = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                    return w;
                };
                float up = 1.f;
                if (k8 && p.bf16) {  // as fp16 numbers times a power of two of the row's own
                    float top = 0.f;
#pragma unroll 4
                    for (int c = 0; c < DH / 8; ++c) {
                        const uint4 w = eight(c);
                        for (uint32_t x : {w.x, w.y, w.z, w.w}) {
                            const float2 two = tmw::unpack2<__nv_bfloat16>(x);
                            top = fmaxf(top, fmaxf(fabsf(two.x), fabsf(two.y)));
                        }
                    }
                    const int e = max((__float_as_int(top) >> 23) - 127, -100);
                    up = __int_as_float((127 + 14 - e) << 23);
                    q_scale *= __int_as_float((127 - 14 + e) << 23);
                }
#pragma unroll 4
                for (int c = g; c < DH / 8; c += 2) {
                    uint4 w = eight(c);
                    if (k8 && p.bf16) {
                        const auto half = [&](uint32_t x) {
                            const float2 two = tmw::unpack2<__nv_bfloat16>(x);
                            return tmw::pack2<__half>(two.x * up, two.y * up);
                        };
                        w = make_uint4(half(w.x), half(w.y), half(w.z), half(w.w));
                    }
                    *reinterpret_cast<uint4*>(smem + c / 8 * L::kQSub + row * 128 + ((c % 8 ^ (row & 7)) << 4)) = w;
                }
                int warp_low = low;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) warp_low = max(warp_low, __shfl_xor_sync(0xffffffffu, warp_low, d));
                if (lane == 0) lows[warp - 4] = warp_low;
                fence_proxy_async_smem();
                named_barrier_sync(3, 256);
                if (lane == 0) mbar_arrive(q_ready);
            }
            const int lowest = max(max(lows[0], lows[1]), max(lows[2], lows[3]));
            const int t_end = t0 + walk.tiles;
            while (t0 < t_end) {
                const int t1 = min(t0 + kTcMost, t_end);
                float m_used = -CUDART_INF_F, l = 0.f;
                int t = t0 + ((t0 & 1) != g ? 1 : 0);
                const bool none = t >= t1;  // (a single tile is the other stream's)
                for (bool begins = true; t < t1; t += 2, begins = false) {
                    const int buf = t & 3, v_stage = t % VS;
                    const uint32_t s_at = tmem + lane_at + buf * KT;
                    mbar_wait(v_full + 8 * v_stage, v_turn(t), &given_up, p.status);
                    mbar_wait(s_full + 8 * buf, turn(t), &given_up, p.status);
                    if constexpr (k8) mbar_wait(parts_full + 8 * (t & 7), (uint32_t)(t >> 3) & 1, &given_up, p.status);
                    tc_fence_after();
                    const TileInfo& info = infos[t & 15];
                    const bool whole = info.first == 0 && info.last == KT - 1 && info.lost == 0 &&
                                       (info.place < 0 || (info.place + KT <= start && info.place >= lowest));
                    uint32_t s[KT];
                    if (warp_there) {
#pragma unroll
                        for (int c = 0; c < KT / 32; ++c) {
                            uint32_t(&part)[32] = *reinterpret_cast<uint32_t(*)[32]>(s + c * 32);
                            tmem_ld32(s_at + c * 32, part);
                        }
                        tc_wait_ld();
                    }
                    const float4* parts = reinterpret_cast<const float4*>(smem + L::kParts) + (t & 7) * KT;
                    if constexpr (k8) {
                        const uint64_t q_scale2 = ptx::pack2(q_scale, q_scale);
#pragma unroll
                        for (int j = 0; j < KT; j += 2) {
                            const float4 part = parts[j / 2];
                            const uint64_t x = mul2(ptx::pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), ptx::pack2(part.x, part.y));
                            float a, b;
                            ptx::unpack2(fma2(x, q_scale2, ptx::pack2(part.z, part.w)), a, b);
                            s[j] = __float_as_uint(a), s[j + 1] = __float_as_uint(b);
                        }
                    }
                    const float scale = k8 ? 1.f : p.scale;  // (of codes the scores are what they are)
                    uint64_t exists = ~0ull >> (63 - info.last) & ~0ull << info.first, bad = 0;
                    if (!whole) {
                        for (uint32_t todo = info.lost; todo != 0; todo &= todo - 1) bad |= (p.run == 64 ? ~0ull : (1ull << p.run) - 1) << (__ffs(todo) - 1) * p.run;
                        uint64_t seen = exists;
                        if (info.place >= 0) {
                            const int nodes_at = start - info.place, from = low - info.place;  // of node 0, of the window's begin
                            const uint64_t of_nodes = nodes_at >= 0 ? (nodes_at < 64 ? nodes << nodes_at : 0) : (nodes_at > -64 ? nodes >> -nodes_at : 0);
                            const uint64_t tokens = nodes_at <= 0 ? 0 : nodes_at >= 64 ? ~0ull : (1ull << nodes_at) - 1;
                            const uint64_t behind = from <= 0 ? ~0ull : from >= 64 ? 0 : ~0ull << from;
                            seen &= (tokens & behind) | (of_nodes & ~tokens);
                        }
                        const uint64_t nan = bad & seen;
#pragma unroll
                        for (int j = 0; j < KT; ++j)
                            if ((seen >> j & 1) == 0) s[j] = 0xff800000u;
                        if (nan != 0) {
#pragma unroll
                            for (int j = 0; j < KT; ++j)
                                if (nan >> j & 1) s[j] = 0x7fffffffu;
                        }
                    }
                    // O may be changed: the products of the stream's last tile are done
                    auto wait_products = [&]() {
                        mbar_wait(v_free + 8 * ((t - 2) % VS), v_turn(t - 2), &given_up, p.status);
                        tc_fence_after();
                    };
                    if (warp_there) {
                        float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                        for (int j = 0; j < KT; j += 2)
                            asm("max.f32 %0, %0, %1, %2;" : "+f"(top[j / 2 & 3]) : "f"(__uint_as_float(s[j])), "f"(__uint_as_float(s[j + 1])));
                        const float tile_top = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
                        if (begins) {
                            m_used = tile_top;
                        } else if (__any_sync(0xffffffffu, tile_top > m_used + 4.f)) {
                            const float now = tile_top > m_used + 4.f ? tile_top : m_used;
                            const float keep = m_used == -CUDART_INF_F ? 1.f : ex2_ftz(m_used - now);  // (nothing to keep: zeros, or NaN)
                            m_used = now;
                            l *= keep;
                            wait_products();
#pragma unroll 1
                            for (int c = 0; c < DH; c += 16) {
                                uint32_t x[16];
                                tmem_ld16(o_at + c, x);
                                tc_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * keep);
                                tmem_st16(o_at + c, x);
                            }
                            tc_wait_st();
                        }
                    }
                    const float less = (m_used == -CUDART_INF_F ? 0.f : m_used) - kRaise;
                    if (warp_there) {
                        const uint64_t scale2 = ptx::pack2(scale, scale), less2 = ptx::pack2(-less, -less);
                        uint64_t sums[2] = {0, 0};  // two at a time
#pragma unroll
                        for (int c = 0; c < KT / 16; ++c) {
                            uint32_t first[8], second[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                float a, b;
                                const uint64_t two_scores = ptx::pack2(__uint_as_float(s[c * 16 + 2 * e]), __uint_as_float(s[c * 16 + 2 * e + 1]));
                                ptx::unpack2(k8 ? add2(two_scores, less2) : fma2(two_scores, scale2, less2), a, b);
                                a = ex2_ftz(a), b = ex2_ftz(b);
                                if constexpr (k8) {
                                    const float4 two = parts[KT / 2 + c * 8 + e];
                                    const uint64_t w = ptx::pack2(a, b);
                                    sums[e & 1] = fma2(w, ptx::pack2(two.z, two.w), sums[e & 1]);
                                    ptx::unpack2(mul2(w, ptx::pack2(two.x, two.y)), a, b);
                                } else {
                                    sums[e & 1] = add2(sums[e & 1], ptx::pack2(a, b));
                                }
                                split_in_two<M>(a, b, first[e], second[e]);
                            }
                            tmem_st8(s_at + c * 8, first);
                            tmem_st8(s_at + 32 + c * 8, second);
                        }
                        float a, b, c, d;
                        ptx::unpack2(sums[0], a, b);
                        ptx::unpack2(sums[1], c, d);
                        l += (a + b) + (c + d);
                        tc_wait_st();
                    }
                    if (kMayBeWild && !whole) {
                        // values that must not count: a thread has half a row of them (of codes they are fp16 numbers already)
                        const int key = row >> 1;
                        unsigned char* half = smem + L::kV + v_stage * L::kTile + key * 128;
                        constexpr int kChunks = DH / 16;  // sixteen-byte pieces of a half
                        auto piece = [&](int c) {
                            c += (row & 1) * kChunks;
                            return reinterpret_cast<uint4*>(half + c / 8 * L::kSub + ((c % 8 ^ (key & 7)) << 4));
                        };
                        constexpr uint32_t up = BF16 ? 0x00800080u : 0x04000400u, inf = BF16 ? 0x7f80u : 0x7c00u;
                        bool found = false;
                        if (((exists & ~bad) >> key & 1) == 0) {
                            for (int c = 0; c < kChunks; ++c) *piece(c) = make_uint4(0, 0, 0, 0);
                        } else {
                            uint32_t any = 0;
                            for (int c = 0; c < kChunks; ++c) {
                                const uint4 v = *piece(c);
                                any |= ((v.x & 0x7fff7fffu) + up) | ((v.y & 0x7fff7fffu) + up) | ((v.z & 0x7fff7fffu) + up) | ((v.w & 0x7fff7fffu) + up);
                            }
                            found = (any & 0x80008000u) != 0;
                            if (found) wild[g] = 1;
                        }
                        named_barrier_sync(1 + g, 128);
                        const bool any_wild = *(volatile int*)&wild[g] != 0;
                        named_barrier_sync(1 + g, 128);  // (all have read it: the next such tile may set it)
                        if (any_wild) {
                            // Infinities and NaN to the rows that see them, number by number, into O: in front of a part's first product O
                            // is made zero, and that product told to add.
                            if (begins) {
                                for (int c = 0; c < DH; c += 16) {
                                    const uint32_t zero[16] = {};
                                    tmem_st16(o_at + c, zero);
                                }
                                tc_wait_st();
                                if (row == 0) first_adds[g] = 1;
                            } else {
                                wait_products();
                            }
                            uint64_t mine = 0;  // keys that have a weight
#pragma unroll
                            for (int j = 0; j < KT; ++j)
                                if (warp_there && !(ex2_ftz(fmaf(__uint_as_float(s[j]), scale, -less)) == 0.f)) mine |= 1ull << j;
                            for (int j = 0; j < KT; ++j) {
                                const unsigned char* v = smem + L::kV + v_stage * L::kTile + j * 128;
                                for (int d = 0; d < DH; ++d) {
                                    const uint32_t x = *reinterpret_cast<const uint16_t*>(v + d / 64 * L::kSub + ((d % 64 / 8 ^ (j & 7)) << 4) + d % 8 * 2);
                                    if ((x & 0x7fffu) < inf) continue;  // (the same for all rows)
                                    uint32_t o;
                                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(o) : "r"(o_at + d) : "memory");
                                    tc_wait_ld();
                                    const float add = (x & 0x7fffu) > inf ? CUDART_NAN_F : x & 0x8000u ? -CUDART_INF_F : CUDART_INF_F;
                                    if (mine >> j & 1) o = __float_as_uint(__uint_as_float(o) + add);
                                    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(o_at + d), "r"(o) : "memory");
                                    tc_wait_st();
                                }
                            }
                            named_barrier_sync(1 + g, 128);
                            if (found) {
                                for (int c = 0; c < kChunks; ++c) {
                                    uint16_t* x = reinterpret_cast<uint16_t*>(piece(c));
                                    for (int e = 0; e < 8; ++e)
                                        if ((x[e] & 0x7fffu) >= inf) x[e] = 0;
                                }
                            }
                            if (row == 0) wild[g] = 0;
                            named_barrier_sync(1 + g, 128);
                        }
                        fence_proxy_async_smem();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready + 8 * buf);
                }
                if (none) {  // (an O of anything, which must not count)
#pragma unroll 1
                    for (int c = 0; c < DH; c += 16) {
                        const uint32_t zero[16] = {};
                        tmem_st16(o_at + c, zero);
                    }
                    tc_wait_st();
                } else {
                    mbar_wait(v_free + 8 * ((t - 2) % VS), v_turn(t - 2), &given_up, p.status);
                }
                const bool goes_on = t0 + walk.tiles > t_end, last = t1 == t_end;
                const long long slot = (blockIdx.x * 2 + (walk.starts ? 1 : 0)) * (long long)p.rows + row;
                t0 = t1;
                float2 before = make_float2(-CUDART_INF_F, 0.f);  // what the part has so far
                if (goes_on && there) before = p.sums[slot];
                if (row == 0) first_adds[g] = 0;
                stream_sums[g][row] = make_float2(m_used, l);
                tc_fence_before();
                named_barrier_sync(3, 256);
                tc_fence_after();
                // both streams' outputs, a half of the dimensions each
                const float2 other = stream_sums[g ^ 1][row];
                const float m = fmaxf(fmaxf(m_used, other.x), before.x), of = m == -CUDART_INF_F ? 0.f : m;
                float own_part = part_weight(m_used, of);
                float* so_far = p.partial + (slot - row) * DH + row;
                if (goes_on) {  // what the part had goes onto this stream's half (sixteen numbers at a time: every tile of codes 2.5 % slower)
                    const float weight = part_weight(before.x, of);
                    if (warp_there) {
#pragma unroll 1
                        for (int c = g * (DH / 2); c < (g + 1) * (DH / 2); c += 8) {
                            uint32_t x[8];
                            tmem_ld8(o_at + c, x);
                            float had[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) had[e] = there ? so_far[(c + e) * p.rows] : 0.f;
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[e] = __float_as_uint(fmaf(had[e], weight, __uint_as_float(x[e]) * own_part));
                            tmem_st8(o_at + c, x);
                        }
                        tc_wait_st();
                    }
                    own_part = 1.f;
                    named_barrier_sync(3, 256);  // (rows of the last outputs lie across what others had)
                }
                if (warp_there) {
                    const float other_part = part_weight(other.x, of);
                    const float sum = l * part_weight(m_used, of) + other.y * other_part + before.y * part_weight(before.x, of);
                    const bool out = walk.starts && walk.ends && last;
                    const float scale = there && out ? inverse_of<true>(p, rows, row, sum) : 1.f;
                    uint16_t* to = static_cast<uint16_t*>(p.o) + (there ? row_at<true>(p, p.os, rows, row) : 0);
#pragma unroll 2
                    for (int c = g * (DH / 2); c < (g + 1) * (DH / 2); c += 16) {
                        uint32_t x[16], y[16];
                        tmem_ld16(o_at + c, x);
                        tmem_ld16(tmem + lane_at + kO + (g ^ 1) * DH + c, y);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            x[e] = __float_as_uint((__uint_as_float(x[e]) * own_part + __uint_as_float(y[e]) * other_part) * scale);
                        if (there && out) {
                            uint32_t w[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float a = __uint_as_float(x[2 * e]), b = __uint_as_float(x[2 * e + 1]);
                                w[e] = (k8 ? p.bf16 : BF16) ? tmw::pack2<__nv_bfloat16>(a, b) : tmw::pack2<__half>(a, b);
                            }
                            if (p.o_wide) {
                                reinterpret_cast<uint4*>(to + c)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                                reinterpret_cast<uint4*>(to + c)[1] = make_uint4(w[4], w[5], w[6], w[7]);
                            } else {
#pragma unroll
                                for (int e = 0; e < 8; ++e) to[c + 2 * e] = (uint16_t)w[e], to[c + 2 * e + 1] = (uint16_t)(w[e] >> 16);
                            }
                        } else if (there && !last) {  // (dimension by dimension: the rows of a warp side by side)
#pragma unroll
                            for (int e = 0; e < 16; ++e) so_far[(c + e) * p.rows] = __uint_as_float(x[e]);
                        } else if (there) {
#pragma unroll
                            for (int e = 0; e < 16; e += 4)
                                *reinterpret_cast<uint4*>(p.partial + slot * DH + c + e) = make_uint4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                        }
                        __syncwarp();  // (the next load is the whole warp's)
                    }
                    if (there && !out && g == 0) p.sums[slot] = make_float2(m, sum);
                }
                tc_fence_before();
                named_barrier_sync(3, 256);  // (O, the queries and the sums may be written again)
            }
            if (walk.starts && !walk.ends && tid == 128) p.joins[blockIdx.x] = make_int4(at.b, at.item, (int)((walk.item_end - 1) / share.per), 0);
        }
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kColumns);

    // sequences without a place
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        int lo, pos, count;
        bool bad;
        if (tiles_of<KT, true>(p, b, lo, pos, count, bad) > 0 || !bad) continue;
        if (tid == 0) atomicCAS(p.status, 0, (int)TMW_ERR_INVALID_ARGUMENT);
        const int heads = p.group * p.map.kv_heads, all = count < 0 || count > p.nodes ? p.nodes : count;
        for (int i = tid; i < all * heads * DH; i += blockDim.x) {
            const int d = i % DH, r = i / DH, node = r / heads, h = r - node * heads;
            put(p, static_cast<Any16*>(p.o) + b * p.os[0] + h * p.os[1] + node * p.os[2] + d, CUDART_NAN_F);
        }
    }
}

struct TcPlan {
    int rows, grid;
    size_t sums_at, partial_at, bytes;
};
TcPlan tc_plan(const tmw_paged_attention_desc& d, int nodes) {
    TcPlan n;
    const int all = d.heads / d.at.kv_heads * nodes, parts = (all + kTcRows - 1) / kTcRows;
    n.rows = all < kTcRows ? all : kTcRows;  // (a tile costs the same however many rows it has)
    const long long capacity = (long long)d.at.columns * d.at.page_size;
    const long long keys = d.window >= 0 && d.window + (long long)nodes < capacity ? d.window + (long long)nodes : capacity;
    const long long tiles = ((d.n_persistent + kTcKeys - 1) / kTcKeys + keys / kTcKeys + 2) * (long long)d.at.kv_heads * parts * d.at.batch;
    n.grid = (int)(tiles < sm_count() ? tiles : sm_count());
    n.sums_at = (size_t)n.grid * sizeof(int4);
    n.partial_at = (n.sums_at + (size_t)n.grid * 2 * n.rows * sizeof(float2) + 15) & ~(size_t)15;
    n.bytes = n.partial_at + (size_t)n.grid * 2 * n.rows * d.at.head_dim * sizeof(float);
    return n;
}

template <typename P, int DH>
int launch_tc(const tmw_paged_attention_desc& d, PagedAttentionBulk& p, const TcPlan& n, cudaStream_t stream) {
    using L = TcLayout<P, DH>;
    const auto make = [&](CUtensorMap* map, const void* base, int rows) {  // (codes as pairs, rows as they lie)
        return rows == 0 || make_map_2d(map, base, TMW_F16, rows, DH * (int)sizeof(P) / 2, DH * (int)sizeof(P) / 2, p.run, L::k8 ? DH / 2 : 64,
                                        L::k8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B);
    };
    const int rows = d.at.pages * d.at.kv_heads * d.at.page_size, pers = d.at.kv_heads * d.n_persistent;
    if (!make(&p.k_map, d.at.k_pages, rows) || !make(&p.v_map, d.at.v_pages, rows) || !make(&p.k_pers_map, d.k_pers, pers) ||
        !make(&p.v_pers_map, d.v_pers, pers))
        return TMW_ERR_CUDA;
    auto kern = paged_tree_tc_kernel<P, DH>;
    const int smem = L::kBytes + 1024, rc = allow_shared_memory(reinterpret_cast<const void*>(kern), smem);
    if (rc != TMW_OK) return rc;
    kern<<<n.grid, L::kThreads, smem, stream>>>(p);
    TMW_CUDA_TRY(cudaGetLastError());
    if (n.grid > 1)
        TMW_CUDA_TRY(launch_ex(tree_join_kernel<DH>, dim3((unsigned)n.grid - 1, (unsigned)((n.rows + kTreeJoinWarps - 1) / kTreeJoinWarps)),
                               dim3(kTreeJoinWarps * 32), 0, stream, true, 1, static_cast<const PagedAttention&>(p)));
    return TMW_OK;
}
template <int DH>
int launch_tc(const tmw_paged_attention_desc& d, int format, PagedAttentionBulk& p, const TcPlan& n, cudaStream_t stream) {
    if (format == TMW_PAGES_INT8) return launch_tc<int8_t, DH>(d, p, n, stream);
    if (format == TMW_PAGES_E4M3) return launch_tc<E4m3, DH>(d, p, n, stream);
    return d.at.dtype == TMW_BF16 ? launch_tc<__nv_bfloat16, DH>(d, p, n, stream) : launch_tc<__half, DH>(d, p, n, stream);
}

}  // namespace

bool tree_scratch_tc(const tmw_paged_attention_desc& d, const tmw_page_scales& s, int nodes, size_t& bytes) {
    if (!tree_takes_tc(d, s, nodes)) return false;
    bytes = tc_plan(d, nodes).bytes;
    return true;
}

bool tree_launch_tc(const tmw_paged_attention_desc& d, const tmw_page_scales& s, const tmw_paged_tree_desc& tree, void* scratch,
                    size_t scratch_bytes, cudaStream_t stream, int& status) {
    if (!tree_takes_tc(d, s, tree.nodes)) return false;
    PagedAttentionBulk p;
    status = tree_arguments(d, s, tree, scratch, p);
    if (status != TMW_OK) return true;
    const TcPlan n = tc_plan(d, tree.nodes);
    if (scratch_bytes < n.bytes) {
        set_error_text("tmw_paged_tree_attention: scratch smaller than tmw_paged_tree_attention_scratch_bytes()");
        status = TMW_ERR_INVALID_ARGUMENT;
        return true;
    }
    unsigned char* at = static_cast<unsigned char*>(scratch);
    p.rows = n.rows;
    p.pers_tiles = (p.np + kTcKeys - 1) / kTcKeys;
    p.joins = reinterpret_cast<int4*>(at);
    p.sums = reinterpret_cast<float2*>(at + n.sums_at);
    p.partial = reinterpret_cast<float*>(at + n.partial_at);
    p.run = d.at.page_size % 64 == 0 ? 64 : d.at.page_size % 32 == 0 ? 32 : d.at.page_size % 16 == 0 ? 16 : 8;
    status = d.at.head_dim == 64 ? launch_tc<64>(d, s.format, p, n, stream) : launch_tc<128>(d, s.format, p, n, stream);
    return true;
}

}  // namespace tmw
