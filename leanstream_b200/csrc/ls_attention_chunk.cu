// Attention of chunks (many new tokens per sequence) over a paged cache, on
// the 5th-generation tensor cores. The formula is that of ls_attention.cu.
//
// Rows are (token, head of the group): all query heads of a kv head stand in
// one 128-row MMA tile, so a key read serves the whole group. One item is two
// such tiles (Q0, Q1) of one kv head; its slots go by in tiles of 128, each
// worked on in two halves of 64. Per half and row tile i
//     S_i = Q_i K^T            M 128, N 64, K head_dim, into tensor memory
//     P_i = exp2(S_i c - m c)  by one thread per row, back into S_i's columns
//     O_i += P_i V             A from tensor memory, V read as it lies (N-major)
// Each row tile has two S buffers of a half, so that the next S is there when
// its warps end with one: they go from exponentials to exponentials, and the
// tensor cores run beside them. (With one buffer of 128 slots per row tile, its
// P handed over in halves: 910 us for a 4096-token chunk over 16384 slots of
// 128-element heads, against 860; 64-element heads 474 against 392 us.) Roles
// of the warps: 0-3 and 4-7 the rows of Q0 and Q1, 8 and 11 issue their MMAs, 9
// the TMA loads (Q by item; K and V tiles through one ring of 128-slot stages,
// one box per page and 64 elements), 10 lays out the CTA's pieces of items for
// the others.
//
// The running maximum is only raised when a row's maximum grows by more than
// 2^kRaise; raising it rescales O_i in tensor memory, which is rare after the
// first tiles. P is rounded once to the 16-bit type (the MMA's operand), where
// float16 takes it times 2^kChunkShift (ls_attention.h); sums and maxima stay in
// 32 bits, the row sum over the unrounded P.
//
// The tiles of all items, in order, are cut evenly over one CTA per SM, so a
// few long sequences fill the GPU as many short ones do. An item cut over
// several CTAs leaves its parts in scratch, and a short kernel joins them in
// order. A 4096-token chunk over 16384 slots, 32 heads of 128 over 8, takes 860
// to 990 us, 0.97 to 1.1 PFLOP/s; there the board's power limit holds the clock
// near 1.6 GHz. What bounds it and the smaller calls is the rows' chain of maximum
// and exponentials, which the two row tiles run at the same time, so that the
// exponential unit and the tensor cores (49 and 46 % of a mixed call's 227 us)
// take turns more than they overlap.
#include <cuda.h>
#include <stdint.h>

#include <atomic>
#include <cerrno>
#include <type_traits>

#include "ls_attention.h"
#include "ls_tc.h"

namespace lsb {
namespace {

using namespace tc;

constexpr int kKeys = kChunkKeys, kHalf = kKeys / 2;
constexpr int kThreads = 384;  // twelve warps, 168 registers per thread
constexpr uint32_t kPanel = 128 * 128;  // 128 rows of 64 elements
constexpr uint64_t kGraceNs = 1000000000ull;

template <int D>
struct Geo {
    static constexpr uint32_t kPanels = D / 64, kTile = kPanels * kPanel;
    static constexpr uint32_t kStages = D == 128 ? 5 : 8;
    static constexpr uint32_t kRing = 2 * kTile, kBars = kRing + kStages * kTile;
    static constexpr uint32_t kSegs = kBars + 320;
    static constexpr uint32_t kSmem = kSegs + 320 + 1024;  // + alignment of the swizzled tiles
};
static_assert(Geo<128>::kSmem <= 227 * 1024 && Geo<64>::kSmem <= 227 * 1024, "shared memory of a CTA");

// Barriers: ring full / empty, Q full / empty; S full and P ready by row tile
// and buffer, the last two P V of a piece by row tile; the last MMAs of the
// CTA, pieces full / empty.
struct Bars {
    uint32_t base;
    __device__ uint32_t full(uint32_t s) const { return base + 8 * s; }
    __device__ uint32_t empty(uint32_t s) const { return base + 8 * (8 + s); }
    __device__ uint32_t q_full() const { return base + 8 * 16; }
    __device__ uint32_t q_empty() const { return base + 8 * 17; }
    __device__ uint32_t s_full(uint32_t i, uint32_t b) const { return base + 8 * (18 + 2 * i + b); }
    __device__ uint32_t p_ready(uint32_t i, uint32_t b) const { return base + 8 * (22 + 2 * i + b); }
    __device__ uint32_t o_done(uint32_t i) const { return base + 8 * (26 + i); }
    __device__ uint32_t drain(uint32_t i) const { return base + 8 * (28 + i); }
    __device__ uint32_t seg_full(uint32_t s) const { return base + 8 * (30 + s); }
    __device__ uint32_t seg_empty(uint32_t s) const { return base + 8 * (34 + s); }
};

// Lays out the items of a call in `plan` and `items`: for the attention
// (WEIGHTS false) the pairs of row tiles of each sequence, counted in tiles of
// 128 slots; for the weights the tiles of 128 slots, counted in row tiles.
template <bool WEIGHTS>
__device__ void lay_out(const AttnParams& p, ChunkPlan* plan, ChunkItem* list, int32_t cap, uint32_t grid) {
    __shared__ int32_t first[257];  // items before each sequence of the batch piece
    __shared__ int64_t wsum[8];
    constexpr uint32_t kShared = 1024;
    __shared__ int64_t before_item[kShared];  // units before the first items, for the search below
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t per_tile = int32_t(chunk_tokens(p.g));
    int32_t items = 0;
    int64_t units = 0;
    auto scan = [&](int64_t v, int64_t& before) {  // over the block
        int64_t inc = v;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
            if (int(lane) >= o) inc += x;
        }
        __syncthreads();
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        int64_t total = 0;
        before = inc - v;
        for (uint32_t w = 0; w < 8; ++w) {
            if (w < warp) before += wsum[w];
            total += wsum[w];
        }
        return total;
    };
    for (uint32_t b0 = 0; b0 < p.B; b0 += 256) {
        SeqRange s{0, 0, 0, 0};
        if (b0 + tid < p.B) s = load_seq(p, b0 + tid);
        int64_t before;
        const int32_t count = WEIGHTS ? (s.nq ? key_range<kKeys>(p, s, 0, s.nq).tiles : 0)
                                      : (s.nq + 2 * per_tile - 1) / (2 * per_tile);
        int32_t total = int32_t(scan(count, before));
        if (total > cap - items) {  // overlapping q_start ranges
            total = max(0, cap - items);
            if (tid == 0 && p.err) atomicOr(p.err, kErrLength);
        }
        first[tid] = int32_t(before);
        __syncthreads();
        for (int32_t i0 = 0; i0 < total; i0 += 256) {
            const int32_t i = i0 + int32_t(tid);
            ChunkItem it{};
            if (i < total) {
                uint32_t lo = 0, hi = 256;  // the sequence: first[lo] <= i < first[lo + 1]
                while (hi - lo > 1) {
                    const uint32_t mid = (lo + hi) / 2;
                    if (first[mid] <= i) lo = mid;
                    else hi = mid;
                }
                it.b = int32_t(b0 + lo);
                const SeqRange q = load_seq(p, uint32_t(it.b));
                it.q0 = q.q0, it.nq = q.nq, it.n = q.n;
                if (WEIGHTS) {
                    it.t0 = tile_at(key_range<kKeys>(p, q, 0, q.nq), i - first[lo]) * kKeys;
                    const RowTiles r = row_tiles(p, q, it.t0);
                    it.tiles = r.end - r.begin;
                } else {
                    it.t0 = (i - first[lo]) * 2 * per_tile;
                    it.tiles = key_range<kKeys>(p, q, it.t0, min(q.nq, it.t0 + 2 * per_tile)).tiles;
                }
            }
            const int64_t sum = scan(it.tiles ? int64_t(it.tiles + kItemCost) * p.Hkv : 0, before);
            it.units = units + before;
            if (i < total) {
                list[items + i] = it;
                if (items + i < int32_t(kShared)) before_item[items + i] = it.units;
            }
            units += sum;
        }
        items += total;
        __syncthreads();
    }
    // CTAs take at least four tiles: below that the joining of parts costs
    // more than the tiles it spreads.
    const int64_t G = max(int64_t(1), min(int64_t(grid), (units + 3) / 4));
    if (tid == 0) {
        plan->units = units;
        plan->items = items;
        plan->ctas = int32_t(G);
    }
    for (uint32_t c = tid; c < kMaxCtas; c += 256) plan->open[c] = make_int2(-1, 0);
    __syncthreads();
    for (int64_t c = tid; c < G && items; c += 256) {  // the item that holds the CTA's first unit
        const int64_t u = cut_begin(units, G, c);
        int32_t at = 0, end = items;
        while (end - at > 1) {
            const int32_t mid = (at + end) / 2;
            if ((mid < int32_t(kShared) ? before_item[mid] : list[mid].units) <= u) at = mid;
            else end = mid;
        }
        plan->start[c] = at;
    }
}

// Lays out the attention's items (block 0) and the weights' (block 1), and
// appends the new keys and values (blocks 2 .., the same number for each
// sequence, a warp per token at a time).
constexpr uint64_t kAppendBlocks = 16384;  // about: max_q may be far above what the sequences bring
__global__ void __launch_bounds__(256) chunk_prepare_kernel(const AttnParams p, const ChunkScratch sc, uint32_t grid) {
    after_start();
    if (blockIdx.x == 0) {
        lay_out<false>(p, sc.plan, sc.items, int32_t(chunk_items(p.tokens, p.B, p.g)), grid);
    } else if (blockIdx.x == 1) {
        if (p.weights) lay_out<true>(p, sc.w_plan, sc.w_items, int32_t(chunk_weight_items(p.B, p.wlen)), grid);
    } else {
        const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const uint32_t pieces = p.D / 8, per_token = p.Hkv * pieces;
        const uint32_t per_seq = (gridDim.x - 2) / p.B, at = blockIdx.x - 2, b = at / per_seq;
        const SeqRange s = load_seq(p, b);
        for (int64_t t = at % per_seq * 8 + warp; t < s.nq; t += per_seq * 8) {
            const int32_t slot = s.f + int32_t(t);
            if (slot < 0) continue;
            const int32_t id = p.table[int64_t(b) * p.table_s + (slot >> p.pshift)];
            if (uint32_t(id) >= p.pages) {
                if (p.err) atomicOr(p.err, kErrPage);
                continue;
            }
            const int64_t in = slot & int32_t(p.P - 1), tok = s.q0 + t;
            for (uint32_t i0 = lane; i0 < per_token; i0 += 128) {  // four pieces of each under way at a time
                uint4 k[4], v[4];
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                    const uint32_t i = i0 + 32 * x;
                    if (i >= per_token) break;
                    const int64_t h = i / pieces, e = (i % pieces) * 8;
                    k[x] = *reinterpret_cast<const uint4*>(p.k_new + tok * p.kn_ts + h * p.kn_hs + e);
                    v[x] = *reinterpret_cast<const uint4*>(p.v_new + tok * p.vn_ts + h * p.vn_hs + e);
                }
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                    const uint32_t i = i0 + 32 * x;
                    if (i >= per_token) break;
                    const int64_t h = i / pieces, e = (i % pieces) * 8;
                    *reinterpret_cast<uint4*>(p.k_pages + int64_t(id) * p.kp_ps + in * p.kp_ss + h * p.kp_hs + e) =
                        k[x];
                    *reinterpret_cast<uint4*>(p.v_pages + int64_t(id) * p.vp_ps + in * p.vp_ss + h * p.vp_hs + e) =
                        v[x];
                }
            }
        }
    }
}

// One piece of an item in shared memory (four in flight): what the roles need.
// Its halves that some row sees are na halves from ha on (of the first slots),
// then those from hb on; each of its tiles has one at least, unless the item
// sees nothing.
struct Seg {
    int32_t steps;       // tiles; 0: no more pieces
    int32_t row0;        // row of q of the item's first token
    int32_t left;        // tokens of the sequence from there
    int32_t pos0;        // their first cache slot
    int32_t h, b, j0;    // kv head, sequence, first tile
    int32_t ns, first;   // as KeyRange
    int32_t lo, hi, sink;
    int32_t whole;       // the item is all in this piece
    int32_t part;        // which of the CTA's two partial results
    int32_t halves;      // of all tiles
    int32_t na, ha, hb;
    int32_t pad[2];
    __device__ int32_t slot0(int32_t step) const {
        const int32_t j = j0 + step;
        return (j < ns ? j : first + j - ns) * kKeys;
    }
    __device__ void set_halves() {
        const int32_t a = (sink + kHalf - 1) / kHalf, w = max(lo / kHalf, a), end = (hi + kHalf - 1) / kHalf;
        const int32_t j1 = j0 + steps;
        ha = 2 * j0;
        na = j0 < ns ? max(0, min(a, 2 * min(j1, ns)) - ha) : 0;
        hb = j0 < ns ? w : max(w, 2 * (first + j0 - ns));
        const int32_t last = j1 > ns ? min(end, 2 * (first + j1 - ns)) : j1 == ns ? min(end, 2 * ns) : hb;
        halves = na + max(0, last - hb);
    }
};
static_assert(sizeof(Seg) == 80, "four pieces fit");
constexpr uint32_t kSegs = 4, kSegReaders = 11;

// Goes through the halves of a piece, and through the ring stages of their keys
// (values) from piece to piece.
struct Halves {
    uint32_t stage, odd;  // ring stage, and how often the ring has gone round
    int32_t t, h;         // half of the piece, and of the sequence
    bool fresh;           // the first half of its tile
    __device__ void begin(int32_t na, int32_t ha, int32_t hb) {
        t = 0;
        h = na ? ha : hb;
        fresh = true;
    }
    // To the next half; true when it leaves its tile.
    __device__ bool next(int32_t count, int32_t na, int32_t hb) {
        const int32_t tile = h >> 1;
        ++t;
        h = t == na ? hb : h + 1;
        fresh = t == count || (h >> 1) != tile;
        return fresh;
    }
    template <uint32_t kStages>
    __device__ void next_stage() {
        stage += 2;
        if (stage >= kStages) stage -= kStages, ++odd;
    }
};

template <class T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_attn_kernel(const AttnParams p, const ChunkScratch sc, const __grid_constant__ CUtensorMap qmap,
                      const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using G = Geo<D>;
    extern __shared__ uint8_t raw[];
    const uint32_t smem = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* const base = raw + (smem - smem_u32(raw));
    const Bars bar{smem + G::kBars};
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(base + G::kBars + 8 * 38);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t per_tile = int32_t(chunk_tokens(p.g));  // tokens of a row tile

    if (tid == 0) {
        for (uint32_t s = 0; s < G::kStages; ++s) {
            bar_init(bar.full(s), 1);
            bar_init(bar.empty(s), 2);  // the two MMA warps
        }
        bar_init(bar.q_full(), 1);
        bar_init(bar.q_empty(), 2);
        for (uint32_t i = 0; i < 2; ++i) {
            for (uint32_t b = 0; b < 2; ++b) {
                bar_init(bar.s_full(i, b), 1);
                bar_init(bar.p_ready(i, b), 4);  // the four warps of the row tile
            }
            bar_init(bar.o_done(i), 1);
            bar_init(bar.drain(i), 1);
        }
        for (uint32_t i = 0; i < kSegs; ++i) {
            bar_init(bar.seg_full(i), 1);
            bar_init(bar.seg_empty(i), kSegReaders);  // all but warp 10
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) alloc<512>(smem_u32(tmem_slot));
    if (warp == 9 && lane == 0) {
        prefetch_map(&qmap);
        prefetch_map(&kmap);
        prefetch_map(&vmap);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    after_start();
    after_wait();
    constexpr uint32_t kS = 0, kO = 256;  // columns: S_0, S_1 (128 each), O_0, O_1 (D each)
    bool ok = true;
    const Seg* const segs = reinterpret_cast<const Seg*>(base + G::kSegs);

    // the next piece; false when there is none (or when a wait gave up)
    uint32_t sg = 0;
    auto next = [&]() -> bool {
        if (!warp_wait(bar.seg_full(sg % kSegs), (sg / kSegs) & 1u, p.timeout_ns)) return ok = false;
        return uniform(segs[sg % kSegs].steps) != 0;
    };
    auto release = [&]() {
        __syncwarp();
        if (lane == 0) bar_arrive(bar.seg_empty(sg % kSegs));
        ++sg;
    };

    if (warp == 10) {
        // ---- pieces
        if (lane == 0) {
            Walk w;
            KeyRange kr{};
            bool more = w.begin(sc.plan);
            for (; ok; ++sg) {
                if (sg >= kSegs && !bar_wait(bar.seg_empty(sg % kSegs), (sg / kSegs - 1) & 1u, p.timeout_ns)) {
                    ok = false;
                    break;
                }
                more = more && w.next(p, sc.plan, sc.items);
                Seg x{};
                if (more) {
                    const SeqRange q{w.it.q0, w.it.nq, w.it.n, w.it.n - w.it.nq};
                    kr = key_range<kKeys>(p, q, w.it.t0, min(w.it.nq, w.it.t0 + 2 * per_tile));
                    x.steps = w.steps, x.row0 = w.it.q0 + w.it.t0, x.left = w.it.nq - w.it.t0;
                    x.pos0 = w.it.n - w.it.nq + w.it.t0, x.h = w.h, x.b = w.it.b, x.j0 = w.j0;
                    x.ns = kr.ns, x.first = kr.first, x.lo = kr.lo, x.hi = kr.hi, x.sink = kr.sink;
                    x.set_halves();
                    x.whole = w.j0 == 0 && w.steps == w.it.tiles;
                    x.part = w.u != w.u_begin;
                    if (!x.whole && !w.j0) sc.plan->open[blockIdx.x] = make_int2(w.i, w.h);
                }
                *reinterpret_cast<Seg*>(base + G::kSegs + (sg % kSegs) * sizeof(Seg)) = x;
                bar_arrive(bar.seg_full(sg % kSegs));
                if (!more) break;
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // ---- loads
        uint32_t slot = 0;  // ring slots filled
        const uint32_t box = min(p.P, 128u), boxes = 128 / box;
        while (ok && next()) {
            const Seg w = segs[sg % kSegs];
            const int32_t two = w.left > per_tile ? 2 : 1;
            if (sg && !warp_wait(bar.q_empty(), (sg - 1) & 1u, p.timeout_ns)) {
                ok = false;
                break;
            }
            if (lane == 0) {
                bar_arrive_tx(bar.q_full(), uint32_t(two) * G::kPanels * uint32_t(per_tile) * p.g * 128);
                for (int32_t i = 0; i < two; ++i)
                    for (uint32_t c = 0; c < G::kPanels; ++c)
                        tma3(smem + uint32_t(i) * G::kTile + c * kPanel, &qmap, bar.q_full(), int32_t(c * 64),
                             w.h * int32_t(p.g), w.row0 + i * per_tile);
            }
            const int32_t* trow = p.table + int64_t(w.b) * p.table_s;
            auto page_of = [&](int32_t step) -> int32_t {  // this lane's page of a step (outside the pool: zeros)
                if (step >= w.steps || lane >= boxes) return int32_t(p.pages);
                const int32_t k0 = w.slot0(step) + int32_t(lane * box), k1 = k0 + int32_t(box);
                if (!((k0 < w.hi && k1 > w.lo) || k0 < w.sink)) return int32_t(p.pages);
                const int32_t id = trow[k0 >> p.pshift];
                if (uint32_t(id) < p.pages) return id;
                if (p.err) atomicOr(p.err, kErrPage);
                return int32_t(p.pages);
            };
            int32_t next_id = page_of(0);
            for (int32_t j = 0; j < w.steps; ++j) {
                const int32_t id = next_id;
                next_id = page_of(j + 1);
                const int32_t in = (w.slot0(j) + int32_t(lane * box)) & int32_t(p.P - 1);
                for (int kv = 0; kv < 2; ++kv, ++slot) {
                    const uint32_t s = slot % G::kStages, n = slot / G::kStages;
                    if (n && !warp_wait(bar.empty(s), (n - 1) & 1u, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) bar_arrive_tx(bar.full(s), G::kTile);
                    __syncwarp();
                    if (lane < boxes)
                        for (uint32_t c = 0; c < G::kPanels; ++c)
                            tma4(smem + G::kRing + s * G::kTile + c * kPanel + lane * box * 128, kv ? &vmap : &kmap,
                                 bar.full(s), int32_t(c * 64), in, w.h, id);
                }
                if (!ok) break;
            }
            release();
        }
        // every load has landed and every stage been released before the CTA ends
        const uint64_t grace = (ok ? p.timeout_ns : 0) + kGraceNs;
        const uint32_t last = min(slot, G::kStages);
        bool rest = ok;
        for (uint32_t x = slot - last; x < slot; ++x) {
            const uint32_t s = x % G::kStages, n = x / G::kStages;
            warp_wait(bar.full(s), n & 1u, grace);
            rest = rest && warp_wait(bar.empty(s), n & 1u, grace);
        }
        if (sg) warp_wait(bar.q_full(), (sg - 1) & 1u, grace);
    } else if (warp < 8) {
        // ---- rows: thread r of row tile i
        const uint32_t i = warp >> 2;
        const uint32_t r = tid & 127u, quarter = (warp & 3u) << 21;  // lane 32 * (warp % 4) of tensor memory
        const uint32_t ts = tmem + quarter + kS + i * 128, to = tmem + quarter + kO + i * D;
        const int32_t lt = int32_t(r / p.g);
        uint32_t n = 0, no = 0;  // halves passed, results of P V waited for
        Halves at{1, 0, 0, 0, false};
        while (ok && next()) {
            const Seg& w = segs[sg % kSegs];
            const int32_t count = w.halves, na = w.na, hb = w.hb, t_tile = int32_t(i) * per_tile;
            if (t_tile >= w.left) {  // the item has one row tile
                for (int32_t j = w.steps; j; --j) at.next_stage<G::kStages>();
                release();
                continue;
            }
            const bool real = lt < per_tile && t_tile + lt < w.left;
            const bool busy = __any_sync(0xffffffffu, real);
            const int32_t pos = real ? max(w.pos0 + t_tile + lt, -1) : -1;
            // slots [all_lo, all_hi) are seen by every row of the tile, [seen_lo, seen_hi) by some row of the item
            const int32_t all_hi = w.pos0 + t_tile + 1, seen_lo = w.lo, seen_hi = w.hi, sink = w.sink;
            const int32_t all_lo =
                p.window ? int32_t(max(int64_t(0), int64_t(w.pos0) + min(w.left, t_tile + per_tile) - p.window)) : 0;
            float m = -INFINITY, l = 0.f;  // reference maximum and sum of the row
            // waits for S of the next half and clears the values that no row sees:
            // they may be anything, and 0 * NaN is not 0 (the other row tile's warps
            // write the same zeros)
            auto arrived = [&](bool there) {
                if (!there && !warp_wait(bar.s_full(i, n & 1u), (n >> 1) & 1u, p.timeout_ns)) return false;
                const int32_t k0 = at.h * kHalf;
                if (at.t && at.t + 1 == count && !warp_wait(bar.o_done(i), no++ & 1u, p.timeout_ns)) return false;
                if ((k0 >= seen_lo && k0 + kHalf <= seen_hi) || k0 + kHalf <= sink) return true;
                if (!warp_wait(bar.full(at.stage), at.odd & 1u, p.timeout_ns)) return false;
                const int32_t k = k0 + int32_t(r & 63u);
                if ((r >> 6) < G::kPanels && !((k >= seen_lo && k < seen_hi) || k < sink)) {
                    uint8_t* v = base + G::kRing + at.stage * G::kTile + (r >> 6) * kPanel +
                                 (uint32_t(at.h & 1) * kHalf + (r & 63u)) * 128;
#pragma unroll
                    for (uint32_t e = 0; e < 8; ++e) *reinterpret_cast<uint4*>(v + e * 16) = make_uint4(0, 0, 0, 0);
                }
                proxy_fence();
                __syncwarp();
                return true;
            };
            auto advance = [&]() {  // P is there; on to the next half
                __syncwarp();
                if (lane == 0) bar_arrive(bar.p_ready(i, n & 1u));
                if (at.next(count, na, hb)) at.next_stage<G::kStages>();
                ++n;
            };
            at.begin(na, w.ha, hb);
            if (!busy) {
                while (at.t < count && (ok = arrived(false))) advance();
            } else if (count) {
                // The halves overlap: while the exponentials of one are computed, the
                // scores of the next come from tensor memory, and their maximum is
                // taken as soon as P is handed over.
                float x[kHalf], mx;
                auto mask_and_max = [&]() {
                    const int32_t k0 = at.h * kHalf;
                    if (k0 + kHalf > all_hi || k0 < all_lo) {
                        // columns [lo, hi) and those below s
                        const int32_t hi = pos + 1 - k0, s = p.window ? int32_t(p.sinks) - k0 : 0;
                        const int32_t lo = p.window ? pos + 1 - int32_t(p.window) - k0 : 0;
#pragma unroll
                        for (int c = 0; c < kHalf; ++c)
                            if (c >= hi || (c < lo && c >= s)) x[c] = -INFINITY;
                    }
                    float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int c = 4; c < kHalf - 4; c += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e) top[e] = max3(top[e], x[c + e], x[c + 4 + e]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = max3(top[e], top[e], x[kHalf - 4 + e]);
                    mx = max3(max3(top[0], top[1], top[2]), top[3], top[3]);
                };
                if ((ok = arrived(false))) {
                    fence_after();
                    ld32(ts + (n & 1u) * kHalf, x);
                    ld32(ts + (n & 1u) * kHalf + 32, x + 32);
                    wait_ld();
                    mask_and_max();
                }
                while (ok) {
                    const uint32_t tb = ts + (n & 1u) * kHalf, tn = ts + (~n & 1u) * kHalf;
                    const bool last = at.t + 1 == count;
                    // (written so that NaN raises too: the row is NaN from there on, as
                    // it is for an infinite logit)
                    const bool raise = m == -INFINITY ? mx != -INFINITY : !((mx - m) * p.c <= T::kRaise);
                    if (__any_sync(0xffffffffu, raise)) {
                        const float nm = !raise ? m : mx == INFINITY ? NAN : mx;
                        const float f2 = nm == -INFINITY ? 1.f : ex2((m - nm) * p.c);
                        l *= f2;
                        m = nm;
                        if (at.t) {  // the P V before has to be in O: it is when the next S is there
                            if (!last && !warp_wait(bar.s_full(i, ~n & 1u), ((n + 1) >> 1) & 1u, p.timeout_ns))
                                gave_up(p);
                            fence_after();
#pragma unroll
                            for (int c = 0; c < D; c += 16) {
                                float o[16];
                                ld16(to + c, o);
                                wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] *= f2;
                                st16(to + c, o);
                            }
                        }
                    }
                    const float ref = m == -INFINITY ? 0.f : fmaf(-m, p.c, T::kChunkShift);
                    const uint64_t c2 = pack2(p.c, p.c), ref2 = pack2(ref, ref);
                    uint64_t sum[2] = {0, 0};
                    auto probabilities = [&](const float* y, uint32_t to_p) {  // of 32 columns
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float a, d;
                            unpack2(fma2(pack2(y[2 * e], y[2 * e + 1]), c2, ref2), a, d);
                            a = ex2(a), d = ex2(d);
                            sum[e & 1] = add2(sum[e & 1], pack2(a, d));
                            pk[e] = T::pack(a, d);
                        }
                        st16(to_p, pk);
                    };
                    probabilities(x, tb);
                    // (128-element heads are bound by the tensor cores, and by the power
                    // that they draw: there the early read costs 860 -> 942 us for a
                    // 4096-token chunk over 16384 slots; 64-element heads, bound by the
                    // exponentials, gain 436 -> 392 us for two chunks of 3000 tokens)
                    const bool early = D == 64 && !last &&
                                       __all_sync(0xffffffffu, bar_try(bar.s_full(i, ~n & 1u), ((n + 1) >> 1) & 1u));
                    if (early) {
                        fence_after();
                        ld32(tn, x);
                    }
                    probabilities(x + 32, tb + 16);
                    float s0, s1;
                    unpack2(add2(sum[0], sum[1]), s0, s1);
                    l += s0 + s1;
                    wait_st();
                    fence_before();
                    advance();
                    if (last || !(ok = arrived(early))) break;
                    fence_after();
                    if (!early) ld32(tn, x);
                    ld32(tn + 32, x + 32);
                    wait_ld();
                    mask_and_max();
                }
            }
            if (!ok) wait_ld();  // (an early read may be under way)
            const bool any = count != 0;  // (otherwise O is not written)
            if (any && ok) ok = warp_wait(bar.o_done(i), no++ & 1u, p.timeout_ns);
            if (!ok) break;
            if (!any)
                for (int32_t j = w.steps; j; --j) at.next_stage<G::kStages>();
            if (busy) {
                fence_after();
                const bool whole = w.whole != 0;
                const int64_t token = w.row0 + t_tile + lt;
                const int32_t head = w.h * int32_t(p.g) + int32_t(r % p.g);
                uint16_t* out = p.out + token * p.o_ts + int64_t(head) * p.o_hs;
                float* part = sc.part + (2 * int64_t(blockIdx.x) + w.part) * (256 * (D + 2));
                const uint32_t row = i * 128 + r;
                const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : NAN;
#pragma unroll
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    ld32(to + c, o);
                    wait_ld();
                    if (!any)
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0.f;
                    if (real && whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint4 v;
                            v.x = T::pack(o[e] * inv, o[e + 1] * inv);
                            v.y = T::pack(o[e + 2] * inv, o[e + 3] * inv);
                            v.z = T::pack(o[e + 4] * inv, o[e + 5] * inv);
                            v.w = T::pack(o[e + 6] * inv, o[e + 7] * inv);
                            *reinterpret_cast<uint4*>(out + c + e) = v;
                        }
                    } else if (real) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)  // (rows side by side)
                            *reinterpret_cast<float4*>(part + ((c + e) * 256 + row * 4)) =
                                make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                    __syncwarp();
                }
                if (real) {
                    const float ref = fmaf(m, p.c, -T::kChunkShift);
                    if (whole) {
                        if (p.lse) p.lse[token * p.Hq + head] = l == 0.f ? -INFINITY : (ref + lg2(l)) * kLn2;
                    } else {
                        part[256 * D + row] = ref;
                        part[256 * D + 256 + row] = l;
                    }
                }
                fence_before();  // O is read before the next item's first P V
            }
            release();
        }
    } else {
        // ---- MMAs of row tile i: the warp goes through the pieces together, one
        // lane issues. A warp per row tile, so that one's waits and counting
        // pass beside the other's MMAs.
        const uint32_t i = warp == 8 ? 0 : 1;
        constexpr uint32_t kIs = instr(T::kUmmaFormat, 128, kHalf, false);
        constexpr uint32_t kIo = instr(T::kUmmaFormat, 128, D, true);
        const uint32_t q_lo = desc_lo(smem + i * G::kTile, 16), k_lo = desc_lo(smem + G::kRing, 16);
        const uint32_t v_lo = desc_lo(smem + G::kRing, kPanel);
        const uint32_t t_s = tmem + kS + i * 128, t_o = tmem + kO + i * D;
        const bool lead = elect();
        uint32_t n = 0;  // halves passed
        Halves cs{0, 0, 0, 0, false}, cp{1, 0, 0, 0, false};  // for S, and two halves behind for P V
        while (ok && next()) {
            const Seg& w = segs[sg % kSegs];
            const int32_t count = uniform(w.halves), na = uniform(w.na), ha = uniform(w.ha), hb = uniform(w.hb);
            ok = warp_wait(bar.q_full(), sg & 1u, p.timeout_ns);
            if (int32_t(i) * per_tile >= uniform(w.left) || !count) {  // no such row tile, or nothing seen
                for (int32_t j = uniform(w.steps); j && ok; --j)
                    for (Halves* c : {&cs, &cp}) {
                        if (!(ok = ok && warp_wait(bar.full(c->stage), c->odd & 1u, p.timeout_ns))) break;
                        if (lead) commit(bar.empty(c->stage));
                        c->next_stage<G::kStages>();
                    }
                if (ok && lead) commit(bar.q_empty());
                release();
                continue;
            }
            cs.begin(na, ha, hb);
            cp.begin(na, ha, hb);
            auto landed = [&](const Halves& c) {
                return !c.fresh || warp_wait(bar.full(c.stage), c.odd & 1u, p.timeout_ns);
            };
            auto advance = [&](Halves& c) {  // a tile's last half releases its stage
                const uint32_t stage = c.stage;
                if (!c.next(count, na, hb)) return;
                if (lead) commit(bar.empty(stage));
                c.next_stage<G::kStages>();
            };
            auto step_s = [&](uint32_t b) {  // S of the next half, into buffer b
                const uint32_t k = uniform(k_lo + cs.stage * (G::kTile / 16) + (cs.h & 1) * (kHalf * 128 / 16));
                const uint32_t d = uniform(t_s + b * kHalf), q = uniform(q_lo);
                if (lead) {
#pragma unroll
                    for (uint32_t x = 0; x < D / 16; ++x) {
                        const uint32_t off = ((x / 4) * kPanel + (x % 4) * 32) / 16;
                        mma_ss(d, desc_of<1024>(q + off), desc_of<1024>(k + off), kIs, x > 0);
                    }
                    commit(bar.s_full(i, b));
                }
                advance(cs);
                if (cs.t == count && lead) commit(bar.q_empty());
            };
            for (uint32_t t = 0; t < 2 && ok && cs.t < count; ++t) {
                if (!(ok = landed(cs))) break;
                step_s((n + t) & 1u);
            }
            for (; ok && cp.t < count; ++n) {
                const uint32_t b = n & 1u;
                const bool more = cs.t < count;
                if (!(ok = landed(cp) && (!more || landed(cs)) &&
                           warp_wait(bar.p_ready(i, b), (n >> 1) & 1u, p.timeout_ns)))
                    break;
                fence_after();
                const uint32_t v = uniform(v_lo + cp.stage * (G::kTile / 16) + (cp.h & 1) * (kHalf * 128 / 16));
                const uint32_t pt = uniform(t_s + b * kHalf), ot = uniform(t_o);
                if (lead) {
#pragma unroll
                    for (uint32_t x = 0; x < kHalf / 16; ++x)
                        mma_ts(ot, pt + x * 8, desc_of<1024>(v + x * 128), kIo, x > 0 || cp.t > 0);
                    if (!more) commit(bar.o_done(i));
                }
                if (more) step_s(b);
                advance(cp);
            }
            release();
        }
        // MMAs in flight end (bounded) before the tensor memory goes
        if (lead) commit(bar.drain(i));
        warp_wait(bar.drain(i), 0, kGraceNs);
    }
    if (!ok) gave_up(p);
    fence_before();
    __syncthreads();
    if (warp == 8) {
        fence_after();
        dealloc<512>(tmem);
    }
}

// Joins the parts of one item cut over several CTAs: block (c, 16 columns), for
// the item that begins in CTA c and goes on; one thread per row. A part holds its
// sums as [D / 4][256 rows][4], then the rows' maxima and sums.
template <class T, int D>
__global__ void __launch_bounds__(256) chunk_join_kernel(const AttnParams p, const ChunkScratch sc) {
    constexpr int64_t kPart = 256 * (D + 2);
    constexpr int kBatch = 4;  // parts under way at a time
    after_start();
    after_wait();
    const int2 open = sc.plan->open[blockIdx.x];
    if (open.x < 0) return;
    const int64_t U = sc.plan->units, G = sc.plan->ctas;
    const ChunkItem it = sc.items[open.x];
    const uint32_t row = threadIdx.x, r = row & 127u;
    const int32_t per_tile = int32_t(chunk_tokens(p.g));
    const int32_t lt = int32_t(r / p.g), t = it.t0 + int32_t(row >> 7) * per_tile + lt;
    if (lt >= per_tile || t >= it.nq) return;
    const int64_t item = it.units + int64_t(open.y) * (it.tiles + kItemCost);
    const int64_t c0 = blockIdx.x, c1 = cut_owner(U, G, item + it.tiles - 1);
    const int32_t parts = int32_t(c1 - c0) + 1;
    const float* const p0 = sc.part + (2 * c0 + (cut_begin(U, G, c0) != item)) * kPart;
    float mx = -INFINITY, sum = 0.f;
    float4 v[4] = {};
    for (int32_t i0 = 0; i0 < parts; i0 += kBatch) {
        float pm[kBatch], ps[kBatch];
        float4 y[kBatch][4];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int32_t i = min(i0 + k, parts - 1);
            const float* from = i ? sc.part + 2 * (c0 + i) * kPart : p0;
            pm[k] = i0 + k < parts ? from[256 * D + row] : -INFINITY;
            ps[k] = from[256 * D + 256 + row];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[k][e] = *reinterpret_cast<const float4*>(from + ((blockIdx.y * 4 + e) * 256 + row) * 4);
        }
        float nm = mx;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) nm = fmaxf(nm, pm[k]);
        const float ref = nm == -INFINITY ? 0.f : nm, old = ex2(mx - ref);
        mx = nm;
        sum *= old;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e].x *= old, v[e].y *= old, v[e].z *= old, v[e].w *= old;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const float f = ex2(pm[k] - ref);
            sum = fmaf(f, ps[k], sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e].x = fmaf(f, y[k][e].x, v[e].x), v[e].y = fmaf(f, y[k][e].y, v[e].y);
                v[e].z = fmaf(f, y[k][e].z, v[e].z), v[e].w = fmaf(f, y[k][e].w, v[e].w);
            }
        }
    }
    const int64_t token = it.q0 + t;
    const int32_t head = open.y * int32_t(p.g) + int32_t(r % p.g);
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
    uint4 w[2];
    w[0] = make_uint4(T::pack(v[0].x * inv, v[0].y * inv), T::pack(v[0].z * inv, v[0].w * inv),
                      T::pack(v[1].x * inv, v[1].y * inv), T::pack(v[1].z * inv, v[1].w * inv));
    w[1] = make_uint4(T::pack(v[2].x * inv, v[2].y * inv), T::pack(v[2].z * inv, v[2].w * inv),
                      T::pack(v[3].x * inv, v[3].y * inv), T::pack(v[3].z * inv, v[3].w * inv));
    uint16_t* out = p.out + token * p.o_ts + int64_t(head) * p.o_hs + blockIdx.y * 16;
    *reinterpret_cast<uint4*>(out) = w[0];
    *reinterpret_cast<uint4*>(out + 8) = w[1];
    if (!blockIdx.y && p.lse) p.lse[token * p.Hq + head] = sum == 0.f ? -INFINITY : (mx + lg2(sum)) * kLn2;
}

// weights[b, h, slot] of a call, once the rows' lse are known: per tile of 128
// slots and row tile S^T = K Q^T (M the slots, N the rows), then each thread
// sums exp2(S c - lse) over the rows of its slot, with no exchange between
// threads and in a fixed order. Four groups of four warps take the row tiles in
// turn, a score buffer in tensor memory each, so that the MMAs of one run under
// the sums of the others. A slot tile cut over several CTAs is summed, in order,
// by the one that arrives last. The exponentials bound it: 128 x 128 of them per
// 2 * 128^2 * head_dim operations. Two sequences of
// up to 4096 slots, 1024 tokens each, 32 heads of 128 over 8: 71 us, 47 us of
// them the exponentials at 16 a clock and SM. (With two groups 103 us; 85 us
// before short items were charged for their start.) Groups that do not divide 128
// leave columns of a row tile empty: all their tiles take the loop with selects.
constexpr uint32_t kGroups = 4, kLoadWarp = 4 * kGroups, kMmaWarp = kLoadWarp + 1, kLseWarp = kMmaWarp + 1;
constexpr uint32_t kThreadsW = 32 * (kLseWarp + 1), kLses = 8;

template <int D>
struct GeoW {
    static constexpr uint32_t kPanels = D / 64, kTile = kPanels * kPanel, kStages = 4;
    static constexpr uint32_t kRing = 2 * kTile, kBars = kRing + kStages * kTile;  // two K tiles, then Q tiles
    static constexpr uint32_t kLse = kBars + 512;           // [kLses][128] floats
    static constexpr uint32_t kSums = kLse + kLses * 512;  // [2][groups][128]
    static constexpr uint32_t kSmem = kSums + 2 * kGroups * 512 + 1024;
};
struct BarsW {
    uint32_t base;
    __device__ uint32_t k_full(uint32_t i) const { return base + 8 * i; }
    __device__ uint32_t k_empty(uint32_t i) const { return base + 8 * (2 + i); }
    __device__ uint32_t q_full(uint32_t i) const { return base + 8 * (4 + i); }
    __device__ uint32_t q_empty(uint32_t i) const { return base + 8 * (8 + i); }
    __device__ uint32_t s_full(uint32_t i) const { return base + 8 * (12 + i); }
    __device__ uint32_t s_empty(uint32_t i) const { return base + 8 * (16 + i); }
    __device__ uint32_t sums(uint32_t i) const { return base + 8 * (20 + i); }
    __device__ uint32_t summed(uint32_t i) const { return base + 8 * (22 + i); }
    __device__ uint32_t drain() const { return base + 8 * 24; }
    __device__ uint32_t l_full(uint32_t i) const { return base + 8 * (25 + i); }
    __device__ uint32_t l_empty(uint32_t i) const { return base + 8 * (25 + kLses + i); }
    static constexpr uint32_t kEnd = 8 * (25 + 2 * kLses);
};

__device__ __forceinline__ void group_sync(uint32_t group) {
    asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
}

template <class T, int D>
__global__ void __launch_bounds__(kThreadsW, 1)
    chunk_weights_kernel(const AttnParams p, const ChunkScratch sc, const __grid_constant__ CUtensorMap qmap,
                         const __grid_constant__ CUtensorMap kmap) {
    using G = GeoW<D>;
    extern __shared__ uint8_t raw[];
    const uint32_t smem = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* const base = raw + (smem - smem_u32(raw));
    const BarsW bar{smem + G::kBars};
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(base + G::kBars + BarsW::kEnd);
    uint32_t* const last_s = tmem_slot + 1;  // by group
    float* const lse_s = reinterpret_cast<float*>(base + G::kLse);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t per_tile = int32_t(chunk_tokens(p.g));

    if (tid == 0) {
        for (uint32_t i = 0; i < 2; ++i) {
            bar_init(bar.k_full(i), 1);
            bar_init(bar.k_empty(i), 1);
            bar_init(bar.sums(i), 128 * (kGroups - 1));
            bar_init(bar.summed(i), 128);
        }
        for (uint32_t i = 0; i < G::kStages; ++i) {
            bar_init(bar.q_full(i), 1);
            bar_init(bar.q_empty(i), 1);
        }
        for (uint32_t i = 0; i < kGroups; ++i) {
            bar_init(bar.s_full(i), 1);
            bar_init(bar.s_empty(i), 4);
        }
        for (uint32_t i = 0; i < kLses; ++i) {
            bar_init(bar.l_full(i), 32);
            bar_init(bar.l_empty(i), 4);
        }
        bar_init(bar.drain(), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) alloc<512>(smem_u32(tmem_slot));
    if (warp == kLoadWarp && lane == 0) {
        prefetch_map(&qmap);
        prefetch_map(&kmap);
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    after_wait();
    bool ok = true;
    Walk w;
    if (w.begin(sc.w_plan)) {
        uint32_t seg = 0, n = 0;  // pieces begun, row tiles passed
        if (warp == kLoadWarp) {
            const uint32_t box = min(p.P, 128u), boxes = 128 / box;
            for (; ok && w.next(p, sc.w_plan, sc.w_items); ++seg) {
                const SeqRange s{w.it.q0, w.it.nq, w.it.n, w.it.n - w.it.nq};
                const int32_t tile0 = row_tiles(p, s, w.it.t0).begin + w.j0;
                const uint32_t kb = seg & 1u;
                if (seg >= 2 && !warp_wait(bar.k_empty(kb), (seg / 2 - 1) & 1u, p.timeout_ns)) {
                    ok = false;
                    break;
                }
                int32_t id = int32_t(p.pages);
                const int32_t k0 = w.it.t0 + int32_t(lane * box);
                if (lane < boxes && k0 < w.it.n) {  // (slots that no row sees may be read: their sums are not kept)
                    const KeyRange kr = key_range<kKeys>(p, s, 0, s.nq);
                    if ((k0 < kr.hi && k0 + int32_t(box) > kr.lo) || k0 < kr.sink) {
                        id = p.table[int64_t(w.it.b) * p.table_s + (k0 >> p.pshift)];
                        if (uint32_t(id) >= p.pages) id = int32_t(p.pages);  // reported by the attention
                    }
                }
                if (lane == 0) bar_arrive_tx(bar.k_full(kb), G::kTile);
                __syncwarp();
                if (lane < boxes)
                    for (uint32_t c = 0; c < G::kPanels; ++c)
                        tma4(smem + kb * G::kTile + c * kPanel + lane * box * 128, &kmap, bar.k_full(kb),
                             int32_t(c * 64), k0 & int32_t(p.P - 1), w.h, id);
                for (int32_t j = 0; j < w.steps; ++j, ++n) {
                    const uint32_t st = n % G::kStages;
                    if (n >= G::kStages && !warp_wait(bar.q_empty(st), (n / G::kStages - 1) & 1u, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        bar_arrive_tx(bar.q_full(st), G::kPanels * uint32_t(per_tile) * p.g * 128);
                        for (uint32_t c = 0; c < G::kPanels; ++c)
                            tma3(smem + G::kRing + st * G::kTile + c * kPanel, &qmap, bar.q_full(st), int32_t(c * 64),
                                 w.h * int32_t(p.g), w.it.q0 + (tile0 + j) * per_tile);
                    }
                    __syncwarp();
                }
                if (!ok) {
                    ++seg;
                    break;
                }
            }
            const uint64_t grace = (ok ? p.timeout_ns : 0) + kGraceNs;
            bool rest = ok;
            for (uint32_t x = n - min(n, G::kStages); x < n; ++x) {
                warp_wait(bar.q_full(x % G::kStages), (x / G::kStages) & 1u, grace);
                rest = rest && warp_wait(bar.q_empty(x % G::kStages), (x / G::kStages) & 1u, grace);
            }
            for (uint32_t x = seg - min(seg, 2u); x < seg; ++x) {
                warp_wait(bar.k_full(x & 1u), (x / 2) & 1u, grace);
                rest = rest && warp_wait(bar.k_empty(x & 1u), (x / 2) & 1u, grace);
            }
        } else if (warp == kMmaWarp) {
            constexpr uint32_t kIs = instr(T::kUmmaFormat, 128, 128, false);
            const uint32_t k_lo = desc_lo(smem, 16), q_lo = desc_lo(smem + G::kRing, 16);
            const bool lead = elect();
            while (ok && w.next(p, sc.w_plan, sc.w_items)) {
                const int32_t steps = uniform(w.steps);
                const uint32_t kb = seg & 1u;
                ok = warp_wait(bar.k_full(kb), (seg / 2) & 1u, p.timeout_ns);
                for (int32_t j = 0; j < steps && ok; ++j, ++n) {
                    const uint32_t st = n % G::kStages, sb = n % kGroups;
                    if (!warp_wait(bar.q_full(st), (n / G::kStages) & 1u, p.timeout_ns) ||
                        (n >= kGroups && !warp_wait(bar.s_empty(sb), (n / kGroups - 1) & 1u, p.timeout_ns))) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    const uint32_t a = k_lo + kb * (G::kTile / 16), b = q_lo + st * (G::kTile / 16);
                    if (lead) {
#pragma unroll
                        for (uint32_t x = 0; x < D / 16; ++x) {
                            const uint32_t off = ((x / 4) * kPanel + (x % 4) * 32) / 16;
                            mma_ss(tmem + sb * 128, desc_of<1024>(a + off), desc_of<1024>(b + off), kIs, x > 0);
                        }
                        commit(bar.s_full(sb));
                        commit(bar.q_empty(st));
                    }
                }
                if (ok && lead) commit(bar.k_empty(kb));
                ++seg;
            }
            if (lead) commit(bar.drain());
            warp_wait(bar.drain(), 0, kGraceNs);
            __syncwarp();
        } else if (warp == kLseWarp) {
            // -lse (base 2) of each row tile, one tile under way while the one before is stored
            float held[4];
            auto store = [&](uint32_t at) {
                const uint32_t sl = at % kLses;
                if (at >= kLses && !warp_wait(bar.l_empty(sl), (at / kLses - 1) & 1u, p.timeout_ns)) return false;
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) lse_s[sl * 128 + x * 32 + lane] = -held[x] * kLog2e;
                bar_arrive(bar.l_full(sl));
                return true;
            };
            int32_t ct[4], ch[4];
#pragma unroll
            for (int32_t x = 0; x < 4; ++x) {
                const int32_t r = x * 32 + int32_t(lane);
                ct[x] = r / int32_t(p.g), ch[x] = r % int32_t(p.g);
            }
            while (ok && w.next(p, sc.w_plan, sc.w_items)) {
                const SeqRange s{w.it.q0, w.it.nq, w.it.n, w.it.n - w.it.nq};
                const int32_t tile0 = row_tiles(p, s, w.it.t0).begin + w.j0;
                for (int32_t j = 0; j < w.steps && ok; ++j, ++n) {
                    float y[4];
#pragma unroll
                    for (int32_t x = 0; x < 4; ++x) {
                        const int32_t t = (tile0 + j) * per_tile + ct[x];
                        y[x] = ct[x] < per_tile && t < s.nq
                                   ? p.lse[int64_t(s.q0 + t) * p.Hq + w.h * int32_t(p.g) + ch[x]] : 0.f;
                    }
                    if (n) ok = store(n - 1);
#pragma unroll
                    for (int32_t x = 0; x < 4; ++x) held[x] = y[x];
                }
            }
            if (ok && n) ok = store(n - 1);
        } else {
            const uint32_t grp = warp >> 2, r = tid & 127u;
            const uint32_t ts = tmem + ((warp & 3u) << 21) + grp * 128;
            float* const sums_s = reinterpret_cast<float*>(base + G::kSums);
            // (after a wait that gave up the pieces still go by, so that every warp
            // meets its group's barriers; it waits for, reads and arrives on nothing
            // else, or a phase could get arrivals of a later one)
            for (; w.next(p, sc.w_plan, sc.w_items); ++seg) {
                const SeqRange s{w.it.q0, w.it.nq, w.it.n, w.it.n - w.it.nq};
                const int32_t tile0 = row_tiles(p, s, w.it.t0).begin + w.j0;
                const int32_t k0 = w.it.t0, k = k0 + int32_t(r);
                const uint32_t closer = (n + uint32_t(w.steps) - 1) % kGroups;  // group of the last row tile
                float* const wt = p.weights + int64_t(w.it.b) * p.w_ss + int64_t(w.h) * p.w_hs + k;
                const bool kept = k < s.n && (!p.window || int64_t(k) > int64_t(s.f) - int64_t(p.window) ||
                                              uint32_t(k) < p.sinks);
                float old = 0.f, acc = 0.f;
                if (grp == closer && kept && k < s.f) old = *wt;
                for (int32_t j = int32_t((grp - n) % kGroups); j < w.steps; j += int32_t(kGroups)) {
                    const uint32_t at = n + uint32_t(j), sl = at % kLses;
                    if (!(ok = ok && warp_wait(bar.l_full(sl), (at / kLses) & 1u, p.timeout_ns) &&
                               warp_wait(bar.s_full(grp), (at / kGroups) & 1u, p.timeout_ns)))
                        break;
                    const int32_t t0 = (tile0 + j) * per_tile, cols = min(per_tile, s.nq - t0) * int32_t(p.g);
                    const int32_t p0 = s.f + t0, p1 = p0 + min(per_tile, s.nq - t0) - 1;
                    const float4* ls = reinterpret_cast<const float4*>(lse_s + sl * 128);
                    const uint64_t c2 = pack2(p.c, p.c);
                    uint64_t sum[2] = {0, 0};
                    auto four = [&](const float* x, const float4 v, float (&y)[4]) {
                        unpack2(fma2(pack2(x[0], x[1]), c2, pack2(v.x, v.y)), y[0], y[1]);
                        unpack2(fma2(pack2(x[2], x[3]), c2, pack2(v.z, v.w)), y[2], y[3]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = ex2(y[i]);
                    };
                    fence_after();
                    if (cols == 128 && k0 + kKeys - 1 <= p0 && (!p.window || int64_t(p1) < int64_t(k0) + p.window)) {
                        float x[2][32];
                        ld32(ts, x[0]);
                        wait_ld();
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (c < 3) ld32(ts + (c + 1) * 32, x[(c + 1) & 1]);
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                float y[4];
                                four(x[c & 1] + e, ls[c * 8 + e / 4], y);
                                sum[0] = add2(sum[0], pack2(y[0], y[1]));
                                sum[1] = add2(sum[1], pack2(y[2], y[3]));
                            }
                            if (c < 3) wait_ld();
                        }
                    } else {
                        // columns [lo, hi): rows whose token sees slot k. A loop of its own: with
                        // the selects in it the loop above took 1.75 times as long
                        const int64_t last = p.window && uint32_t(k) >= p.sinks ? int64_t(k) + p.window - p0 : per_tile;
                        const int32_t lo = min(max(k - p0, 0), per_tile) * int32_t(p.g);
                        const int32_t hi =
                            min(int32_t(max(int64_t(0), min(last, int64_t(per_tile)))) * int32_t(p.g), cols);
#pragma unroll 1
                        for (int c = 0; c < 128; c += 16) {
                            if (!__any_sync(0xffffffffu, max(lo, c) < min(hi, c + 16))) continue;
                            float x[16];
                            ld16(ts + c, x);
                            wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e += 4) {
                                float y[4];
                                four(x + e, ls[(c + e) / 4], y);
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (c + e + i < lo || c + e + i >= hi) y[i] = 0.f;
                                sum[0] = add2(sum[0], pack2(y[0], y[1]));
                                sum[1] = add2(sum[1], pack2(y[2], y[3]));
                            }
                        }
                    }
                    float s0, s1, s2, s3;
                    unpack2(sum[0], s0, s1);
                    unpack2(sum[1], s2, s3);
                    acc += (s0 + s1) + (s2 + s3);
                    fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        bar_arrive(bar.s_empty(grp));
                        bar_arrive(bar.l_empty(sl));
                    }
                }
                n += uint32_t(w.steps);
                // the group that had the last row tile adds the groups' sums, in their order
                const uint32_t pb = seg & 1u;
                float* const sums = sums_s + pb * kGroups * 128;
                // (every group meets every phase of `summed`: a closer that ran ahead would
                // take the phase of `sums` two pieces back for its own)
                if (seg >= 2) ok = ok && warp_wait(bar.summed(pb), (seg / 2 - 1) & 1u, p.timeout_ns);
                if (grp != closer) {
                    if (ok) {
                        sums[grp * 128 + r] = acc;
                        bar_arrive(bar.sums(pb));
                    }
                    continue;
                }
                ok = ok && warp_wait(bar.sums(pb), (seg / 2) & 1u, p.timeout_ns);
                const float own = acc;
                acc = 0.f;
#pragma unroll
                for (uint32_t x = 0; x < kGroups; ++x) acc += x == grp ? own : sums[x * 128 + r];
                if (ok) bar_arrive(bar.summed(pb));
                bool write = true;
                if (w.steps != w.it.tiles) {
                    const int64_t c0 = cut_owner(w.U, w.G, w.item);
                    const int64_t c1 = cut_owner(w.U, w.G, w.item + w.it.tiles - 1);
                    auto piece = [&](int64_t c) {
                        return sc.w_part + (2 * c + (c == c0 && cut_begin(w.U, w.G, c0) != w.item ? 1 : 0)) * 128;
                    };
                    sc.w_part[(2 * int64_t(blockIdx.x) + (w.u == w.u_begin ? 0 : 1)) * 128 + r] = acc;
                    __threadfence();
                    group_sync(grp);
                    if (r == 0) {
                        const bool last = atomicAdd(p.count + c0, 1u) == uint32_t(c1 - c0);
                        if (last) p.count[c0] = 0;
                        last_s[grp] = last;
                    }
                    group_sync(grp);
                    write = last_s[grp] != 0;
                    if (write) {
                        __threadfence();
                        acc = 0.f;
                        for (int64_t c = c0; c <= c1; ++c) acc += __ldcg(piece(c) + r);
                    }
                    group_sync(grp);  // last_s is free again
                }
                if (write && kept && ok) *wt = old + acc;
            }
        }
        if (!ok) gave_up(p);
    }
    fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        fence_after();
        dealloc<512>(tmem);
    }
}

template <class T, int D>
int launch_chunk_weights(const AttnParams& p, const ChunkScratch& s, uint32_t grid, const CUtensorMap& qm,
                         const CUtensorMap& km, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return int(e);
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!bit || !(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(chunk_weights_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(GeoW<D>::kSmem));
        if (e != cudaSuccess) return int(e);
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    return int(launch_after(chunk_weights_kernel<T, D>, grid, kThreadsW, GeoW<D>::kSmem, stream, p, s, qm, km));
}

template <class T, int D>
int launch(const AttnParams& p, bool bf16, const ChunkScratch& s, uint32_t grid, cudaStream_t stream) {
    CUtensorMap qm, km, vm;
    const uint64_t qd[3] = {D, p.Hq, p.tokens};
    const int64_t qs[2] = {p.q_hs, p.q_ts};
    const uint32_t qb[3] = {64, p.g, chunk_tokens(p.g)};
    const uint64_t kd[4] = {D, p.P, p.Hkv, p.pages};
    const int64_t ks[3] = {p.kp_ss, p.kp_hs, p.kp_ps}, vs[3] = {p.vp_ss, p.vp_hs, p.vp_ps};
    const uint32_t kb[4] = {64, p.P < 128 ? p.P : 128, 1, 1};
    if (!encode_map(&qm, bf16, p.q, 3, qd, qs, qb) || !encode_map(&km, bf16, p.k_pages, 4, kd, ks, kb) ||
        !encode_map(&vm, bf16, p.v_pages, 4, kd, vs, kb))
        return EINVAL;
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return int(e);
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!bit || !(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(chunk_attn_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(Geo<D>::kSmem));
        if (e != cudaSuccess) return int(e);
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    const uint64_t most = (uint64_t(p.max_q < p.tokens ? p.max_q : p.tokens) + 7) / 8, fair = kAppendBlocks / p.B + 1;
    const uint32_t append = p.k_new ? p.B * uint32_t(most < fair ? most : fair) : 0;
    chunk_prepare_kernel<<<2 + append, 256, 0, stream>>>(p, s, grid);
    e = cudaGetLastError();
    if (e == cudaSuccess)
        e = launch_after(chunk_attn_kernel<T, D>, grid, kThreads, Geo<D>::kSmem, stream, p, s, qm, km, vm);
    if (e == cudaSuccess) e = launch_after(chunk_join_kernel<T, D>, dim3(grid, D / 16), 256, 0, stream, p, s);
    if (e != cudaSuccess || !p.weights) return int(e);
    return launch_chunk_weights<T, D>(p, s, grid, qm, km, stream);
}

using Encode = decltype(&cuTensorMapEncodeTiled);
Encode encoder() {
    static const Encode fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &res) !=
                cudaSuccess ||
            res != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<Encode>(f);
    }();
    return fn;
}

}  // namespace

bool encode_map(CUtensorMap* map, bool bf16, const void* base, uint32_t rank, const uint64_t* dims,
                const int64_t* strides, const uint32_t* box) {
    cuuint64_t size[5], bytes[4];
    cuuint32_t part[5];
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    for (uint32_t i = 0; i < rank; ++i) {
        size[i] = dims[i];
        part[i] = box[i];
        if (i)  // the stride of a dimension of one is never used
            bytes[i - 1] = dims[i] > 1 ? cuuint64_t(strides[i - 1]) * 2 : 128;
    }
    return encoder() &&
           encoder()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                     const_cast<void*>(base), size, bytes, part, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_chunk(const AttnParams& p, uint32_t dtype, const ChunkScratch& s, uint32_t sms, cudaStream_t stream) {
    const uint32_t grid = sms < kMaxCtas ? sms : kMaxCtas;
    if (p.D == 64)
        return dtype == LS_B200_BF16 ? launch<BF16, 64>(p, true, s, grid, stream)
                                     : launch<F16, 64>(p, false, s, grid, stream);
    return dtype == LS_B200_BF16 ? launch<BF16, 128>(p, true, s, grid, stream)
                                 : launch<F16, 128>(p, false, s, grid, stream);
}

}  // namespace lsb
