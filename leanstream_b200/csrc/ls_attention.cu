// Attention of new tokens over a paged key/value cache.
//
// Sequence b of the call holds n = kv_len[b] cache slots, the last of which
// are its new tokens; query token t stands at slot p = f + t (f the slot of
// the first new token). It sees the slots k <= p, and under a window W only
// those with k > p - W or k < S (the first S slots stay visible). Per query
// head, with s_k = scale * q . k over the visible slots:
//     lse = log sum_k exp(s_k),   out = sum_k exp(s_k - lse) v_k,
// and where weights are kept, weights[b, kv head, k] += sum over the new
// tokens and the query heads of the group of exp(s_k - lse).
//
// One pass over the cache: every warp keeps the running maximum m and sum l of
// its rows and rescales its fp32 output sum when m grows, so keys and values
// are read once and no logit goes to memory (a call with weights stores its
// logits, 4 B per row and slot beside the 4 * head_dim B of its key and value,
// because the weights need the final lse).
#include <stdint.h>

#include <atomic>
#include <cerrno>
#include <cmath>
#include <type_traits>

#include "ls_attention.h"
#include "ls_tc.h"

namespace lsb {
namespace {

using namespace tc;

constexpr int kDecWarps = 4, kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16;                    // slots of one warp's step
constexpr int kDecTile = kDecKeys * kDecWarps;  // slots of one unit of work
constexpr uint32_t kDecSegs = 12;               // pieces of items listed at a time
constexpr int64_t kDecItemCost = 2;             // units that beginning and joining an item counts as
constexpr int64_t kDecMinUnits = 2 + kDecItemCost;  // units that a CTA takes at least
constexpr uint64_t kGraceNs = 1000000000ull;
constexpr uint64_t kShortNs = 100000;  // bounds that a barrier's try may sleep over: a load takes less

// Three CTAs per SM by registers; the ring takes the shared memory that leaves.
template <int D>
struct GeoD {
    static constexpr int kCtas = 3, kRows = 16;
    static constexpr uint32_t kHalf = kDecKeys * D * 2, kStage = 2 * kHalf;  // a step's keys, and its values
    static constexpr int kStages = 2 * (128 / D);
    static constexpr uint32_t kRing = kDecWarps * kStages * kStage;
    static constexpr uint32_t kJoin = kRing, kJoinBytes = kRows * D * 4;  // sums of the warps
    static constexpr uint32_t kSegs = kJoin + kJoinBytes, kBars = kSegs + kDecSegs * 64;
    static constexpr uint32_t kStat = kBars + 8 * kDecWarps * kStages;  // scan words, flags; row maxima and sums
    static constexpr uint32_t kSmem = kStat + 128 + 2 * kDecWarps * kRows * 4;
    static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

// A piece of an item: `steps` tiles from tile j0 of a sequence and kv head.
struct DecSeg {
    int32_t b, h, q0, rows;
    int32_t f, hi, lo, sink;  // as SeqRange, KeyRange
    int32_t ns, first, j0, steps;
    int32_t tiles, own;       // tiles of the item; own: it does not begin the CTA's range
    int64_t item;             // first unit of the item
    __device__ __forceinline__ int32_t slot0(int32_t step, uint32_t warp) const {
        const int32_t j = j0 + step;
        return (j < ns ? j : first + j - ns) * kDecTile + int32_t(warp) * kDecKeys;
    }
};
static_assert(sizeof(DecSeg) == 64, "list entries");

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {  // zeros where off (src is not read)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_arrive(uint32_t bar) {  // one arrival, when this thread's copies have landed
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
// 16-byte piece of a row in a tile of ROWS rows: panels of 64 elements, each
// row's pieces XORed with its low bits (the 128-byte swizzle of the TMA), so
// that the eight rows of an ldmatrix lie in different banks.
template <int ROWS>
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t piece) {
    return (piece >> 3) * (ROWS * 128) + row * 128 + (((piece ^ row) & 7u) << 4);
}

// Sums of (x, y) over the block, and over the threads before this one.
struct Pair {
    int64_t x;
    int32_t y;
};
__device__ __forceinline__ Pair block_scan(Pair v, Pair* sh, Pair& before) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Pair inc = v;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc.x, o);
        const int32_t y = __shfl_up_sync(0xffffffffu, inc.y, o);
        if (int(lane) >= o) inc.x += x, inc.y += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = inc;
    __syncthreads();
    Pair total{0, 0};
    before = Pair{inc.x - v.x, inc.y - v.y};
    for (uint32_t w = 0; w < kDecWarps; ++w) {
        if (w < warp) before.x += sh[w].x, before.y += sh[w].y;
        total.x += sh[w].x, total.y += sh[w].y;
    }
    return total;
}

// The kernel for few rows per sequence and kv head (decoding, drafts): bound
// by the read of the cache. An item is a sequence and kv head; its rows are
// (token, head of the group), so all heads that share a key read it once. The
// units (64 slots) of all items, in order, are cut evenly over the CTAs. A
// CTA's four warps take 16 slots of a unit each, with rings, maxima and sums
// of their own, and meet only at the end of a piece; the loads run on into the
// next piece meanwhile. A step's keys and values are one TMA box each; steps
// with new tokens or with slots that no row sees come by 16-byte copies
// instead, row by row, with zeros for those. An item cut over several CTAs is
// joined, in the order of its pieces, by the CTA that arrives last. The
// probabilities meet the values as the sum of two 16-bit numbers, about twice the
// bits of one (down to float16's smallest step, 2^-40 of the row's largest): the
// multiplier is idle beside the loads. Two sequences
// of up to 131072 slots, 64 heads of 128 over 8: 180 us, 5.7 TB/s of the cache;
// 32 of up to 4096 slots, 32 heads: 60 us, 4.6 TB/s; one of 97 slots: 8.5 us.
template <class T, int D>
__global__ void __launch_bounds__(kDecThreads, GeoD<D>::kCtas)
    attn_decode_kernel(const AttnParams p, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
    using G = GeoD<D>;
    constexpr int MR = G::kRows, KS = D / 16, PIECES = D / 8, RPI = 32 / PIECES, ITERS = kDecKeys / RPI;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    DecSeg* const segs = reinterpret_cast<DecSeg*>(smem + G::kSegs);
    float* const join = reinterpret_cast<float*>(smem + G::kJoin);
    Pair* const scan = reinterpret_cast<Pair*>(smem + G::kStat);
    volatile uint32_t* const flag = reinterpret_cast<uint32_t*>(scan + kDecWarps);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t g = int32_t(p.g);
    const uint32_t bar0 = sbase + G::kBars + 8 * warp * G::kStages;  // this warp's stages
    const uint32_t ring = sbase + warp * (G::kStages * G::kStage);

    after_start();
    if (lane == 0) {
        for (int i = 0; i < G::kStages; ++i) bar_init(bar0 + 8 * i, 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // units of this thread's sequence (of the first 128), and of the call; y: 1
    // where the sequence has rows
    auto units_of = [&](uint32_t b, SeqRange& s) -> Pair {
        s = SeqRange{0, 0, 0, 0};
        if (b < p.B) s = load_seq(p, b);
        if (!s.nq) return Pair{0, 0};
        return Pair{(key_range<kDecTile>(p, s, 0, s.nq).tiles + kDecItemCost) * p.Hkv, 1};
    };
    SeqRange seq0;
    const Pair v0 = units_of(tid, seq0);
    Pair before0;
    const Pair total0 = block_scan(v0, scan, before0);
    int64_t U = total0.x;
    for (uint32_t b0 = kDecThreads; b0 < p.B; b0 += kDecThreads) {
        SeqRange s;
        Pair before;
        U += block_scan(units_of(b0 + tid, s), scan, before).x;
    }
    if (!U) return;
    const int64_t NC = max(int64_t(1), min(int64_t(gridDim.x), (U + kDecMinUnits - 1) / kDecMinUnits));
    if (int64_t(blockIdx.x) >= NC) return;
    const int64_t cta = blockIdx.x, u_begin = cut_begin(U, NC, cta), u_end = cut_begin(U, NC, cta + 1);
    // after a wait that gave up the warp loads, computes and appends no more, and
    // only meets the CTA's barriers
    bool ok = true;
    uint32_t used = 0, filled = 0;  // steps of this warp: landed, loaded

    for (int64_t u = u_begin; u < u_end;) {
        // the next pieces, listed by the threads of their sequences: items (y
        // counts sequences with rows) from the one that holds unit u
        if (tid == 0) flag[0] = flag[1] = 0;
        __syncthreads();
        int64_t base = 0;
        int32_t seqs = 0;
        for (uint32_t b0 = 0; b0 < p.B && base < u_end; b0 += kDecThreads) {
            SeqRange s = seq0;
            Pair v = v0, before = before0, total = total0;
            if (b0) {
                v = units_of(b0 + tid, s);
                total = block_scan(v, scan, before);
            }
            const int64_t at = base + before.x, item_units = v.y ? v.x / p.Hkv : 1;
            const int32_t seq = seqs + before.y;
            if (v.y && u >= at && u < at + v.x)
                flag[1] = uint32_t(seq * int32_t(p.Hkv) + int32_t((u - at) / item_units));
            __syncthreads();
            const int64_t from = max(u, at), to = min(u_end, at + v.x);
            if (from < to) {
                const KeyRange kr = key_range<kDecTile>(p, s, 0, s.nq);
                int32_t h = int32_t((from - at) / item_units);
                int32_t idx = seq * int32_t(p.Hkv) + h - int32_t(flag[1]);
                for (; h < int32_t(p.Hkv) && idx < int32_t(kDecSegs); ++h, ++idx) {
                    DecSeg x;
                    x.item = at + h * item_units + kDecItemCost;
                    const int64_t a = max(x.item, u), e = min(x.item + kr.tiles, u_end);
                    if (a >= e) break;  // only the item's cost lies in the range
                    x.b = int32_t(b0 + tid), x.h = h, x.q0 = s.q0, x.rows = s.nq * g;
                    x.f = s.f, x.hi = kr.hi, x.lo = kr.lo, x.sink = kr.sink, x.ns = kr.ns, x.first = kr.first;
                    x.tiles = kr.tiles;
                    x.j0 = int32_t(a - x.item), x.steps = int32_t(e - a);
                    x.own = a != u_begin;
                    segs[idx] = x;
                    atomicMax(const_cast<uint32_t*>(flag), uint32_t(idx + 1));
                }
            }
            base += total.x;
            seqs += total.y;
        }
        __syncthreads();
        const uint32_t count = flag[0];
        if (!count) break;  // what is left of the range is the cost of an item

        // Steps in blocks of 32, laid out by the lanes side by side: lane i holds
        // step base + i, its first slot (a multiple of 16) with flags below.
        constexpr int32_t kSeen = 1, kEdge = 2, kMasked = 4;
        auto lay_out = [&](uint32_t c, int32_t step) -> int32_t {
            if (c >= count) return 0;
            const DecSeg& x = segs[c];
            if (step >= x.steps) return 0;
            const int32_t k0 = x.slot0(step, warp), k1 = k0 + kDecKeys;
            if (!((k0 < x.hi && k1 > x.lo) || k0 < x.sink)) return 0;
            // edge: new tokens, or slots that no row sees; masked: a row does not see all
            const bool edge = (p.fused && k1 > x.f) || k1 > x.hi || (k0 < x.lo && k1 > x.sink);
            const bool masked = k1 - 1 > x.f || (p.window && int64_t(k0) <= int64_t(x.hi) - 1 - int64_t(p.window));
            return k0 | kSeen | (edge ? kEdge : 0) | (masked ? kMasked : 0);
        };
        // ---- loads of this warp, ahead of its computation: the block
        // of piece l_seg, and the one after it, whose page indices are under way
        uint32_t l_seg = 0, n_seg = 0;
        int32_t n_base = 0;
        auto after = [&](uint32_t& c, int32_t& b) {
            b += 32;
            if (c < count && b >= segs[c].steps) ++c, b = 0;
        };
        auto page_of = [&](uint32_t c, int32_t k) -> int32_t {
            if (!(k & kSeen)) return 0;
            const int32_t id = p.table[int64_t(segs[c].b) * p.table_s + (k >> p.pshift)];
            if (uint32_t(id) < p.pages) return id;
            if (p.err) atomicOr(p.err, kErrPage);
            return int32_t(p.pages);
        };
        int32_t l_k = lay_out(0, int32_t(lane)), l_id = page_of(0, l_k), n_k, n_id;
        after(n_seg, n_base);
        n_k = lay_out(n_seg, n_base + int32_t(lane));
        n_id = page_of(n_seg, n_k);
        uint32_t l_todo = __ballot_sync(0xffffffffu, l_k & kSeen);  // steps of the block to load
        auto load = [&]() {  // the next step that some row sees
            while (!l_todo) {
                l_seg = n_seg;
                if (l_seg >= count) return;
                l_k = n_k, l_id = n_id;
                l_todo = __ballot_sync(0xffffffffu, l_k & kSeen);
                after(n_seg, n_base);
                n_k = lay_out(n_seg, n_base + int32_t(lane));
                n_id = page_of(n_seg, n_k);
            }
            const int32_t i = __ffs(int(l_todo)) - 1;
            l_todo &= l_todo - 1;
            const int32_t kf = __shfl_sync(0xffffffffu, l_k, i), id = __shfl_sync(0xffffffffu, l_id, i);
            const int32_t k0 = kf & ~15, in = k0 & int32_t(p.P - 1);
            const uint32_t st = filled % G::kStages, dst = ring + st * G::kStage, bar = bar0 + 8 * st;
            ++filled;
            if (!(kf & kEdge)) {
                if (lane == 0) {
                    const int32_t h = segs[l_seg].h;
                    bar_arrive_tx(bar, G::kStage);
                    tma5(dst, &kmap, bar, 0, in, 0, h, id);
                    tma5(dst + G::kHalf, &vmap, bar, 0, in, 0, h, id);
                } else {
                    bar_arrive(bar);
                }
                return;
            }
            const DecSeg& x = segs[l_seg];
            const bool there = uint32_t(id) < p.pages;
            const uint16_t* kb = p.k_pages + (there ? int64_t(id) * p.kp_ps : 0) + int64_t(x.h) * p.kp_hs;
            const uint16_t* vb = p.v_pages + (there ? int64_t(id) * p.vp_ps : 0) + int64_t(x.h) * p.vp_hs;
            const uint32_t piece = lane % PIECES;
#pragma unroll 1
            for (int i = 0; i < ITERS; ++i) {
                const int32_t row = i * RPI + int32_t(lane / PIECES), key = k0 + row;
                const bool fresh = p.fused && key >= x.f;
                const bool on = ((key < x.hi && key >= x.lo) || key < x.sink) && (fresh || there);
                const int64_t tok = int64_t(x.q0) + key - x.f;
                const uint16_t* ks = !on ? p.k_pages
                                     : fresh ? p.k_new + tok * p.kn_ts + int64_t(x.h) * p.kn_hs
                                             : kb + int64_t(in + row) * p.kp_ss;
                const uint16_t* vs = !on ? p.v_pages
                                     : fresh ? p.v_new + tok * p.vn_ts + int64_t(x.h) * p.vn_hs
                                             : vb + int64_t(in + row) * p.vp_ss;
                cp16(dst + swz<kDecKeys>(row, piece), ks + piece * 8, on);
                cp16(dst + G::kHalf + swz<kDecKeys>(row, piece), vs + piece * 8, on);
            }
            cp_arrive(bar);
        };
        uint32_t qf[KS][4];
        auto queries = [&](const DecSeg& x) {  // as A fragments; zero past the rows
            const uint16_t* q[2];
            bool on[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int32_t r = int32_t(lane >> 2) + 8 * i;
                on[i] = r < x.rows;
                q[i] = p.q + int64_t(x.q0 + (on[i] ? r / g : 0)) * p.q_ts +
                       int64_t(x.h * g + (on[i] ? r % g : 0)) * p.q_hs + (lane & 3u) * 2;
            }
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    qf[kk][i] = on[i & 1] ? *reinterpret_cast<const uint32_t*>(q[i & 1] + kk * 16 + (i >> 1) * 8) : 0u;
        };
        queries(segs[0]);  // ahead of the cache's stream
#pragma unroll 1
        for (int i = 0; ok && i < G::kStages; ++i) load();

        for (uint32_t c = 0; c < count; ++c) {
            const DecSeg& x = segs[c];
            const int32_t R = x.rows, steps = x.steps, h = x.h;
            int32_t pos[2];  // slot of the token of this lane's rows (-1: no row)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int32_t row = int32_t(lane >> 2) + 8 * i;
                pos[i] = row < R ? max(x.f + row / g, -1) : -1;
            }
            float o[2 * KS][4], m[2], l[2];
#pragma unroll
            for (int n = 0; n < 2 * KS; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
            m[0] = m[1] = -INFINITY;
            l[0] = l[1] = 0.f;

            for (int32_t block = 0; ok && block < steps; block += 32) {
                const int32_t c_k = lay_out(c, block + int32_t(lane));
                for (uint32_t todo = __ballot_sync(0xffffffffu, c_k & kSeen); todo; todo &= todo - 1) {
                    const int32_t kf = __shfl_sync(0xffffffffu, c_k, __ffs(int(todo)) - 1), k0 = kf & ~15;
                    const uint32_t st = used % G::kStages, ks = ring + st * G::kStage, vs = ks + G::kHalf;
                    const uint32_t landed = bar0 + 8 * st, phase = (used / G::kStages) & 1u;
                    ok = p.timeout_ns < kShortNs ? warp_wait_short(landed, phase, uint32_t(p.timeout_ns))
                                                 : warp_wait(landed, phase, p.timeout_ns);
                    if (!ok) break;
                    ++used;
                    // S = Q K^T
                    float sc[2][4] = {};
#pragma unroll
                    for (int kk = 0; kk < KS; ++kk) {
                        uint32_t bf[4];
                        ldsm4(bf, ks + swz<kDecKeys>((lane & 7u) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1u)));
                        T::mma(sc[0], qf[kk], bf[0], bf[1]);
                        T::mma(sc[1], qf[kk], bf[2], bf[3]);
                    }
                    if (kf & kMasked) {
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (!sees(p, pos[e >> 1], k0 + nt * 8 + int32_t(lane & 3u) * 2 + (e & 1)))
                                    sc[nt][e] = -INFINITY;
                    }
                    if (p.logits) {
                        float* lg = p.logits + ((int64_t(x.b) * p.Hkv + h) * p.wlen) * p.rows;
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int32_t row = int32_t(lane >> 2) + 8 * (e >> 1);
                                const int32_t key = k0 + nt * 8 + int32_t(lane & 3u) * 2 + (e & 1);
                                if (row < R && key < x.hi) lg[int64_t(key) * p.rows + row] = sc[nt][e] * p.c;
                            }
                    }
                    // running maximum, probabilities and sums
                    uint32_t ph[4], pl[4];
                    float nm[2], bs[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float y = fmaxf(fmaxf(sc[0][2 * i], sc[0][2 * i + 1]),
                                        fmaxf(sc[1][2 * i], sc[1][2 * i + 1]));
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 1));
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 2));
                        nm[i] = fmaxf(m[i], y);
                        bs[i] = nm[i] == -INFINITY ? 0.f : fmaf(nm[i], p.c, -T::kShift);
                    }
                    if (__any_sync(0xffffffffu, nm[0] > m[0] || nm[1] > m[1])) {
                        const float al[2] = {ex2(fmaf(m[0], p.c, -T::kShift) - bs[0]),
                                             ex2(fmaf(m[1], p.c, -T::kShift) - bs[1])};
#pragma unroll
                        for (int n = 0; n < 2 * KS; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[n][e] *= al[e >> 1];
#pragma unroll
                        for (int i = 0; i < 2; ++i) l[i] *= al[i], m[i] = nm[i];
                    }
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float a = ex2(fmaf(sc[nt][2 * i], p.c, -bs[i]));
                            const float d = ex2(fmaf(sc[nt][2 * i + 1], p.c, -bs[i]));
                            l[i] += a + d;
                            // A fragment: registers (row, row + 8) x (keys 0-7, 8-15)
                            ph[nt * 2 + i] = T::pack(a, d);
                            float ha, hd;
                            T::unpack(ph[nt * 2 + i], ha, hd);
                            pl[nt * 2 + i] = T::pack(a - ha, d - hd);
                        }
                    // O += P V. P enters as its 16-bit rounding plus the 16-bit
                    // rounding of what that leaves: the tensor cores are far from
                    // busy here, and the sum keeps about twice the bits.
#pragma unroll
                    for (int n = 0; n < KS; ++n) {
                        uint32_t vf[4];
                        ldsm4t(vf, vs + swz<kDecKeys>((lane & 7u) + (((lane >> 3) & 1u) << 3), n * 2 + (lane >> 4)));
                        T::mma(o[2 * n], ph, vf[0], vf[1]);
                        T::mma(o[2 * n + 1], ph, vf[2], vf[3]);
                        T::mma(o[2 * n], pl, vf[0], vf[1]);
                        T::mma(o[2 * n + 1], pl, vf[2], vf[3]);
                    }
                    // the new tokens' keys and values go to their slots
                    if (p.fused && (kf & kEdge) && k0 + kDecKeys > x.f) {
                        const int32_t id = p.table[int64_t(x.b) * p.table_s + (k0 >> p.pshift)];
                        const uint32_t piece = lane % PIECES;
                        if (uint32_t(id) < p.pages) {
#pragma unroll 2
                            for (int i = 0; i < ITERS; ++i) {
                                const int32_t row = i * RPI + int32_t(lane / PIECES), key = k0 + row;
                                if (key >= x.f && key < x.hi) {
                                    const int64_t at = key & int32_t(p.P - 1);
                                    const uint8_t* kk = smem + (ks - sbase) + swz<kDecKeys>(row, piece);
                                    *reinterpret_cast<uint4*>(p.k_pages + int64_t(id) * p.kp_ps + at * p.kp_ss +
                                                              int64_t(h) * p.kp_hs + piece * 8) =
                                        *reinterpret_cast<const uint4*>(kk);
                                    *reinterpret_cast<uint4*>(p.v_pages + int64_t(id) * p.vp_ps + at * p.vp_ss +
                                                              int64_t(h) * p.vp_hs + piece * 8) =
                                        *reinterpret_cast<const uint4*>(kk + G::kHalf);
                                }
                            }
                        }
                    }
                    // the stage's next contents come through the TMA's proxy: what the
                    // copies wrote is ordered before
                    if (kf & kEdge) proxy_fence();
                    __syncwarp();
                    load();
                }
            }

            // The warps' sums meet: maxima first, then the rows, those of several
            // warps at a time where they fit beside one another.
            float* const sm = reinterpret_cast<float*>(smem + G::kStat) + 32;  // [4][MR]
            float* const sl = sm + kDecWarps * MR;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float y = l[i];
                y += __shfl_xor_sync(0xffffffffu, y, 1);
                y += __shfl_xor_sync(0xffffffffu, y, 2);
                if ((lane & 3u) == 0) {
                    const uint32_t row = (lane >> 2) + 8 * i;
                    sm[warp * MR + row] = fmaf(m[i], p.c, -T::kShift);  // (the reference)
                    sl[warp * MR + row] = y;
                }
            }
            __syncthreads();
            const uint32_t side = R * 4 <= MR ? 4 : R * 2 <= MR ? 2 : 1;
            for (uint32_t turn = 0; turn < kDecWarps / side; ++turn) {
                if (warp / side == turn) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t row = (lane >> 2) + 8 * i, at = warp % side * uint32_t(R) + row;
                        if (int32_t(row) >= R) continue;
                        float mx = sm[row];
#pragma unroll
                        for (int w = 1; w < kDecWarps; ++w) mx = fmaxf(mx, sm[w * MR + row]);
                        const float f = mx == -INFINITY ? 0.f : ex2(fmaf(m[i], p.c, -T::kShift) - mx);
                        float* to = join + at * D + (lane & 3u) * 2;
#pragma unroll
                        for (int n = 0; n < 2 * KS; ++n) {
                            float2* cell = reinterpret_cast<float2*>(to + ((n * 8) ^ (at & 7u) * 8));
                            float2 v = make_float2(o[n][2 * i] * f, o[n][2 * i + 1] * f);
                            if (turn) v.x += cell->x, v.y += cell->y;
                            *cell = v;
                        }
                    }
                }
                __syncthreads();
            }
            if (c + 1 < count) queries(segs[c + 1]);
            // rows by warps, D / 32 elements of a row per lane
            constexpr int E = D / 32;
            const bool whole = x.j0 == 0 && steps == x.tiles;
            constexpr int64_t kPart = MR * (D + 2);
            float* const slot = p.part + (2 * cta + x.own) * kPart;
            auto finish = [&](int32_t row, const float (&v)[E], float mx, float sum) {
                const int32_t token = x.q0 + row / g;
                const int64_t head = h * g + row % g;
                const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
                uint16_t* out = p.out + int64_t(token) * p.o_ts + head * p.o_hs + lane * E;
                if constexpr (E == 4)
                    *reinterpret_cast<uint2*>(out) =
                        make_uint2(T::pack(v[0] * inv, v[1] * inv), T::pack(v[2] * inv, v[3] * inv));
                else
                    *reinterpret_cast<uint32_t*>(out) = T::pack(v[0] * inv, v[1] * inv);
                if (lane == 0 && p.lse)
                    p.lse[int64_t(token) * p.Hq + head] = sum == 0.f ? -INFINITY : (mx + lg2(sum)) * kLn2;
            };
            for (int32_t row = int32_t(warp); row < R; row += kDecWarps) {
                float mx = sm[row], sum = 0.f, v[E];
#pragma unroll
                for (int w = 1; w < kDecWarps; ++w) mx = fmaxf(mx, sm[w * MR + row]);
#pragma unroll
                for (int w = 0; w < kDecWarps; ++w)
                    sum = fmaf(mx == -INFINITY ? 0.f : ex2(sm[w * MR + row] - mx), sl[w * MR + row], sum);
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = 0.f;
                for (uint32_t w = 0; w < side; ++w) {
                    const uint32_t at = w * uint32_t(R) + uint32_t(row);
                    const float* from = join + at * D + ((lane * E) ^ (at & 7u) * 8);
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] += from[e];
                }
                if (whole) {
                    finish(row, v, mx, sum);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) slot[row * D + lane * E + e] = v[e];
                    if (lane == 0) slot[MR * D + row] = mx, slot[MR * D + MR + row] = sum;
                }
            }
            if (!whole) {
                const int64_t c0 = cut_owner(U, NC, x.item), c1 = cut_owner(U, NC, x.item + x.tiles - 1);
                __threadfence();
                __syncthreads();
                if (tid == 0) {
                    const bool last = atomicAdd(p.count + c0, 1u) == uint32_t(c1 - c0);
                    if (last) p.count[c0] = 0;
                    *flag = last;
                }
                __syncthreads();
                if (*flag) {
                    __threadfence();
                    const int32_t pieces = int32_t(c1 - c0) + 1;
                    const float* const p0 = p.part + (2 * c0 + (cut_begin(U, NC, c0) != x.item)) * kPart;
                    auto piece = [&](int32_t i) { return i ? p.part + 2 * (c0 + i) * kPart : p0; };
                    for (int32_t row = int32_t(warp); row < R; row += kDecWarps) {
                        float mx = -INFINITY, sum = 0.f, v[E] = {};
                        for (int32_t i0 = 0; i0 < pieces; i0 += 32) {
                            const int32_t i = i0 + int32_t(lane), n = min(32, pieces - i0);
                            const float pm = i < pieces ? __ldcg(piece(i) + MR * D + row) : -INFINITY;
                            const float ps = i < pieces ? __ldcg(piece(i) + MR * D + MR + row) : 0.f;
                            float f = 0.f;
                            for (int32_t k0 = 0; k0 < n; k0 += 8) {
                                float y[8][E];
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float* from = piece(min(i0 + k0 + k, pieces - 1)) + row * D + lane * E;
                                    using Vec = typename std::conditional<E == 4, float4, float2>::type;
                                    *reinterpret_cast<Vec*>(y[k]) = __ldcg(reinterpret_cast<const Vec*>(from));
                                }
                                if (!k0) {  // the maximum may grow with each 32 pieces
                                    float nm = pm;
#pragma unroll
                                    for (int d = 16; d; d >>= 1) nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, d));
                                    nm = fmaxf(nm, mx);
                                    const float ref = nm == -INFINITY ? 0.f : nm, old = ex2(mx - ref);
                                    f = ex2(pm - ref);
                                    sum = fmaf(f, ps, sum * old);
#pragma unroll
                                    for (int e = 0; e < E; ++e) v[e] *= old;
                                    mx = nm;
                                }
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float fk = __shfl_sync(0xffffffffu, f, (k0 + k) & 31);
                                    if (k0 + k < n)
#pragma unroll
                                        for (int e = 0; e < E; ++e) v[e] = fmaf(fk, y[k][e], v[e]);
                                }
                            }
                        }
#pragma unroll
                        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                        finish(row, v, mx, sum);
                    }
                }
            }
            __syncthreads();  // the joined sums and maxima have been read
        }
        u = segs[count - 1].item + segs[count - 1].j0 + segs[count - 1].steps;
    }
    // every load has landed before the CTA ends (they all have, unless a wait gave
    // up: a stage is filled again only after its last load was waited for, so each
    // of the rest is the one fill under way in its stage)
    for (uint32_t i = used; i != filled; ++i)
        warp_wait(bar0 + 8 * (i % G::kStages), (i / G::kStages) & 1u, kGraceNs);
    if (!ok) gave_up(p);
}

// weights[b, h, slot] from the stored logits, once the rows' lse are known.
// One thread per slot sums its rows in order. New slots start here (their old
// weight is not read); slots that no row sees keep theirs. Bound by the logits'
// way through L2: about 10 us for 16 sequences of up to 8192 slots, 32 heads
// over 8, beside 70 us of attention.
__global__ void __launch_bounds__(256) attn_weights_kernel(const AttnParams p) {
    __shared__ float lse2[256];
    __shared__ int32_t pos[256];
    after_wait();
    const uint32_t chunks = (p.wlen + 255) / 256;
    const uint32_t chunk = blockIdx.x % chunks, bh = blockIdx.x / chunks, h = bh % p.Hkv, b = bh / p.Hkv;
    const SeqRange s = load_seq(p, b);
    if (int64_t(chunk) * 256 >= s.n || !s.nq) return;
    const int32_t k = int32_t(chunk * 256 + threadIdx.x), rows = s.nq * int32_t(p.g);
    const float* lg = p.logits + (int64_t(bh) * p.wlen + k) * p.rows;
    float sum = 0.f;
    for (int32_t r0 = 0; r0 < rows; r0 += 256) {
        const int32_t r = r0 + int32_t(threadIdx.x);
        __syncthreads();
        if (r < rows) {
            const int32_t t = r / int32_t(p.g);
            lse2[threadIdx.x] = p.lse[int64_t(s.q0 + t) * p.Hq + h * p.g + r % p.g] * kLog2e;
            pos[threadIdx.x] = s.f + t;
        }
        __syncthreads();
        const int32_t end = min(256, rows - r0);
        if (k < s.n)
            for (int32_t i = 0; i < end; ++i)
                if (sees(p, pos[i], k)) sum += ex2(lg[r0 + i] - lse2[i]);
    }
    if (k < s.n) {
        float* w = p.weights + int64_t(b) * p.w_ss + int64_t(h) * p.w_hs + k;
        *w = (k >= s.f ? 0.f : *w) + sum;
    }
}

bool al16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }
constexpr uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }
constexpr uint64_t kMaxTimeoutNs = 60000000000ull;
constexpr uint64_t kTimeoutNs = 2000000000ull;

uint32_t sm_count() {
    static std::atomic<uint32_t> known[16];
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return 148;
    }
    const bool slot = dev >= 0 && dev < 16;
    if (const uint32_t n = slot ? known[dev].load(std::memory_order_relaxed) : 0) return n;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
        cudaGetLastError();
        return 148;
    }
    if (slot) known[dev].store(uint32_t(sms), std::memory_order_relaxed);
    return uint32_t(sms);
}
// Rows of a sequence and kv head beyond which the call goes to the 128-row
// tensor-core tiles of ls_attention_chunk.cu: what one 16-row MMA tile holds.
// (Two such tiles in the decode kernel: 90 us for 7 new tokens of 16 sequences
// of up to 6000 slots, 28 rows, against 63 us there.)
constexpr uint64_t kChunkRows = 16;
bool is_chunk(const ls_b200_attention_args& a) {
    const uint32_t g = a.q_heads / a.kv_heads;
    return uint64_t(a.max_q) * g > kChunkRows;
}

struct ScratchPlan {
    uint64_t count, part, lse, logits, plan, items, chunk_part, w_plan, w_items, w_part, total;
};
ScratchPlan scratch_plan(const ls_b200_attention_args& a) {
    ScratchPlan s{};
    const bool w = a.weights_length != 0;
    s.count = 0;
    s.part = up256(kMaxCtas * sizeof(uint32_t));
    if (is_chunk(a)) {
        const uint32_t g = a.q_heads / a.kv_heads;
        s.plan = s.part;
        s.items = s.plan + up256(sizeof(ChunkPlan));
        s.chunk_part = s.items + up256(chunk_items(a.tokens, a.batch, g) * sizeof(ChunkItem));
        s.w_plan = s.chunk_part + up256(2ull * sm_count() * chunk_part_floats(a.head_dim) * sizeof(float));
        s.w_items = s.w_plan + (w ? up256(sizeof(ChunkPlan)) : 0);
        s.w_part = s.w_items + (w ? up256(chunk_weight_items(a.batch, a.weights_length) * sizeof(ChunkItem)) : 0);
        s.lse = s.w_part + (w ? up256(2ull * sm_count() * 128 * sizeof(float)) : 0);
        s.total = s.lse + (w ? up256(uint64_t(a.tokens) * a.q_heads * sizeof(float)) : 0);
        return s;
    }
    s.lse = s.part + up256(2ull * kMaxCtas * 16 * (a.head_dim + 2) * sizeof(float));
    s.logits = s.lse + (w ? up256(uint64_t(a.tokens) * a.q_heads * sizeof(float)) : 0);
    s.total = s.logits + (w ? up256(uint64_t(a.batch) * a.q_heads * a.weights_length * a.max_q * sizeof(float)) : 0);
    return s;
}

// Scratch of every call of at most this batch, tokens, max_q and
// weights_length. Either layout grows with them, but a call of few rows among the
// smaller ones goes to the other one (stored logits).
uint64_t scratch_bytes(ls_b200_attention_args a) {
    uint64_t total = scratch_plan(a).total;
    const uint32_t g = a.q_heads / a.kv_heads;
    if (is_chunk(a) && g <= kChunkRows) {
        a.max_q = uint32_t(kChunkRows) / g;
        const uint64_t few = scratch_plan(a).total;
        total = few > total ? few : total;
    }
    return total;
}

bool stride8(int64_t v) { return v % 8 == 0 && v >= 0; }

// The call's shape: everything that does not depend on pointers.
int check_shape(const ls_b200_attention_args& a) {
    if (a.dtype > LS_B200_BF16 || !a.kv_heads || !a.q_heads || a.q_heads % a.kv_heads || a.q_heads / a.kv_heads > 128 ||
        a.q_heads > 65536 || (a.head_dim != 64 && a.head_dim != 128))
        return EINVAL;
    if (a.page_size < 16 || a.page_size > 256 || (a.page_size & (a.page_size - 1))) return EINVAL;
    if (uint64_t(a.table_pages) * a.page_size > kMaxSlots || a.pages > 0x7fffffffu || a.batch > (1u << 22) ||
        a.tokens > 0x7fffff00u || uint64_t(a.max_q) * (a.q_heads / a.kv_heads) > 0x3fffffffull ||
        a.weights_length > kMaxSlots || a.window > 0x7fffffffu || a.sinks > 0x7fffffffu)
        return EINVAL;
    if (!(a.scale > 0.f) || std::isinf(a.scale) || a.timeout_ns > kMaxTimeoutNs) return EINVAL;
    return 0;
}

template <class T, int D>
int launch_decode(const AttnParams& p, bool bf16, cudaStream_t s) {
    using G = GeoD<D>;
    CUtensorMap km, vm;
    const uint64_t dims[5] = {64, p.P, D / 64, p.Hkv, p.pages};
    const int64_t ks[4] = {p.kp_ss, 64, p.kp_hs, p.kp_ps}, vs[4] = {p.vp_ss, 64, p.vp_hs, p.vp_ps};
    const uint32_t box[5] = {64, uint32_t(kDecKeys), D / 64, 1, 1};
    if (!encode_map(&km, bf16, p.k_pages, 5, dims, ks, box) || !encode_map(&vm, bf16, p.v_pages, 5, dims, vs, box))
        return EINVAL;
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return int(e);
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!bit || !(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(attn_decode_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(G::kSmem));
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attn_decode_kernel<T, D>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     int(cudaSharedmemCarveoutMaxShared));
        if (e != cudaSuccess) return int(e);
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    const uint32_t grid = sm_count() * uint32_t(G::kCtas);
    attn_decode_kernel<T, D><<<grid < kMaxCtas ? grid : kMaxCtas, kDecThreads, G::kSmem, s>>>(p, km, vm);
    return int(cudaGetLastError());
}
}  // namespace
}  // namespace lsb

extern "C" {

uint64_t ls_b200_attention_scratch_bytes(const ls_b200_attention_args* a) {
    if (!a || lsb::check_shape(*a)) return 0;
    return lsb::scratch_bytes(*a);
}

int ls_b200_paged_attention(const ls_b200_attention_args* a, void* stream) {
    using namespace lsb;
    if (!a) return EINVAL;
    if (const int e = check_shape(*a)) return e;
    if (!a->batch || !a->tokens || !a->max_q) return 0;  // no new token: nothing to write
    if (!a->q || !a->output || !a->k_pages || !a->v_pages || !a->page_table || !a->q_start || !a->kv_len ||
        !a->scratch || !a->pages || !a->table_pages || (!a->k_new) != (!a->v_new) ||
        (!a->weights) != (!a->weights_length))
        return EINVAL;
    if (!al16(a->q) || !al16(a->output) || !al16(a->k_pages) || !al16(a->v_pages) || !al16(a->k_new) ||
        !al16(a->v_new) || !al16(a->scratch))
        return EINVAL;
    for (const int64_t v : {a->q_token_stride, a->q_head_stride, a->k_new_token_stride, a->k_new_head_stride,
                            a->v_new_token_stride, a->v_new_head_stride, a->output_token_stride, a->output_head_stride,
                            a->k_page_stride, a->k_slot_stride, a->k_head_stride, a->v_page_stride, a->v_slot_stride,
                            a->v_head_stride})
        if (!stride8(v)) return EINVAL;
    const ScratchPlan plan = scratch_plan(*a);
    if (a->scratch_bytes < plan.total) return ENOSPC;
    uint8_t* scratch = static_cast<uint8_t*>(a->scratch);
    AttnParams p{};
    p.q = static_cast<const uint16_t*>(a->q);
    p.k_new = static_cast<const uint16_t*>(a->k_new);
    p.v_new = static_cast<const uint16_t*>(a->v_new);
    p.k_pages = static_cast<uint16_t*>(a->k_pages);
    p.v_pages = static_cast<uint16_t*>(a->v_pages);
    p.out = static_cast<uint16_t*>(a->output);
    p.table = a->page_table;
    p.q_start = a->q_start;
    p.kv_len = a->kv_len;
    p.lse = a->lse ? a->lse : a->weights ? reinterpret_cast<float*>(scratch + plan.lse) : nullptr;
    p.weights = a->weights;
    p.part = reinterpret_cast<float*>(scratch + plan.part);
    p.count = reinterpret_cast<uint32_t*>(scratch + plan.count);
    p.logits = a->weights ? reinterpret_cast<float*>(scratch + plan.logits) : nullptr;
    p.err = a->error;
    p.q_ts = a->q_token_stride, p.q_hs = a->q_head_stride;
    p.kn_ts = a->k_new_token_stride, p.kn_hs = a->k_new_head_stride;
    p.vn_ts = a->v_new_token_stride, p.vn_hs = a->v_new_head_stride;
    p.o_ts = a->output_token_stride, p.o_hs = a->output_head_stride;
    p.kp_ps = a->k_page_stride, p.kp_ss = a->k_slot_stride, p.kp_hs = a->k_head_stride;
    p.vp_ps = a->v_page_stride, p.vp_ss = a->v_slot_stride, p.vp_hs = a->v_head_stride;
    p.table_s = a->table_stride, p.w_ss = a->weights_sequence_stride, p.w_hs = a->weights_head_stride;
    p.c = a->scale * kLog2e;
    p.B = a->batch, p.Hq = a->q_heads, p.Hkv = a->kv_heads, p.g = a->q_heads / a->kv_heads, p.D = a->head_dim;
    p.P = a->page_size, p.pages = a->pages, p.tpages = a->table_pages, p.tokens = a->tokens, p.max_q = a->max_q;
    while ((1u << p.pshift) < p.P) ++p.pshift;
    // (a window that no cache of this table fills is none)
    p.window = uint64_t(a->window) < uint64_t(a->table_pages) * a->page_size ? a->window : 0;
    p.sinks = a->sinks, p.wlen = a->weights_length;
    p.rows = p.max_q * p.g;
    p.timeout_ns = a->timeout_ns ? a->timeout_ns : kTimeoutNs;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (is_chunk(*a)) {
        const ChunkScratch c{reinterpret_cast<ChunkPlan*>(scratch + plan.plan),
                             reinterpret_cast<ChunkItem*>(scratch + plan.items),
                             reinterpret_cast<float*>(scratch + plan.chunk_part),
                             reinterpret_cast<ChunkPlan*>(scratch + plan.w_plan),
                             reinterpret_cast<ChunkItem*>(scratch + plan.w_items),
                             reinterpret_cast<float*>(scratch + plan.w_part)};
        return launch_chunk(p, a->dtype, c, sm_count(), s);
    }
    p.fused = p.k_new != nullptr;
    const bool bf16 = a->dtype == LS_B200_BF16;
    const int rc = p.D == 64 ? (bf16 ? launch_decode<BF16, 64>(p, true, s) : launch_decode<F16, 64>(p, false, s))
                             : (bf16 ? launch_decode<BF16, 128>(p, true, s) : launch_decode<F16, 128>(p, false, s));
    if (rc || !p.weights) return rc;
    return int(launch_after(attn_weights_kernel, p.B * p.Hkv * ((p.wlen + 255) / 256), 256, 0, s, p));
}

}  // extern "C"
