// Internal types of the paged-cache attention (ls_attention.cu), of the append
// (ls_append.cu) and of the cache eviction (ls_evict.cu). Not part of the public ABI.
#pragma once
#include <cuda.h>
#include <stdint.h>
#include <cuda_runtime.h>
#include "../../include/leanstream_b200.h"

namespace lsb {

constexpr uint32_t kErrLength = 1u << 1;  // a sequence's lengths do not fit the call
constexpr uint32_t kErrPage = 1u << 2;    // a visible slot's page index is outside the pool

constexpr uint32_t kMaxSlots = 0x7fff0000u;  // of a sequence: a tile past the last slot still counts in 32 bits

// The cache in 8 bits: slots that share an exponent, and the exponent of a block
// with a value that is not finite (it reads as NaN).
constexpr int kBlockShift = 4, kBlock = 1 << kBlockShift;
constexpr int32_t kNoExponent = -128;
static_assert(kBlock == LS_B200_CACHE_BLOCK, "public block size");

// ls_b200_attention_args in the kernels' units. Strides are in elements.
struct AttnParams {
    const uint16_t* q;
    const uint16_t* k_new;
    const uint16_t* v_new;
    uint16_t* k_pages;
    uint16_t* v_pages;
    uint16_t* out;
    const int32_t* table;
    const int32_t* q_start;
    const int32_t* kv_len;
    float* lse;       // [tokens][Hq]: the caller's, or scratch where only the weights need it
    float* weights;
    float* part;      // partial results of split items
    uint32_t* count;  // [grid] arrived pieces of the item that begins in a CTA (zero at rest)
    float* logits;    // [B][Hkv][wlen][rows] base-2 logits of a call with weights
    uint32_t* err;
    int64_t q_ts, q_hs, kn_ts, kn_hs, vn_ts, vn_hs, o_ts, o_hs;
    int64_t kp_ps, kp_ss, kp_hs, vp_ps, vp_ss, vp_hs;
    int64_t table_s, w_ss, w_hs;
    const uint8_t* ex;  // a cache in 8 bits: its exponents (keys, values of a block side by side)
    int64_t ex_ps, ex_hs;
    float c;  // scale * log2(e)
    uint32_t B, Hq, Hkv, g, D, P, pshift, pages, tpages, tokens, max_q, window, sinks, wlen;
    uint32_t rows;   // max_q * g: row capacity of `logits`
    uint32_t fused;  // 1: the attention kernel appends the new keys and values
    uint64_t timeout_ns;
};

// The tensor-core path of chunks (ls_attention_chunk.cu): one item is two
// 128-row tiles of one kv head, a row being a (token, head of the group).
constexpr uint32_t kMaxCtas = 512;  // CTAs of a launch, and counters in the scratch header
constexpr int kChunkKeys = 128;     // slots of a tile
struct ChunkItem {                  // written by the plan kernel
    int32_t b, q0, nq, n;           // the sequence, as SeqRange
    int32_t t0, tiles;              // attention: first token, tiles of slots; weights: first slot, row tiles
    int64_t units;                  // tiles of the items before, over all kv heads
};
struct ChunkPlan {
    int64_t units;                  // tiles of the call
    int32_t items, ctas;            // items; CTAs that share the tiles
    int32_t start[kMaxCtas];        // item in which each CTA begins
    int2 open[kMaxCtas];            // item and kv head that begin in a CTA and go on in the next (x < 0: none)
};
struct ChunkScratch {
    ChunkPlan* plan;
    ChunkItem* items;
    float* part;
    ChunkPlan* w_plan;  // of the weights
    ChunkItem* w_items;
    float* w_part;      // [2 * CTAs][128]
};
__host__ __device__ inline uint32_t chunk_tokens(uint32_t g) { return 128 / g; }  // of one 128-row tile
__host__ __device__ inline uint64_t chunk_items(uint64_t tokens, uint64_t batch, uint32_t g) {
    return tokens / (2 * chunk_tokens(g)) + batch;
}
__host__ __device__ inline uint64_t chunk_weight_items(uint64_t batch, uint64_t wlen) {
    return batch * (wlen / kChunkKeys + 2);
}
inline uint64_t chunk_part_floats(uint32_t D) { return 256ull * (D + 2); }  // one partial result
// A tensor map of 16-bit elements with 128-byte swizzle; strides in elements,
// from the second dimension on. False when the driver refuses it.
bool encode_map(CUtensorMap* map, bool bf16, const void* base, uint32_t rank, const uint64_t* dims,
                const int64_t* strides, const uint32_t* box);
// One of codes: boxes of `slots` rows of a head, rows of D bytes in its swizzle.
bool encode_codes(CUtensorMap* map, const void* base, const AttnParams& p, int64_t ss, int64_t hs, int64_t ps,
                  uint32_t slots);
uint32_t sm_count();  // of the current device
// Few rows of a kv head over a cache in 8 bits (ls_attention8.cu).
constexpr uint32_t kMaxRows8 = 32;
int launch_decode8(const AttnParams& p, uint32_t dtype, cudaStream_t stream);
int launch_chunk(const AttnParams& p, uint32_t dtype, const ChunkScratch& s, uint32_t sms, cudaStream_t stream);

// A sequence of the call: its new tokens are rows q0 .. q0 + nq - 1 of q and
// take cache slots f .. n - 1. Row t sees the slots k <= f + t that its window
// leaves; f < 0 (more tokens than slots) leaves the first rows empty.
struct SeqRange {
    int32_t q0, nq, n, f;
};

__device__ __forceinline__ SeqRange load_seq(const AttnParams& p, uint32_t b) {
    SeqRange s;
    s.q0 = p.q_start[b];
    s.nq = p.q_start[b + 1] - s.q0;
    s.n = p.kv_len[b];
    const bool ok = s.q0 >= 0 && s.nq >= 0 && uint32_t(s.nq) <= p.max_q && uint32_t(s.q0) <= p.tokens &&
                    uint32_t(s.nq) <= p.tokens - uint32_t(s.q0) && s.n >= 0 &&
                    uint64_t(s.n) <= uint64_t(p.tpages) << p.pshift && (!p.weights || uint32_t(s.n) <= p.wlen);
    if (!ok) {
        if (p.err) atomicOr(p.err, kErrLength);
        s.q0 = s.nq = s.n = 0;
    }
    s.f = s.n - s.nq;
    return s;
}

// The cache slots that the rows of tokens [t0, t1) see between them: [0, sink)
// and [lo, hi), cut into tiles of TK slots: `ns` tiles of the first slots, then
// the tiles from `first`. Rows without any visible slot keep one (empty) tile,
// so that somebody writes their output.
struct KeyRange {
    int32_t lo, hi, sink, ns, first, tiles;
};

template <int TK>
__device__ __forceinline__ KeyRange key_range(const AttnParams& p, const SeqRange& s, int32_t t0, int32_t t1) {
    KeyRange r;
    r.hi = max(0, s.f + t1);
    r.lo = p.window ? max(0, int32_t(max(int64_t(s.f) + t0 + 1 - int64_t(p.window), int64_t(0)))) : 0;
    r.lo = min(r.lo, r.hi);
    r.sink = int32_t(min(p.window ? p.sinks : 0u, uint32_t(r.lo)));
    r.ns = (r.sink + TK - 1) / TK;
    r.first = max(r.lo / TK, r.ns);
    r.tiles = max(1, r.ns + max(0, (r.hi + TK - 1) / TK - r.first));
    return r;
}

__device__ __forceinline__ int32_t tile_at(const KeyRange& r, int32_t j) { return j < r.ns ? j : r.first + j - r.ns; }

// The row tiles (of chunk_tokens tokens) with a token that sees one of the 128
// slots from k0.
struct RowTiles {
    int32_t begin, end;
};
__device__ __forceinline__ RowTiles row_tiles(const AttnParams& p, const SeqRange& s, int32_t k0) {
    const int32_t T = int32_t(chunk_tokens(p.g)), t_lo = max(0, k0 - s.f);
    int32_t t_hi = s.nq;
    if (p.window && uint32_t(k0) >= p.sinks)
        t_hi = int32_t(max(int64_t(0), min(int64_t(s.nq), int64_t(k0) + kChunkKeys - 1 + p.window - s.f)));
    const int32_t begin = t_lo / T;
    return {begin, t_lo < t_hi ? (t_hi + T - 1) / T : begin};
}

// A wait of this warp gave up.
__device__ __forceinline__ void gave_up(const AttnParams& p) {
    if ((threadIdx.x & 31u) == 0 && p.err) atomicOr(p.err, uint32_t(LS_B200_ATTN_TIMEOUT));
}

// Whether position pos sees slot k (pos < 0: nothing).
__device__ __forceinline__ bool sees(const AttnParams& p, int32_t pos, int32_t k) {
    return k <= pos && (!p.window || int64_t(k) > int64_t(pos) - int64_t(p.window) || uint32_t(k) < p.sinks);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float two_to(int32_t e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLog2e = 1.44269504088896341f;

// The 16-bit element types: conversions and the pair forms the MMAs take.
// A probability enters its MMA relative to a reference of its row, times 2^kShift:
// float16 ends at 2^-24, so the row's largest is put near its upper end. The decode
// kernel's reference is the running maximum. The chunk kernel raises its own when
// the maximum has grown by 2^kRaise, and takes 2^kChunkShift. The largest is at most
// 2^15 in both; what rounds to zero is below 2^-40, or 2^-32, of the row's largest.
// (kRaise 4 and kChunkShift 11: 273 -> 296 us for 2048 tokens over 8192 slots, 32
// heads of 128, with logits of deviation 4, whose maxima grow often.)
// kLowest to kHighest: exponents of a cache in 8 bits that the type holds with any code.
struct F16 {
    static constexpr uint32_t kUmmaFormat = 0;
    static constexpr int32_t kLowest = -24, kHighest = 9;
    static constexpr float kShift = 15.f, kRaise = 8.f, kChunkShift = 7.f;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ void unpack(uint32_t v, float& lo, float& hi) {
        asm("{.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;}"
            : "=f"(lo), "=f"(hi) : "r"(v));
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
struct BF16 {  // (the exponents of 32-bit numbers)
    static constexpr uint32_t kUmmaFormat = 1;
    static constexpr int32_t kLowest = -126, kHighest = 120;
    static constexpr float kShift = 0.f, kRaise = 8.f, kChunkShift = 0.f;
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ void unpack(uint32_t v, float& lo, float& hi) {
        lo = __uint_as_float(v << 16);
        hi = __uint_as_float(v & 0xffff0000u);
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// First unit of CTA c when U units are cut evenly over G CTAs, and the CTA of a unit.
__device__ __forceinline__ int64_t cut_begin(int64_t U, int64_t G, int64_t c) { return c * U / G; }
__device__ __forceinline__ int64_t cut_owner(int64_t U, int64_t G, int64_t u) { return ((u + 1) * G - 1) / U; }

// The pieces of items that a CTA works on, in order.
// Each (item, kv head) counts as kItemCost tiles more than it has: its start,
// its end and its masked tiles. With 0, 1, 2 and 4 the attention of 2 x 1024 new
// tokens took 141, 139, 135, 135 us, and its weights with 0, 2, 4 85, 71, 69.
constexpr int kItemCost = 2;
struct Walk {
    int64_t U, G, u, u_begin, u_end;
    int64_t item;  // first unit of (item, kv head)
    int32_t i, h, j0, steps, taken;
    ChunkItem it;
    __device__ bool begin(const ChunkPlan* plan) {
        U = plan->units;
        G = plan->ctas;
        if (int64_t(blockIdx.x) >= G || !U) return false;
        u = u_begin = cut_begin(U, G, blockIdx.x);
        u_end = cut_begin(U, G, blockIdx.x + 1);
        i = plan->start[blockIdx.x] - 1;
        it.units = it.tiles = taken = 0;
        return true;
    }
    __device__ bool next(const AttnParams& p, const ChunkPlan* plan, const ChunkItem* items) {
        do {
            u += taken;
            if (u >= u_end) return false;
            while (u >= it.units + int64_t(it.tiles + kItemCost) * p.Hkv || !it.tiles) {
                if (++i >= plan->items) return false;
                it = items[i];
            }
            h = int32_t((u - it.units) / (it.tiles + kItemCost));
            item = it.units + int64_t(h) * (it.tiles + kItemCost);
            j0 = int32_t(u - item);
            taken = int32_t(min(u_end, item + it.tiles + kItemCost) - u);
            steps = min(taken, it.tiles - j0);
        } while (steps <= 0);
        return true;
    }
};

}  // namespace lsb
