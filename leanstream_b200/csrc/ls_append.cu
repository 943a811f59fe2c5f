// New keys and values into a paged cache, in 16 or 8 bits, with the position
// rotation on the way; the queries are rotated by the same call.
//
// Rotation of the first r elements of a head by the angles of its position,
// with pairs (i, i + r / 2), or (2 i, 2 i + 1) where interleaved:
//     x_a' = x_a cos - x_b sin,   x_b' = x_b cos + x_a sin,
// in 32 bits, each product and sum rounded by itself, and one rounding to 16
// bits at the end (none before the 8-bit codes are formed).
//
// The cache in 8 bits: a value is code * 2^e, the code a whole number of
// [-127, 127], e one exponent for the 16 slots of a block, kv head, and keys or
// values. e is the smallest with max |x| <= 127 * 2^e, so that a code is off by
// at most half a step 2^e. A block that grows by later tokens keeps the larger of
// its exponent and theirs; where that is theirs, its older codes are rounded to
// the new step, which doubles at least, so that an old row's errors add up to
// less than one step (1/2 + 1/4 + ...). Powers of two, because then a value is
// exact in the 16-bit operand of a matrix instruction (scales of any size would
// cost the attention a rounding, or two products a logit) and a block grows by a
// shift; a step is up to twice as wide for that.
//
// Bound by memory, queries in and out, keys and values in, rows out, and by its
// latency: 4096 tokens with 32 query heads of 128 over 8 into 16-bit pages (103 MB) take
// 22 us, 4.7 TB/s; four prompts' chunks of up to 900 tokens into codes 25 us; one token 3.8.
#include <stdint.h>

#include <cerrno>

#include "ls_attention.h"
#include "ls_tc.h"

namespace lsb {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
// Heads that a warp has under way, and CTAs per SM: with 4 and 3 (80 registers, spilled)
// 4096 tokens take 23.3 us, with 2 and 3 24.7, 2 and 4 24.1, with these 22.1.
constexpr int kHeads = 4;
constexpr int kCtasPerSm = 2;
constexpr uint32_t kMaxTokens = 1u << 27;  // blocks of 256 sequences count in 32 bits, even of overlapping ones

struct AppendParams {
    const uint16_t* q;
    const uint16_t* k_new;
    const uint16_t* v_new;
    uint16_t* q_out;
    void* k_pages;
    void* v_pages;
    int8_t* exponents;
    const int32_t* table;
    const int32_t* q_start;
    const int32_t* kv_len;
    const int32_t* positions;
    const float* cos_sin;
    uint32_t* err;
    int64_t q_ts, q_hs, qo_ts, qo_hs, kn_ts, kn_hs, vn_ts, vn_hs;
    int64_t kp_ps, kp_ss, kp_hs, vp_ps, vp_ss, vp_hs, ex_ps, ex_hs, table_s, cs_s;
    uint32_t B, Hq, Hkv, P, pshift, pages, tpages, tokens, rotary, angles;
    uint32_t interleaved;
    uint32_t per_task, splits;      // heads of a task, and tasks that share a block's rows
    int32_t lowest, highest;        // exponents that the 16-bit type holds exactly
};

// An item: up to 16 new tokens of a sequence whose slots lie in one block.
struct Rows {
    int32_t b, block;
    int32_t token, slot, n;  // first row of q, its slot, rows
    bool fresh;              // the block holds no older row of the sequence
};

__device__ __forceinline__ SeqRange append_seq(const AppendParams& p, uint32_t b) {
    SeqRange s;
    s.q0 = p.q_start[b];
    s.nq = p.q_start[b + 1] - s.q0;
    s.n = p.kv_len[b];
    const bool ok = s.q0 >= 0 && s.nq >= 0 && uint32_t(s.q0) <= p.tokens &&
                    uint32_t(s.nq) <= p.tokens - uint32_t(s.q0) && s.n >= 0 &&
                    uint64_t(s.n) <= uint64_t(p.tpages) << p.pshift;
    if (!ok) {
        if (p.err) atomicOr(p.err, kErrLength);
        s.q0 = s.nq = s.n = 0;
    }
    s.f = s.n - s.nq;
    return s;
}

// A lane's 16 elements of a head: pieces (of 8) a and b, laid out so that the
// pairs of the rotation meet in one lane. lane i of a row: pieces (i, i + r / 16)
// while i < r / 16 (halves), else (2 i, 2 i + 1).
template <int D>
struct Lane {
    static constexpr int kPerRow = D / 16, kRows = 32 / kPerRow, kIters = kBlock / kRows;
    uint32_t row, i;
    int32_t a, b;  // elements
    bool turned;
    __device__ Lane(uint32_t lane, uint32_t rotary, bool interleaved) : row(lane / kPerRow), i(lane % kPerRow) {
        turned = i * 16 < rotary;
        const bool halves = turned && !interleaved;
        a = int32_t(halves ? i * 8 : i * 16);
        b = int32_t(halves ? i * 8 + rotary / 2 : i * 16 + 8);
    }
};

template <class T>
__device__ __forceinline__ void widen(const uint4& v, float* x) {
    T::unpack(v.x, x[0], x[1]);
    T::unpack(v.y, x[2], x[3]);
    T::unpack(v.z, x[4], x[5]);
    T::unpack(v.w, x[6], x[7]);
}
template <class T>
__device__ __forceinline__ uint4 narrow(const float* x) {
    return make_uint4(T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7]));
}

// Angles of a lane's eight pairs. (Scalar products: the packed ones of two pairs come
// out fused with the sums.)
struct Turn {
    float c[8], s[8];
    __device__ __forceinline__ void load(const float* row, uint32_t i, uint32_t half) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            *reinterpret_cast<float4*>(c + e) = *reinterpret_cast<const float4*>(row + i * 8 + e);
            *reinterpret_cast<float4*>(s + e) = *reinterpret_cast<const float4*>(row + half + i * 8 + e);
        }
    }
    template <int step, int next>  // from a pair's first to its second, and to the next pair
    __device__ __forceinline__ void pairs(float* x) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = x[next * e], b = x[next * e + step];
            x[next * e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
            x[next * e + step] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
        }
    }
    __device__ __forceinline__ void apply(float* x, bool interleaved) const {  // x: pieces a and b
        if (interleaved) pairs<1, 2>(x);
        else pairs<8, 1>(x);
    }
};

// Row of the angles for a token, or -1 (reported) where its position has none.
__device__ __forceinline__ int32_t angle_row(const AppendParams& p, int32_t token, int32_t slot) {
    if (!p.cos_sin) return 0;
    const int32_t at = p.positions ? p.positions[token] : slot;
    if (uint32_t(at) < p.angles) return at;
    if (p.err && (p.positions || slot >= 0)) atomicOr(p.err, uint32_t(LS_B200_ATTN_POSITION));
    return -1;
}

// Four numbers, of at most 127 units of 1 / inv, to codes: x inv + 1.5 * 2^23 ends in
// the nearest whole number's low byte (inv is a power of two: one rounding).
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
    uint32_t v[4], lo, hi, r;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(fmaf(x[e], inv, 12582912.f));
    asm("prmt.b32 %0, %1, %2, 0x0040;" : "=r"(lo) : "r"(v[0]), "r"(v[1]));
    asm("prmt.b32 %0, %1, %2, 0x0040;" : "=r"(hi) : "r"(v[2]), "r"(v[3]));
    asm("prmt.b32 %0, %1, %2, 0x5410;" : "=r"(r) : "r"(lo), "r"(hi));
    return r;
}

// Where the rows of a task come from and go to: queries, or keys or values in 16 bits.
struct Heads {
    const uint16_t* from;  // of head 0
    uint16_t* to;
    int64_t from_ts, from_hs, to_ts, to_hs;
    uint32_t heads;
    bool turned;
};

// kHeads heads at a time, from head0 to head1 - 1, of the rows it0 * kRows .. of a
// task: a row's angles are read once for them.
template <class T, int D>
__device__ __forceinline__ void move_rows(const AppendParams& p, const Rows& t, const Heads& w, int32_t to_row,
                                          uint32_t head0, uint32_t head1, int32_t it) {
    const Lane<D> at(threadIdx.x & 31u, w.turned ? p.rotary : 0, p.interleaved);
    const int32_t r = it * Lane<D>::kRows + int32_t(at.row);
    if (r >= t.n) return;
    const int64_t token = t.token + r;
    const uint16_t* from = w.from + token * w.from_ts;
    uint16_t* to = w.to + int64_t(to_row + r) * w.to_ts;
    int32_t angle = 0;
    Turn turn;
    for (uint32_t h = head0; h < head1; h += kHeads) {
        uint4 a[kHeads], b[kHeads];
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            const uint16_t* row = from + int64_t(min(h + i, head1 - 1)) * w.from_hs;
            a[i] = *reinterpret_cast<const uint4*>(row + at.a);
            b[i] = *reinterpret_cast<const uint4*>(row + at.b);
        }
        if (h == head0) {
            angle = angle_row(p, int32_t(token), t.slot + r);
            if (angle >= 0 && at.turned) turn.load(p.cos_sin + int64_t(angle) * p.cs_s, at.i, p.rotary / 2);
        }
        if (angle < 0) return;
#pragma unroll
        for (int i = 0; i < kHeads; ++i) {
            if (h + i >= head1) break;
            if (at.turned) {
                float x[16];
                widen<T>(a[i], x);
                widen<T>(b[i], x + 8);
                turn.apply(x, p.interleaved);
                a[i] = narrow<T>(x);
                b[i] = narrow<T>(x + 8);
            }
            uint16_t* row = to + int64_t(h + i) * w.to_hs;
            *reinterpret_cast<uint4*>(row + at.a) = a[i];
            *reinterpret_cast<uint4*>(row + at.b) = b[i];
        }
    }
}

// Page of a task's block; -1 where it has none (no slot, or reported).
__device__ __forceinline__ int32_t page_of(const AppendParams& p, const Rows& t) {
    if (t.slot + t.n <= 0) return -1;
    const int32_t id = p.table[int64_t(t.b) * p.table_s + ((t.block * kBlock) >> p.pshift)];
    if (uint32_t(id) < p.pages) return id;
    if ((threadIdx.x & 31u) == 0 && p.err) atomicOr(p.err, kErrPage);
    return -1;
}

// Keys (VALUES false) or values of one kv head into a block of codes. The rows stay in
// registers as they come, all of them under way at a time, and are rotated twice, for
// the largest value and for the codes: kept in 32 bits they take 172 registers, one CTA
// per SM (33 us for four prompts' chunks, where this takes 25).
template <class T, int D, bool VALUES>
__device__ __forceinline__ void append_codes(const AppendParams& p, const Rows& t, int32_t h) {
    const uint32_t lane = threadIdx.x & 31u;
    const Lane<D> at(lane, VALUES ? 0 : p.rotary, p.interleaved);
    constexpr int R = Lane<D>::kRows, N = Lane<D>::kIters;
    const uint16_t* from = (VALUES ? p.v_new + int64_t(h) * p.vn_hs : p.k_new + int64_t(h) * p.kn_hs) +
                           int64_t(t.token + int32_t(at.row)) * (VALUES ? p.vn_ts : p.kn_ts);
    const int64_t from_s = R * (VALUES ? p.vn_ts : p.kn_ts);
    uint4 a[N], b[N];
    int32_t angle[N];  // -1: no row
#pragma unroll
    for (int it = 0; it < N; ++it) {
        const int32_t r = it * R + int32_t(at.row);
        angle[it] = -1;
        if (r < t.n && t.slot + r >= 0) {
            a[it] = *reinterpret_cast<const uint4*>(from + it * from_s + at.a);
            b[it] = *reinterpret_cast<const uint4*>(from + it * from_s + at.b);
            angle[it] = angle_row(p, t.token + r, t.slot + r);
        }
    }
    const int32_t id = page_of(p, t);
    if (id < 0) return;
    auto row_of = [&](int it, float* x) {
        // (or the compiler keeps the first pass's numbers for the second)
        asm volatile("" : "+r"(a[it].x), "+r"(a[it].y), "+r"(a[it].z), "+r"(a[it].w));
        asm volatile("" : "+r"(b[it].x), "+r"(b[it].y), "+r"(b[it].z), "+r"(b[it].w));
        widen<T>(a[it], x);
        widen<T>(b[it], x + 8);
        if (!VALUES && at.turned) {
            Turn turn;
            turn.load(p.cos_sin + int64_t(angle[it]) * p.cs_s, at.i, p.rotary / 2);
            turn.apply(x, p.interleaved);
        }
    };
    const int32_t in = (t.block * kBlock) & int32_t(p.P - 1), skip = t.slot - t.block * kBlock;
    int8_t* to = VALUES ? static_cast<int8_t*>(p.v_pages) + int64_t(id) * p.vp_ps + int64_t(h) * p.vp_hs
                        : static_cast<int8_t*>(p.k_pages) + int64_t(id) * p.kp_ps + int64_t(h) * p.kp_hs;
    const int64_t to_s = VALUES ? p.vp_ss : p.kp_ss;
    int8_t* ex = p.exponents + int64_t(id) * p.ex_ps + int64_t(h) * p.ex_hs + (in / kBlock) * 2 + VALUES;
    const int32_t was = t.fresh ? p.lowest : *ex;
    float largest = 0.f;  // NaN where one is
    bool any = false;
#pragma unroll
    for (int it = 0; it < N; ++it) {
        if (angle[it] < 0) continue;
        any = true;
        float x[16];
        row_of(it, x);
#pragma unroll
        for (int e = 0; e < 16; e += 2) largest = tc::max3(largest, fabsf(x[e]), fabsf(x[e + 1]));
    }
    if (!__any_sync(0xffffffffu, any)) return;
    // as bits they keep their order, infinities and NaN above every number
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(largest) & 0x7fffffffu);
    const bool bad = top >= 0x7f800000u || was == kNoExponent;
    // 127 = 1.984375 * 2^6 (numbers below 2^-126 only meet the lowest exponent)
    int32_t e = int32_t(top >> 23) - 127 - 6 + ((top & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    e = max(min(max(e, p.lowest), p.highest), was);
    if (!bad && !t.fresh && e > was) {
        // older rows to the new step, 16 bytes per lane and row
        constexpr uint32_t kPieces = D / 16;
        const float shift = two_to(max(was - e, -100));
        for (int32_t r = int32_t(lane / kPieces); r < skip; r += 32 / int32_t(kPieces)) {
            uint4* cell = reinterpret_cast<uint4*>(to + int64_t(in + r) * to_s + (lane % kPieces) * 16);
            uint4 v = *cell;
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                float c[4];
#pragma unroll
                for (int z = 0; z < 4; ++z) c[z] = float(int8_t(w[y] >> (8 * z)));
                w[y] = codes4(c, shift);
            }
            *cell = v;
        }
    }
    const float inv = two_to(-e);
    const bool beyond = !bad && __uint_as_float(top) > 127.f * two_to(min(e, 120));  // (of the largest exponent)
#pragma unroll
    for (int it = 0; it < N; ++it) {
        if (angle[it] < 0) continue;
        float x[16];
        row_of(it, x);
        if (bad || beyond) {
            const float most = bad ? 0.f : 127.f * two_to(e);
#pragma unroll
            for (int y = 0; y < 16; ++y) x[y] = bad ? 0.f : fminf(fmaxf(x[y], -most), most);
        }
        int8_t* row = to + int64_t(in + skip + it * R + int32_t(at.row)) * to_s;
        *reinterpret_cast<uint2*>(row + at.a) = make_uint2(codes4(x, inv), codes4(x + 4, inv));
        *reinterpret_cast<uint2*>(row + at.b) = make_uint2(codes4(x + 8, inv), codes4(x + 12, inv));
    }
    if (lane == 0) *ex = int8_t(bad ? kNoExponent : e);
}

template <class T, int D, bool Q8>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) append_kernel(const AppendParams p) {
    __shared__ int32_t first[kThreads + 1];  // items before each sequence of the batch piece
    __shared__ int32_t sums[kWarps];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // tasks of an item: keys, values (codes: a head each; else groups of heads as the
    // queries), queries
    const uint32_t groups = (p.Hkv + p.per_task - 1) / p.per_task;
    const uint32_t k_tasks = Q8 ? p.Hkv : groups * p.splits;
    const int64_t tasks = 2 * int64_t(k_tasks) + (p.Hq + p.per_task - 1) / p.per_task * p.splits;
    const uint32_t period = max(1u, gridDim.x * kWarps / uint32_t(tasks));
    tc::after_wait();
    tc::after_start();
    int64_t base = 0, task = int64_t(blockIdx.x) * kWarps + warp;
    for (uint32_t b0 = 0; b0 < p.B; b0 += kThreads) {
        SeqRange s{0, 0, 0, 0};
        if (b0 + tid < p.B) s = append_seq(p, b0 + tid);
        // blocks that hold a new token's slot (slots below 0, of rows that see nothing, have blocks too)
        const int32_t count = s.nq ? ((s.n - 1) >> kBlockShift) - (s.f >> kBlockShift) + 1 : 0;
        int32_t inc = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t x = __shfl_up_sync(0xffffffffu, inc, o);
            if (int(lane) >= o) inc += x;
        }
        if (lane == 31) sums[warp] = inc;
        __syncthreads();
        int32_t before = inc - count, total = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        first[tid] = before;
        if (tid == 0) first[kThreads] = total;
        __syncthreads();
        for (; task < (base + total) * tasks; task += int64_t(gridDim.x) * kWarps) {
            const int32_t item = int32_t(task / tasks - base);
            // (a warp's next task lies about `period` items on: there the kinds go backwards, so
            // that codes, which take longest, and queries fall to the same warps)
            const uint32_t at = uint32_t(task - (base + item) * tasks);
            const uint32_t kind = uint32_t(item) / period & 1u ? uint32_t(tasks) - 1 - at : at;
            uint32_t lo = 0, hi = kThreads;  // the sequence: first[lo] <= item < first[lo + 1]
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (first[mid] <= item) lo = mid;
                else hi = mid;
            }
            Rows t;
            t.b = int32_t(b0 + lo);
            const SeqRange q = append_seq(p, b0 + lo);
            t.block = (q.f >> kBlockShift) + item - first[lo];
            const int32_t start = t.block * kBlock;
            t.slot = max(q.f, start);
            t.n = min(q.n, start + kBlock) - t.slot;
            t.token = q.q0 + t.slot - q.f;
            t.fresh = q.f <= start;
            if (Q8 && kind < 2 * k_tasks) {
                if (kind < k_tasks) append_codes<T, D, false>(p, t, int32_t(kind));
                else append_codes<T, D, true>(p, t, int32_t(kind - k_tasks));
                continue;
            }
            Heads w;
            uint32_t part = kind;
            int32_t to_row = t.token;
            if (kind < 2 * k_tasks) {
                const bool values = kind >= k_tasks;
                const int32_t id = page_of(p, t);
                if (id < 0) continue;
                // (rows at slots below 0 come before the block's first: none of it)
                to_row = t.slot & int32_t(p.P - 1);
                w.from = values ? p.v_new : p.k_new;
                w.from_ts = values ? p.vn_ts : p.kn_ts, w.from_hs = values ? p.vn_hs : p.kn_hs;
                w.to = static_cast<uint16_t*>(values ? p.v_pages : p.k_pages) +
                       int64_t(id) * (values ? p.vp_ps : p.kp_ps);
                w.to_ts = values ? p.vp_ss : p.kp_ss, w.to_hs = values ? p.vp_hs : p.kp_hs;
                w.heads = p.Hkv, w.turned = !values;
                if (values) part -= k_tasks;
            } else {
                w.from = p.q, w.from_ts = p.q_ts, w.from_hs = p.q_hs;
                w.to = p.q_out, w.to_ts = p.qo_ts, w.to_hs = p.qo_hs;
                w.heads = p.Hq, w.turned = true;
                part -= 2 * k_tasks;
            }
            const uint32_t head0 = part / p.splits * p.per_task, head1 = min(head0 + p.per_task, w.heads);
            for (int32_t it = int32_t(part % p.splits); it * Lane<D>::kRows < t.n; it += int32_t(p.splits))
                move_rows<T, D>(p, t, w, to_row, head0, head1, it);
        }
        base += total;
        __syncthreads();  // the counts have been read
    }
}

template <class T, int D>
int launch_append(const AppendParams& p, bool int8, uint32_t grid, cudaStream_t s) {
    return int(tc::launch_after(int8 ? append_kernel<T, D, true> : append_kernel<T, D, false>, grid, kThreads, 0, s,
                                p));
}

}  // namespace
}  // namespace lsb

extern "C" int ls_b200_append_cache(const ls_b200_append_args* a, void* stream) {
    using namespace lsb;
    if (!a || a->dtype > LS_B200_BF16 || (a->cache_dtype != a->dtype && a->cache_dtype != LS_B200_INT8) ||
        !a->kv_heads || a->kv_heads > 65536 || a->q_heads > 65536 || (a->head_dim != 64 && a->head_dim != 128) ||
        a->page_size < 16 || a->page_size > 256 || (a->page_size & (a->page_size - 1)) || a->batch > (1u << 22) ||
        uint64_t(a->table_pages) * a->page_size > kMaxSlots || a->pages > 0x7fffffffu || a->tokens > kMaxTokens ||
        a->interleaved > 1 || a->reserved)
        return EINVAL;
    const bool int8 = a->cache_dtype == LS_B200_INT8;
    if (a->rotary_dim % 16 || a->rotary_dim > a->head_dim || a->angles > 0x7fffffffu) return EINVAL;
    if (!a->batch || !a->tokens) return 0;  // (an empty tensor's address may be NULL)
    if (a->cos_sin ? !a->rotary_dim || !a->angles : a->rotary_dim || a->positions || a->q) return EINVAL;
    if ((!a->q) != (!a->q_out) || (!a->q) != (!a->q_heads)) return EINVAL;
    if (!a->k_new || !a->v_new || !a->k_pages || !a->v_pages || !a->page_table || !a->q_start || !a->kv_len ||
        !a->pages || !a->table_pages || int8 != (a->exponents != nullptr))
        return EINVAL;
    for (const void* x : {a->q, static_cast<const void*>(a->q_out), a->k_new, a->v_new,
                          static_cast<const void*>(a->k_pages), static_cast<const void*>(a->v_pages),
                          static_cast<const void*>(a->cos_sin)})
        if (reinterpret_cast<uintptr_t>(x) & 15u) return EINVAL;
    if (reinterpret_cast<uintptr_t>(a->exponents) & 1u) return EINVAL;
    for (const int64_t v : {a->q_token_stride, a->q_head_stride, a->q_out_token_stride, a->q_out_head_stride,
                            a->k_new_token_stride, a->k_new_head_stride, a->v_new_token_stride, a->v_new_head_stride})
        if (v % 8 || v < 0) return EINVAL;
    for (const int64_t v :
         {a->k_page_stride, a->k_slot_stride, a->k_head_stride, a->v_page_stride, a->v_slot_stride, a->v_head_stride})
        if (v % (int8 ? 16 : 8) || v < 0) return EINVAL;
    if (a->exponents_page_stride % 2 || a->exponents_head_stride % 2 || a->exponents_page_stride < 0 ||
        a->exponents_head_stride < 0 || a->cos_sin_stride % 4 || a->cos_sin_stride < 0 || a->table_stride < 0)
        return EINVAL;
    AppendParams p{};
    p.q = static_cast<const uint16_t*>(a->q), p.q_out = static_cast<uint16_t*>(a->q_out);
    p.k_new = static_cast<const uint16_t*>(a->k_new), p.v_new = static_cast<const uint16_t*>(a->v_new);
    p.k_pages = a->k_pages, p.v_pages = a->v_pages, p.exponents = a->exponents;
    p.table = a->page_table, p.q_start = a->q_start, p.kv_len = a->kv_len, p.positions = a->positions;
    p.cos_sin = a->cos_sin, p.err = a->error;
    p.q_ts = a->q_token_stride, p.q_hs = a->q_head_stride;
    p.qo_ts = a->q_out_token_stride, p.qo_hs = a->q_out_head_stride;
    p.kn_ts = a->k_new_token_stride, p.kn_hs = a->k_new_head_stride;
    p.vn_ts = a->v_new_token_stride, p.vn_hs = a->v_new_head_stride;
    p.kp_ps = a->k_page_stride, p.kp_ss = a->k_slot_stride, p.kp_hs = a->k_head_stride;
    p.vp_ps = a->v_page_stride, p.vp_ss = a->v_slot_stride, p.vp_hs = a->v_head_stride;
    p.ex_ps = a->exponents_page_stride, p.ex_hs = a->exponents_head_stride;
    p.table_s = a->table_stride, p.cs_s = a->cos_sin_stride;
    p.B = a->batch, p.Hq = a->q_heads, p.Hkv = a->kv_heads, p.P = a->page_size, p.pages = a->pages;
    p.tpages = a->table_pages, p.tokens = a->tokens, p.rotary = a->rotary_dim, p.angles = a->angles;
    p.interleaved = a->interleaved;
    while ((1u << p.pshift) < p.P) ++p.pshift;
    p.lowest = a->dtype == LS_B200_FP16 ? F16::kLowest : BF16::kLowest;
    p.highest = a->dtype == LS_B200_FP16 ? F16::kHighest : BF16::kHighest;
    // Few tokens: a warp takes all of a block's rows. Many: every row group is a task, of
    // twice the heads.
    const bool many = p.tokens > 2 * p.B;
    p.per_task = many ? 2 * kHeads : kHeads;
    p.splits = !many ? 1 : a->head_dim == 128 ? Lane<128>::kIters : Lane<64>::kIters;
    // at most tokens / 16 blocks, and two that are cut for each sequence
    uint64_t items = uint64_t(p.tokens) / kBlock + 2ull * p.B;
    items = items < p.tokens ? items : p.tokens;
    const uint64_t k_tasks = int8 ? p.Hkv : (p.Hkv + p.per_task - 1) / p.per_task * p.splits;
    const uint64_t tasks = 2 * k_tasks + (p.Hq + p.per_task - 1) / p.per_task * p.splits;
    const uint64_t ctas = (items * tasks + kWarps - 1) / kWarps;
    const uint64_t most = uint64_t(sm_count()) * kCtasPerSm;
    const uint32_t grid = uint32_t(ctas < most ? ctas : most);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->head_dim == 64)
        return a->dtype == LS_B200_BF16 ? launch_append<BF16, 64>(p, int8, grid, s)
                                        : launch_append<F16, 64>(p, int8, grid, s);
    return a->dtype == LS_B200_BF16 ? launch_append<BF16, 128>(p, int8, grid, s)
                                    : launch_append<F16, 128>(p, int8, grid, s);
}
