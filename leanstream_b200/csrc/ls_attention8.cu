// Attention of few new tokens per sequence (decoding, drafts) over a paged cache
// in 8 bits. The formula is that of ls_attention.cu; a value of the cache is code *
// 2^e, one e for the 16 slots of a block, kv head, and keys or values.
//
// An item is a sequence and kv head, or some neighbouring kv heads where the codes of
// one fill less than a line of memory; the rows of a head are (token, head of the
// group). The slots go by in units of 32 (two blocks), a step for each of the heads;
// the units of all items, in order, are cut evenly over one CTA per SM. Two warps of a
// CTA load, keys and values (four where a step's blocks lie in two pages: a box takes
// its warp about 75 cycles to issue, and 48 sequences in pages of 16 slots take 63 us
// with two, 58 with four). They lay out up to 32 steps at a time, a lane each, and fill
// one ring of stages with what each step needs (first slot, exponents, codes). The
// other warps take the steps in turn, with maxima and sums of their own, and meet at
// the end of an item's piece; the loads run on into the next piece meanwhile. An item
// cut over several CTAs is joined, in the order of its pieces, by the CTA that arrives
// last. Which warp takes which step follows from the step, so results do not depend on
// timing.
//
// Slots and elements are the M dimension of the products and rows their N, so that
// few rows leave no tile half empty, and a code is turned into a number once for
// all of them:
//     S^T = K Q^T     16 slots x 8 rows,     O^T += V^T P^T     16 elements x 8 rows.
// Codes enter as whole numbers in float16, whatever the type of the queries; those
// enter it by a power of two of their own per row (bfloat16: what lies 2^-29 below
// a row's largest loses bits). The exponents meet the logits in 32 bits, and the
// probabilities as 2^(e - E), E the largest exponent of the values so far; when that
// grows the sums are scaled down. A row's reference is only raised when a logit
// passes it by 2^kRaise. P is rounded once, to float16, times 2^kChunkShift.
//
// Bound by the read of the cache: two sequences of up to 150000 slots, 64 heads of 128
// over 8, take 99 to 104 us, of which 90 stream at 5.9 TB/s; 48 of up to 5000 slots, 32
// heads, 59 us; 12 of up to 9000 slots with up to 5 tokens (20 rows, six warps) 57 us; one
// of 130 slots 7.2 us. Rows as the M dimension, one CTA of four warps that load for
// themselves: 163, 90 and (on the chunk kernel) 80 us.
#include <stdint.h>

#include <atomic>
#include <cerrno>
#include <type_traits>

#include "ls_attention.h"
#include "ls_tc.h"

namespace lsb {
namespace {

using namespace tc;

constexpr int kStep = 2 * kBlock;          // slots of a step
constexpr int kSegCount = 48;              // pieces listed at a time
// Steps that beginning and joining an item counts as, and that a CTA takes at least.
// (With 10 and 24 as the cost 48 sequences of up to 5000 slots take 59.0 us, with 16
// 57.6; with 40 as the least, or a cost of 10, one of 130 slots is cut: 9.7 against 6.9.)
constexpr int64_t kItemCost8 = 16, kMinSteps8 = 16;
constexpr uint64_t kGraceNs = 1000000000ull;
constexpr uint64_t kShortNs = 100000;      // bounds that a barrier's try may sleep over: a load takes less

// NT tiles of eight rows, kWarps that compute. One CTA per SM; the ring takes the
// shared memory that the sums of kSide warps at a time leave.
template <int D, int NT>
struct Geo8 {
    static constexpr int kWarps = NT <= 2 ? 8 : 6, kLoaders = NT <= 2 ? 4 : 2, kThreads = 32 * (kWarps + kLoaders);
    static constexpr int kSide = NT >= 3 && D == 64 ? 4 : (kWarps + 1) / 2;
    // kv heads of an item, at most: the codes of 64 elements take half a line of 128 bytes
    // (48 sequences of up to 5000 slots, 16 kv heads: 98 us with one, 72 with two, 68 with
    // four; of 128 elements no gain)
    static constexpr int kHeads = D == 128 || NT == 4 ? 1 : NT == 1 ? 4 : 2;
    static_assert(kWarps % kHeads == 0 && kSide % kHeads == 0, "a warp takes one of them");
    static constexpr bool kSharedQ = NT > 1;  // one tile's queries stay in registers, more in shared memory
    static constexpr int kRows = 8 * NT;
    static constexpr uint32_t kHalf = kStep * D, kStage = 2 * kHalf;  // a step's keys, and its values
    // A stage is always the same warp's: then its next round cannot be taken for the
    // one before, whose load may still be under way.
    static constexpr int kStages = kWarps * (NT == 2 ? 2 : 3) * (128 / D);
    static constexpr uint32_t kJoin = kStages * kStage, kSegs = kJoin + kSide * kRows * D * 4;
    static constexpr uint32_t kQ = kSegs + kSegCount * 64, kQBytes = kSharedQ ? kRows * (D * 2 + 4) : 0;  // of a head
    static constexpr uint32_t kNotes = kQ + kHeads * kQBytes;
    static constexpr uint32_t kBars = kNotes + 8 * kStages;
    static constexpr uint32_t kStat = kBars + 16 * kStages, kScan = kStat + 8 * kWarps * kRows;
    static constexpr uint32_t kSmem = kScan + 16 * (kWarps + kLoaders + 1) + 1024;  // + alignment of the tiles
    static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
};

// A piece of an item: `units` units from unit j0 of a sequence and its kv heads from h.
struct Seg8 {
    int32_t b, h, q0, rows;
    int32_t f, hi, lo, sink;  // as SeqRange, KeyRange
    int32_t ns, first, j0, units;
    int32_t tiles, own;       // units of the item; own: it does not begin the CTA's range
    int64_t item;             // first unit of the item
    __device__ __forceinline__ int32_t slot0(int32_t unit) const {
        const int32_t j = j0 + unit;
        return (j < ns ? j : first + j - ns) * kStep;
    }
    // steps of 2^hs heads (rows that see nothing have a unit, but no step)
    __device__ __forceinline__ int32_t steps(uint32_t hs) const { return hi ? units << hs : 0; }
};
static_assert(sizeof(Seg8) == 64, "list entries");

// What a stage's step needs beside its codes: its first slot, 1 where a row does
// not see all of it; the exponents of both blocks (key's, value's), kNeutral where no
// row sees the block or its page is outside the pool.
struct Note {
    uint32_t k, ex;
};

// The exponent of a block that is not read: below every other, so that it is never the
// largest of a sequence.
constexpr int32_t kNeutral = -127;
// Exponents of blocks as the products take them, four bytes of v: those that are
// `held` (bytes of ones) as they are, but outside T's range they are reported and read
// as NaN; the others are kNeutral.
template <class T>
__device__ __forceinline__ uint32_t known_exponents(uint32_t v, uint32_t held, uint32_t* err) {
    constexpr uint32_t kAll = 0x01010101u, kLow = 0x7f * kAll, kTop = 0x80 * kAll;
    constexpr uint32_t kSpan = uint32_t(T::kHighest - T::kLowest);
    // byte by byte, without a carry: above the lowest; then the top bit where that passes kSpan
    const uint32_t above = ((v & kLow) + kAll * uint32_t(-T::kLowest)) ^ (v & kTop);
    const uint32_t over = (above & kLow) + kAll * ((kSpan < 128 ? 127 : 255) - kSpan);
    const uint32_t wrong = (kSpan < 128 ? over | above : over & above) & held & kTop;
    if (wrong) {
        const uint32_t bytes = (wrong >> 7) * 0xffu;
        if (err && (bytes & ~__vcmpeq4(v, kAll * uint8_t(kNoExponent))))
            atomicOr(err, uint32_t(LS_B200_ATTN_EXPONENT));
        v = (v & ~bytes) | (kAll * uint8_t(kNoExponent) & bytes);
    }
    return (v & held) | (kAll * uint8_t(kNeutral) & ~held);
}

// 16-byte piece of a row in a tile of codes, rows of D bytes, as the TMA's swizzle
// lays them, so that the eight rows of an ldmatrix lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t swz8(uint32_t row, uint32_t piece) {
    return D == 128 ? row * 128 + (((piece ^ row) & 7u) << 4) : row * 64 + (((piece ^ (row >> 1)) & 3u) << 4);
}
// Pairs of the four codes of v to float16, exactly: a code + 128 in the low byte of
// 1024 reads 1024 + 128 + code. `v` with the codes' highest bits turned.
__device__ __forceinline__ uint32_t codes_f16(uint32_t v, uint32_t select) {
    uint32_t r;
    asm("{.reg .b32 t;\n\tprmt.b32 t, %1, %2, %3;\n\tsub.rn.f16x2 %0, t, %4;}"
        : "=r"(r) : "r"(v), "r"(0x64646464u), "r"(select), "r"(0x64806480u));
    return r;
}
constexpr uint32_t kCodes01 = 0x4140, kCodes23 = 0x4342, kCodes02 = 0x4240, kCodes13 = 0x4341;

// The rows of a warp. Lane (g, t) = (lane / 4, lane % 4) holds the rows 2 t and
// 2 t + 1 of each tile for the slots g and g + 8 of a block, and for the elements 16 n
// + 2 g and + 1 of all n.
template <class T, int D, int NT>
struct Rows8 {
    static constexpr int KS = D / 16;
    static constexpr bool kSharedQ = Geo8<D, NT>::kSharedQ;
    // Row g of a tile: elements 4 t .. 4 t + 3 of each 16, as the codes come. Of the
    // one tile, or of the tile that this warp puts to shared memory.
    uint2 q[KS];
    float cq[NT][2];     // scale * log2 e and the rows' own powers of two
    float o[NT][KS][4];  // in units of 2^(most - kChunkShift)
    float m[NT][2], l[NT][2];  // l: of this lane's slots
    int32_t most;

    __device__ __forceinline__ void queries(const AttnParams& p, const Seg8& x, int32_t h, int tile,
                                            uint32_t lane) {
        const int32_t g = int32_t(p.g), r = int32_t(lane >> 2) + 8 * tile;
        const bool on = r < x.rows;
        const uint16_t* at = p.q + int64_t(x.q0 + (on ? r / g : 0)) * p.q_ts +
                             int64_t(h * g + (on ? r % g : 0)) * p.q_hs + (lane & 3u) * 4;
#pragma unroll
        for (int k = 0; k < KS; ++k) q[k] = on ? *reinterpret_cast<const uint2*>(at + k * 16) : make_uint2(0u, 0u);
    }
    // To float16; the row's factor of the logits.
    __device__ __forceinline__ float convert(float c) {
        if constexpr (std::is_same_v<T, BF16>) {
            uint32_t top = 0;  // bits of the largest |q| of the row
#pragma unroll
            for (int k = 0; k < KS; ++k)
                top = max(max(top, max(q[k].x & 0x7fffu, (q[k].x >> 16) & 0x7fffu)),
                          max(q[k].y & 0x7fffu, (q[k].y >> 16) & 0x7fffu));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // to [2^14, 2^15); infinities and NaN stay what they are
            const int32_t e = top >= 0x7f80u ? 0 : max(int32_t(top >> 7) - 127 - 14, -112);
            const float f = two_to(-e);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                float a, b;
                BF16::unpack(q[k].x, a, b);
                q[k].x = F16::pack(a * f, b * f);
                BF16::unpack(q[k].y, a, b);
                q[k].y = F16::pack(a * f, b * f);
            }
            c *= two_to(e);
        }
        return c;
    }
    // A tile's queries to shared memory: [tile][D / 32][lane] of two k's, then the factors.
    __device__ __forceinline__ void share(uint8_t* to, float c, int tile, uint32_t lane) {
        c = convert(c);
#pragma unroll
        for (int k = 0; k < KS; k += 2)
            *reinterpret_cast<uint4*>(to + ((tile * (KS / 2) + k / 2) * 32 + lane) * 16) =
                make_uint4(q[k].x, q[k].y, q[k + 1].x, q[k + 1].y);
        if ((lane & 3u) == 0) reinterpret_cast<float*>(to + NT * KS * 256)[8 * tile + (lane >> 2)] = c;
    }
    __device__ __forceinline__ void begin(const uint8_t* shared, float scale, uint32_t lane) {
        const int32_t t = int32_t(lane & 3u);
        float c = scale;
        if constexpr (!kSharedQ) c = convert(scale);
        most = -126;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                cq[i][y] = kSharedQ ? reinterpret_cast<const float*>(shared + NT * KS * 256)[8 * i + 2 * t + y]
                                    : __shfl_sync(0xffffffffu, c, (2 * t + y) * 4);
                m[i][y] = -INFINITY, l[i][y] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < KS; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
        }
    }
    // 32 slots, codes of their keys and values at ks and vs
    __device__ __forceinline__ void step(const AttnParams& p, const Seg8& x, const uint8_t* shared, uint32_t ks,
                                         uint32_t vs, Note note, uint32_t lane) {
        const int32_t k0 = int32_t(note.k & ~1u);
        float s[2][NT][4] = {};
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
            uint4 qk[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i)
                qk[i] = kSharedQ ? *reinterpret_cast<const uint4*>(shared + ((i * (KS / 2) + k / 2) * 32 + lane) * 16)
                                 : make_uint4(q[k].x, q[k].y, q[k + 1].x, q[k + 1].y);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                uint32_t v[4];  // slots 0-7 and 8-15 (v[2], v[3]) of two 16-byte pieces
                ldsm4(v, ks + z * (kBlock * D) + swz8<D>((lane & 7u) + ((lane >> 4) << 3), k + ((lane >> 3) & 1u)));
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] ^= 0x80808080u;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t a[4] = {codes_f16(v[y], kCodes01), codes_f16(v[2 + y], kCodes01),
                                           codes_f16(v[y], kCodes23), codes_f16(v[2 + y], kCodes23)};
#pragma unroll
                    for (int i = 0; i < NT; ++i)
                        F16::mma(s[z][i], a, y ? qk[i].z : qk[i].x, y ? qk[i].w : qk[i].y);
                }
            }
        }
        int32_t ev[2];
        float fk[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int32_t ek = int8_t(note.ex >> (16 * z));
            ev[z] = int8_t(note.ex >> (16 * z + 8));
            fk[z] = ek == kNoExponent ? NAN : two_to(max(ek, -126));
        }
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[z][i][e] *= cq[i][e & 1] * fk[z];
        if (note.k & 1u) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    // slot of the row's token (-1: no row)
                    const int32_t row = 8 * i + 2 * int32_t(lane & 3u) + y;
                    const int32_t pos = row < x.rows ? max(x.f + row / int32_t(p.g), -1) : -1;
#pragma unroll
                    for (int z = 0; z < 2; ++z)
#pragma unroll
                        for (int e = y; e < 4; e += 2)
                            if (!sees(p, pos, k0 + z * kBlock + int32_t(lane >> 2) + 8 * (e >> 1)))
                                s[z][i][e] = -INFINITY;
                }
        }
        bool raise = false;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float top = fmaxf(fmaxf(s[0][i][y], s[0][i][2 + y]), fmaxf(s[1][i][y], s[1][i][2 + y]));
                raise = raise | (top > m[i][y] + F16::kRaise);
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float top = fmaxf(fmaxf(s[0][i][y], s[0][i][2 + y]), fmaxf(s[1][i][y], s[1][i][2 + y]));
                    top = fmaxf(m[i][y], top);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const float f = top == -INFINITY ? 1.f : ex2(m[i][y] - top);
                    m[i][y] = top;
                    l[i][y] *= f;
#pragma unroll
                    for (int n = 0; n < KS; ++n) o[i][n][y] *= f, o[i][n][2 + y] *= f;
                }
        }
        if (max(ev[0], ev[1]) > most) {
            const int32_t top = max(ev[0], ev[1]);
            const float f = most - top < -126 ? 0.f : two_to(most - top);
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int n = 0; n < KS; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][n][e] *= f;
            most = top;
        }
        uint32_t b[2][NT][2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const float pw = ev[z] == kNoExponent ? NAN : two_to(max(ev[z] - most + int(F16::kChunkShift), -126));
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float a[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a[e] = ex2(s[z][i][e] - (m[i][e & 1] == -INFINITY ? 0.f : m[i][e & 1]));
                    l[i][e & 1] += a[e];
                    a[e] *= pw;
                }
#pragma unroll
                for (int y = 0; y < 2; ++y)  // slots by rows, to rows by slots
                    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;"
                                 : "=r"(b[z][i][y]) : "r"(F16::pack(a[2 * y], a[2 * y + 1])));
            }
        }
#pragma unroll
        for (int n = 0; n < KS; n += 2)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                // of two 16-byte pieces, slots 0-7 and 8-15 each; a register holds elements 2 g, 2 g + 1
                uint32_t v[4];
                ldsm4t(v, vs + z * (kBlock * D) + swz8<D>((lane & 7u) + (((lane >> 3) & 1u) << 3), n + (lane >> 4)));
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] ^= 0x80808080u;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const uint32_t a[4] = {codes_f16(v[2 * y], kCodes02), codes_f16(v[2 * y], kCodes13),
                                           codes_f16(v[2 * y + 1], kCodes02), codes_f16(v[2 * y + 1], kCodes13)};
#pragma unroll
                    for (int i = 0; i < NT; ++i) F16::mma(o[i][n + y], a, b[z][i][0], b[z][i][1]);
                }
            }
    }
    // Maxima and sums of the rows to sm, sl [8 NT].
    __device__ __forceinline__ void stats(float* sm, float* sl, uint32_t lane) const {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float sum = l[i][y];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const uint32_t row = 8 * i + 2 * lane + y;
                if (lane < 4) sm[row] = m[i][y], sl[row] = sum;
            }
    }
    // The sums' unit, 2^(most - kChunkShift), may lie below the smallest factor: they take
    // what that lacks. (Within `sums` 5 drafted tokens of 12 sequences took 58.1 us for
    // 56.9, with other registers.)
    __device__ __forceinline__ void lower() {
        const int32_t e = most - int32_t(F16::kChunkShift);
        if (e >= -126) return;
        const float f = two_to(e + 126);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int n = 0; n < KS; ++n)
#pragma unroll
                for (int y = 0; y < 4; ++y) o[i][n][y] *= f;
    }
    // The sums times 2^(own maximum - top(row)) (`own`: as they are) to row at0 + row of
    // `join`, or added there.
    template <class F>
    __device__ __forceinline__ void sums(float* join, uint32_t at0, int32_t R, bool own, bool add, F top,
                                         uint32_t lane) const {
        const float unit = two_to(max(most - int(F16::kChunkShift), -126));
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const uint32_t row = 8 * i + 2 * (lane & 3u) + y, at = at0 + row;
                if (int32_t(row) >= R) continue;
                const float mx = own ? m[i][y] : top(row);
                const float f = mx == -INFINITY ? 0.f : own ? unit : ex2(m[i][y] - mx) * unit;
                float* to = join + at * D;
#pragma unroll
                for (int n = 0; n < KS; ++n) {
                    float2* cell = reinterpret_cast<float2*>(to + ((n * 16 + (lane >> 2) * 2) ^ (at & 7u) * 8));
                    float2 v = make_float2(o[i][n][y] * f, o[i][n][2 + y] * f);
                    if (add) v.x += cell->x, v.y += cell->y;
                    *cell = v;
                }
            }
    }
};

// Sums of (x, y) over the block, and over the threads before this one.
struct Pair8 {
    int64_t x;
    int32_t y;
};
template <int WARPS>
__device__ __forceinline__ Pair8 block_scan8(Pair8 v, Pair8* sh, Pair8& before) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Pair8 inc = v;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc.x, o);
        const int32_t y = __shfl_up_sync(0xffffffffu, inc.y, o);
        if (int(lane) >= o) inc.x += x, inc.y += y;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = inc;
    __syncthreads();
    Pair8 total{0, 0};
    before = Pair8{inc.x - v.x, inc.y - v.y};
    for (uint32_t w = 0; w < WARPS; ++w) {
        if (w < warp) before.x += sh[w].x, before.y += sh[w].y;
        total.x += sh[w].x, total.y += sh[w].y;
    }
    return total;
}

// A quotient of two counts, in 32 bits where they fit (nearly always).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return uint64_t(a | b) >> 32 ? a / b : int64_t(uint32_t(a) / uint32_t(b));
}
// U units cut over G CTAs: the first U % G take one more than the others.
struct Cut {
    int64_t each, more;
    __device__ __forceinline__ Cut(int64_t U, int64_t G) : each(quotient(U, G)), more(U - each * G) {}
    __device__ __forceinline__ int64_t begin(int64_t c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int64_t owner(int64_t u) const {
        const int64_t head = more * (each + 1);
        return u < head ? quotient(u, each + 1) : more + quotient(u - head, each);
    }
};

template <class T, int D, int NT>
__global__ void __launch_bounds__(Geo8<D, NT>::kThreads, 1)
    attn_decode8_kernel(const AttnParams p, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap) {
    using G = Geo8<D, NT>;
    constexpr int W = G::kWarps, MR = G::kRows;
    extern __shared__ uint8_t raw[];
    const uint32_t sbase = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* const smem = raw + (sbase - smem_u32(raw));
    Seg8* const segs = reinterpret_cast<Seg8*>(smem + G::kSegs);
    Note* const notes = reinterpret_cast<Note*>(smem + G::kNotes);
    float* const join = reinterpret_cast<float*>(smem + G::kJoin);
    Pair8* const scan = reinterpret_cast<Pair8*>(smem + G::kScan);
    volatile uint32_t* const flag = reinterpret_cast<uint32_t*>(scan + W + G::kLoaders);
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t g = int32_t(p.g);
    auto full = [&](uint32_t s) { return sbase + G::kBars + 8 * s; };
    auto empty = [&](uint32_t s) { return sbase + G::kBars + 8 * (G::kStages + s); };
    auto wait = [&](uint32_t bar, uint32_t parity) {
        return p.timeout_ns < kShortNs ? warp_wait_short(bar, parity, uint32_t(p.timeout_ns))
                                       : warp_wait(bar, parity, p.timeout_ns);
    };

    if (warp == W) {
        const uint32_t loaders = p.P >= uint32_t(kStep) ? 2 : G::kLoaders;
        for (uint32_t i = lane; i < 2u * G::kStages; i += 32) bar_init(full(i), i < uint32_t(G::kStages) ? loaders : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (lane < 2) prefetch_map(lane ? &vmap : &kmap);
    }
    if (tid == 0) flag[0] = flag[1] = flag[3] = 0;
    after_start();
    after_wait();
    // tiles of this thread's sequence (of the first kThreads), and of the call; y: 1
    // where the sequence has rows
    auto tiles_of = [&](uint32_t b, SeqRange& s) -> Pair8 {
        s = SeqRange{0, 0, 0, 0};
        if (b < p.B) s = load_seq(p, b);
        if (!s.nq) return Pair8{0, 0};
        return Pair8{key_range<kStep>(p, s, 0, s.nq).tiles, 1};
    };
    SeqRange seq0;
    const Pair8 v0 = tiles_of(tid, seq0);
    Pair8 before0;
    const Pair8 total0 = block_scan8<W + G::kLoaders>(v0, scan, before0);
    Pair8 all = total0;
    for (uint32_t b0 = G::kThreads; b0 < p.B; b0 += G::kThreads) {
        SeqRange s;
        Pair8 before;
        const Pair8 more = block_scan8<W + G::kLoaders>(tiles_of(b0 + tid, s), scan, before);
        all.x += more.x, all.y += more.y;
    }
    if (!all.y) return;
    // heads of an item: 2^hs, as many as leave items for half of the CTAs (fewer items
    // are cut into more parts, which one CTA joins)
    uint32_t hs = 0;
    for (uint32_t more = 1; 1 << more <= G::kHeads; ++more)
        if (p.Hkv % (1u << more) == 0 && int64_t(all.y) * (p.Hkv >> more) * 2 >= gridDim.x) hs = more;
    const uint32_t side_by = (1u << hs) - 1;
    const int64_t Hi = p.Hkv >> hs, item_cost = kItemCost8 >> hs, min_units = kMinSteps8 >> hs;
    auto units = [&](Pair8 v) { return (v.x + v.y * item_cost) * Hi; };
    const int64_t U = units(all);
    const int64_t NC = max(int64_t(1), min(int64_t(gridDim.x), quotient(U + min_units - 1, min_units)));
    if (int64_t(blockIdx.x) >= NC) return;
    const Cut cut(U, NC);
    const int64_t cta = blockIdx.x, u_begin = cut.begin(cta), u_end = cut.begin(cta + 1);
    // after a wait that gave up the warp loads and computes no more, and only meets
    // the others
    bool ok = true;
    uint32_t done = 0;                      // steps of the pieces so far
    uint32_t turn = warp, t_stage = warp, t_round = 0;  // this warp's next step, its stage and its round
    uint32_t loaded = 0;                    // steps loaded in whole blocks
    uint32_t again = 0;                     // lanes of the block that was given up which have loaded
    static_assert(G::kStages % W == 0, "a stage is always the same warp's");
    Rows8<T, D, NT> rows;

    for (int64_t u = u_begin; u < u_end;) {
        // the next pieces, listed by the threads of their sequences: items (y
        // counts sequences with rows) from the one that holds unit u
        if (u != u_begin) {
            if (tid == 0) flag[0] = flag[1] = flag[3] = 0;
            __syncthreads();
        }
        int64_t base = 0;
        int32_t seqs = 0;
        for (uint32_t b0 = 0; b0 < p.B && base < u_end; b0 += G::kThreads) {
            SeqRange s = seq0;
            Pair8 v = v0, before = before0, total = total0;
            if (b0) {
                v = tiles_of(b0 + tid, s);
                total = block_scan8<W + G::kLoaders>(v, scan, before);
            }
            const int64_t at = base + units(before), item_units = v.y ? v.x + item_cost : 1, end = at + units(v);
            const int32_t seq = seqs + before.y;
            if (v.y && u >= at && u < end)
                flag[1] = uint32_t(seq * int32_t(Hi) + int32_t(quotient(u - at, item_units)));
            __syncthreads();
            const int64_t from = max(u, at), to = min(u_end, end);
            if (from < to) {
                const KeyRange kr = key_range<kStep>(p, s, 0, s.nq);
                int32_t h = int32_t(quotient(from - at, item_units));
                int32_t idx = seq * int32_t(Hi) + h - int32_t(flag[1]);
                for (; h < int32_t(Hi) && idx < kSegCount; ++h, ++idx) {
                    Seg8 x;
                    x.item = at + h * item_units + item_cost;
                    const int64_t a = max(x.item, u), e = min(x.item + kr.tiles, u_end);
                    if (a >= e) break;  // only the item's cost lies in the range
                    x.b = int32_t(b0 + tid), x.h = h << hs, x.q0 = s.q0, x.rows = s.nq * g;
                    x.f = s.f, x.hi = kr.hi, x.lo = kr.lo, x.sink = kr.sink, x.ns = kr.ns, x.first = kr.first;
                    x.tiles = kr.tiles;
                    x.j0 = int32_t(a - x.item), x.units = int32_t(e - a);
                    x.own = a != u_begin;
                    segs[idx] = x;
                    atomicMax(const_cast<uint32_t*>(flag), uint32_t(idx + 1));
                }
            }
            base += units(total);
            seqs += total.y;
        }
        __syncthreads();
        const uint32_t count = flag[0];
        if (!count) break;  // what is left of the range is the cost of an item

        if (warp >= W + 2 && p.P >= uint32_t(kStep)) {  // (a step lies in one page: two warps load)
        } else if (warp >= W) {
            // ---- loads: blocks of steps of a piece, a lane and a stage each; the pages of
            // the block after it are under way. One of the warps also takes the exponents.
            const bool keys = (warp - W) % 2 == 0, note = warp == W;
            const bool first = G::kLoaders == 2 || warp < W + 2, second = G::kLoaders == 2 || warp >= W + 2;  // blocks
            const CUtensorMap* const map = keys ? &kmap : &vmap;
            constexpr int32_t kBlockSteps = G::kStages < 32 ? G::kStages : 32;
            static_assert(kBlockSteps % G::kHeads == 0, "a unit's steps stay together");
            const bool pairs = p.P >= uint32_t(kStep);  // a step lies in one page
            auto seen = [&](const Seg8& x, int32_t k) { return (k < x.hi && k + kBlock > x.lo) || k < x.sink; };
            // pages of both blocks of a step (-1: no row sees the block)
            auto pages_of = [&](uint32_t c, int32_t step) -> int2 {
                int2 id = make_int2(-1, -1);
                if (c >= count) return id;
                const Seg8& x = segs[c];
                if (step >= x.steps(hs)) return id;
                const int32_t k = x.slot0(step >> hs);
                const int32_t* row = p.table + int64_t(x.b) * p.table_s;
                auto page = [&](int32_t slot) {
                    const int32_t at = row[slot >> p.pshift];
                    if (uint32_t(at) < p.pages) return at;
                    if (note && p.err) atomicOr(p.err, kErrPage);
                    return int32_t(p.pages);
                };
                if (seen(x, k)) id.x = page(k);
                if (seen(x, k + kBlock)) id.y = pairs && id.x >= 0 ? id.x : page(k + kBlock);
                return id;
            };
            auto exponents_of = [&](uint32_t c, int32_t step, int2 id) -> uint32_t {
                uint32_t x0 = 0, x1 = 0;
                if (!note || c >= count) return 0;
                const Seg8& x = segs[c];
                const int32_t in = step < x.steps(hs) ? x.slot0(step >> hs) & int32_t(p.P - 1) : 0;
                const uint8_t* at = p.ex + int64_t(x.h + int32_t(uint32_t(step) & side_by)) * p.ex_hs;
                if (uint32_t(id.x) < p.pages)
                    x0 = *reinterpret_cast<const uint16_t*>(at + int64_t(id.x) * p.ex_ps + (in >> 3));
                if (uint32_t(id.y) < p.pages)
                    x1 = *reinterpret_cast<const uint16_t*>(at + int64_t(id.y) * p.ex_ps +
                                                            (((in + kBlock) & int32_t(p.P - 1)) >> 3));
                return x0 | x1 << 16;
            };
            uint32_t c = 0, n_c = 0;
            int32_t at = 0, n_at = 0;
            auto after = [&]() {
                n_at += kBlockSteps;
                if (n_c < count && n_at >= segs[n_c].steps(hs)) ++n_c, n_at = 0;
            };
            int2 id = pages_of(0, int32_t(lane)), n_id;
            uint32_t ex = exponents_of(0, int32_t(lane), id), n_ex = 0;
            bool known = false;  // the next block's pages: of the second looked up when the first loads
            after();
            while (ok && c < count) {
                const Seg8& x = segs[c];
                const int32_t n = min(kBlockSteps, x.steps(hs) - at), h = x.h + int32_t(lane & side_by);
                const bool mine = int32_t(lane) < n;
                const int32_t k = mine ? x.slot0((at + int32_t(lane)) >> hs) : 0, in = k & int32_t(p.P - 1);
                const bool masked = k + kStep - 1 > x.f ||
                                    (p.window && int64_t(k) <= int64_t(x.hi) - 1 - int64_t(p.window));
                const uint32_t boxes = (first && id.x >= 0) + (second && id.y >= 0);  // of a block
                const uint32_t bytes = pairs ? G::kHalf : boxes * (G::kHalf / 2);
                const uint32_t st = (loaded + lane) % G::kStages, round = (loaded + lane) / G::kStages;
                const uint32_t dst = sbase + st * G::kStage + (keys ? 0 : G::kHalf), bar = full(st);
                // Each lane loads when its stage is free. That ends, as every wait of the warps
                // that compute does; once they are through, what is free is loaded by every
                // loading warp and the rest by none, so that each stage's barrier completes.
                bool left = mine, through = false;
                for (uint32_t spin = 1;; ++spin) {
                    if (left && (!round || bar_test(empty(st), (round - 1) & 1u))) {
                        if (pairs) {
                            tma4(dst, map, bar, 0, in, h, max(id.x, id.y));
                        } else {
                            if (first && id.x >= 0) tma4(dst, map, bar, 0, in, h, id.x);
                            if (second && id.y >= 0) tma4(dst + kBlock * D, map, bar, 0, 0, h, id.y);
                        }
                        if (note) {
                            // (blocks that are not read leave the sums' unit alone; -16 to -1 need no
                            // look: one at all of them costs 48 sequences 0.6 us, and by the warps that
                            // compute, 4 drafted tokens of 24 sequences, 64 elements, 0.9 of 42)
                            uint32_t e = ex;
                            if ((e & 0xf0f0f0f0u) != 0xf0f0f0f0u)
                                e = known_exponents<T>(e, (uint32_t(id.x) < p.pages ? 0xffffu : 0u) |
                                                              (uint32_t(id.y) < p.pages ? 0xffff0000u : 0u), p.err);
                            notes[st] = Note{uint32_t(k) | uint32_t(masked), e};
                        }
                        bar_arrive_tx(bar, bytes);
                        left = false;
                    }
                    if (!__any_sync(0xffffffffu, left)) break;
                    if (through) {
                        ok = false;
                        again = __ballot_sync(0xffffffffu, mine && !left);
                        if (mine && !left) bar_wait(bar, round & 1u, kGraceNs);
                        break;
                    }
                    if (spin % 16 == 0) {
                        through = __all_sync(0xffffffffu, flag[3] == uint32_t(W));
                        __threadfence_block();
                    }
                }
                __syncwarp();
                if (!known) n_id = pages_of(n_c, n_at + int32_t(lane));
                known = true;
                n_ex = exponents_of(n_c, n_at + int32_t(lane), n_id);
                if (ok) loaded += uint32_t(max(n, 0));
                c = n_c, at = n_at, id = n_id, ex = n_ex;
                after();
                n_id = pages_of(n_c, n_at + int32_t(lane));
            }
        } else {
            // ---- rows
            float* const sm = reinterpret_cast<float*>(smem + G::kStat);  // [W][MR]
            float* const sl = sm + W * MR;
            auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * W) : "memory"); };
            const uint32_t mine = warp & side_by;  // the head of an item that this warp takes
            auto top_of = [&](uint32_t of, uint32_t row) {
                float mx = sm[of * MR + row];
#pragma unroll
                for (uint32_t w = 1; w < uint32_t(W); ++w)
                    if ((w & side_by) == of) mx = fmaxf(mx, sm[w * MR + row]);
                return mx;
            };
            auto top = [&](uint32_t row) { return top_of(mine, row); };
            uint8_t* const shared = smem + G::kQ + mine * G::kQBytes;
            const int tile = G::kSharedQ ? int(warp >> hs) : 0;  // of the queries that this warp reads
            if (tile < NT) rows.queries(p, segs[0], segs[0].h + int32_t(mine), tile, lane);
            if constexpr (G::kSharedQ) {
                if (tile < NT) rows.share(shared, p.c, tile, lane);
                meet();
            }
            for (uint32_t c = 0; c < count; ++c) {
                const Seg8& x = segs[c];
                const int32_t R = x.rows;
                const uint32_t n = uint32_t(x.steps(hs));
                rows.begin(shared, p.c, lane);
                while (ok && turn - done < n) {
                    if (!(ok = wait(full(t_stage), t_round & 1u))) break;
                    const uint32_t ks = sbase + t_stage * G::kStage;
                    rows.step(p, x, shared, ks, ks + G::kHalf, notes[t_stage], lane);
                    __syncwarp();
                    if (lane == 0) bar_arrive(empty(t_stage));
                    turn += W;
                    t_stage += W;
                    if (t_stage >= uint32_t(G::kStages)) t_stage -= G::kStages, ++t_round;
                }
                done += n;
                // the warps' sums meet: where they all fit each as it is; else maxima first,
                // then some of the warps at a time
                const bool own = W * R <= G::kSide * MR;
                const int32_t side = own ? W : G::kSide;
                rows.lower();
                rows.stats(sm + warp * MR, sl + warp * MR, lane);
                if (!own) meet();
                for (int32_t w0 = 0; w0 < W; w0 += side) {
                    if (uint32_t(int32_t(warp) - w0) < uint32_t(side))
                        rows.sums(join, uint32_t((int32_t(warp) - w0) * R), R, own, w0 != 0, top, lane);
                    if (w0 + side >= W && c + 1 < count && tile < NT)
                        rows.queries(p, segs[c + 1], segs[c + 1].h + int32_t(mine), tile, lane);
                    meet();
                }
                if (G::kSharedQ && c + 1 < count && tile < NT) rows.share(shared, p.c, tile, lane);
                // rows by warps, D / 32 elements of a row per lane
                constexpr int E = D / 32;
                const bool whole = x.j0 == 0 && x.units == x.tiles;
                constexpr int64_t kPart = MR * (D + 2);  // of a head
                float* const slot = p.part + ((2 * cta + x.own) << hs) * kPart;
                auto finish = [&](int32_t of, int32_t row, const float (&v)[E], float mx, float sum) {
                    const int32_t token = x.q0 + row / g;
                    const int64_t head = (x.h + of) * g + row % g;
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
                for (int32_t i = int32_t(warp); i < R << hs; i += W) {
                    const int32_t of = hs ? i / R : 0, row = i - of * R;  // head of the item
                    const float mx = top_of(uint32_t(of), uint32_t(row));
                    float sum = 0.f, v[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        if ((uint32_t(w) & side_by) != uint32_t(of)) continue;
                        const float f = mx == -INFINITY ? 0.f : ex2(sm[w * MR + row] - mx);
                        sum = fmaf(f, sl[w * MR + row], sum);
                        if (w >= side) continue;
                        const uint32_t at = uint32_t(w * R + row);
                        const float* from = join + at * D + ((lane * E) ^ (at & 7u) * 8);
#pragma unroll
                        for (int e = 0; e < E; ++e) v[e] = fmaf(own ? f : 1.f, from[e], v[e]);
                    }
                    if (whole) {
                        finish(of, row, v, mx, sum);
                    } else {
                        float* const to = slot + of * kPart;
#pragma unroll
                        for (int e = 0; e < E; ++e) to[row * D + lane * E + e] = v[e];
                        if (lane == 0) to[MR * D + row] = mx, to[MR * D + MR + row] = sum;
                    }
                }
                if (!whole) {
                    const int64_t c0 = cut.owner(x.item), c1 = cut.owner(x.item + x.tiles - 1);
                    __threadfence();
                    meet();
                    if (tid == 0) {
                        const bool last = atomicAdd(p.count + c0, 1u) == uint32_t(c1 - c0);
                        if (last) p.count[c0] = 0;
                        flag[2] = last;
                    }
                    meet();
                    if (flag[2]) {
                        __threadfence();
                        const int32_t pieces = int32_t(c1 - c0) + 1;
                        const int64_t first = 2 * c0 + (cut.begin(c0) != x.item);
                        for (int32_t j = int32_t(warp); j < R << hs; j += W) {
                            const int32_t of = hs ? j / R : 0, row = j - of * R;
                            auto piece = [&](int32_t i) {
                                return p.part + (((i ? 2 * (c0 + i) : first) << hs) + of) * kPart;
                            };
                            float mx = -INFINITY, sum = 0.f, v[E] = {};
                            for (int32_t i0 = 0; i0 < pieces; i0 += 32) {
                                const int32_t i = i0 + int32_t(lane), n = min(32, pieces - i0);
                                const float pm = i < pieces ? __ldcg(piece(i) + MR * D + row) : -INFINITY;
                                const float ps = i < pieces ? __ldcg(piece(i) + MR * D + MR + row) : 0.f;
                                float f = 0.f;
                                for (int32_t k0 = 0; k0 < n; k0 += 16) {
                                    float y[16][E];
#pragma unroll
                                    for (int k = 0; k < 16; ++k) {
                                        const float* from = piece(min(i0 + k0 + k, pieces - 1)) + row * D + lane * E;
                                        using Vec = std::conditional_t<E == 4, float4, float2>;
                                        *reinterpret_cast<Vec*>(y[k]) = __ldcg(reinterpret_cast<const Vec*>(from));
                                    }
                                    if (!k0) {  // the maximum may grow with each 32 pieces
                                        float nm = pm;
#pragma unroll
                                        for (int d = 16; d; d >>= 1)
                                            nm = fmaxf(nm, __shfl_xor_sync(0xffffffffu, nm, d));
                                        nm = fmaxf(nm, mx);
                                        const float ref = nm == -INFINITY ? 0.f : nm, old = ex2(mx - ref);
                                        f = ex2(pm - ref);
                                        sum = fmaf(f, ps, sum * old);
#pragma unroll
                                        for (int e = 0; e < E; ++e) v[e] *= old;
                                        mx = nm;
                                    }
#pragma unroll
                                    for (int k = 0; k < 16; ++k) {
                                        const float fk = __shfl_sync(0xffffffffu, f, (k0 + k) & 31);
                                        if (k0 + k < n)
#pragma unroll
                                            for (int e = 0; e < E; ++e) v[e] = fmaf(fk, y[k][e], v[e]);
                                    }
                                }
                            }
#pragma unroll
                            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                            finish(of, row, v, mx, sum);
                        }
                    }
                }
                meet();  // the joined sums and maxima have been read
            }
            __threadfence_block();
            if (lane == 0) atomicAdd(const_cast<uint32_t*>(flag) + 3, 1u);
        }
        if (count < uint32_t(kSegCount)) break;  // the list was the whole range
        __syncthreads();                         // it has been read
        u = segs[count - 1].item + segs[count - 1].j0 + segs[count - 1].units;
    }
    if (warp >= W)  // every load has landed before the CTA ends
        for (uint32_t i = loaded - min(loaded, uint32_t(G::kStages)); i != loaded; ++i) {
            const uint32_t j = i + G::kStages - loaded;  // the lane whose stage this is in the next block
            if (j < 32 && again >> j & 1u) continue;     // (it landed, and a load after it)
            warp_wait(full(i % G::kStages), (i / G::kStages) & 1u, kGraceNs);
        }
    if (!ok) gave_up(p);
}

template <class T, int D, int NT>
int launch8(const AttnParams& p, cudaStream_t s) {
    using G = Geo8<D, NT>;
    CUtensorMap km, vm;
    const uint32_t slots = p.P < uint32_t(kStep) ? p.P : uint32_t(kStep);
    if (!encode_codes(&km, p.k_pages, p, p.kp_ss, p.kp_hs, p.kp_ps, slots) ||
        !encode_codes(&vm, p.v_pages, p, p.vp_ss, p.vp_hs, p.vp_ps, slots))
        return EINVAL;
    const auto kernel = attn_decode8_kernel<T, D, NT>;
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return int(e);
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!bit || !(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(G::kSmem));
        if (e != cudaSuccess) return int(e);
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    const uint32_t sms = sm_count(), most = kMaxCtas * 16 / (G::kRows * G::kHeads);  // (by the scratch)
    // (the append before it lets it begin early)
    return int(launch_after(kernel, sms < most ? sms : most, G::kThreads, G::kSmem, s, p, km, vm));
}
template <class T, int D>
int launch8(const AttnParams& p, cudaStream_t s) {
    return p.rows <= 8    ? launch8<T, D, 1>(p, s)
           : p.rows <= 16 ? launch8<T, D, 2>(p, s)
           : p.rows <= 24 ? launch8<T, D, 3>(p, s)
                          : launch8<T, D, 4>(p, s);
}

}  // namespace

int launch_decode8(const AttnParams& p, uint32_t dtype, cudaStream_t s) {
    if (p.D == 64) return dtype == LS_B200_BF16 ? launch8<BF16, 64>(p, s) : launch8<F16, 64>(p, s);
    return dtype == LS_B200_BF16 ? launch8<BF16, 128>(p, s) : launch8<F16, 128>(p, s);
}

}  // namespace lsb
