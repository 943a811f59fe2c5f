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

#include "ls_attention.h"

namespace lsb {
namespace {

constexpr int kDecWarps = 4, kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16;                     // keys of one warp's step
constexpr int kDecTile = kDecKeys * kDecWarps;   // slots of one unit of work
constexpr int kDecStages = 3;
constexpr int kDecCtasPerSm = 2;

__host__ __device__ constexpr uint32_t dec_ring(int D) { return uint32_t(kDecWarps * kDecStages * kDecKeys * D * 2 * 2); }
__host__ __device__ constexpr uint32_t dec_smem(int D, int MT) { return dec_ring(D) + uint32_t(16 * MT * D * 2) + 1024; }

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }
// 16 bytes from global memory, or zeros where `on` is false (src is then not read)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

// Row r of a tile of D-element rows: 16-byte pieces XORed with the row's low
// bits, so that the eight rows of an ldmatrix lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t swz(uint32_t row, uint32_t piece) {
    return row * (D * 2) + ((piece ^ (row & 7u)) << 4);
}

// Units of work of one sequence: tiles of its row tiles, over the kv heads.
template <int MR>
__device__ int64_t seq_units(const AttnParams& p, const SeqRange& s) {
    int64_t tiles = 0;
    const int32_t rows = s.nq * int32_t(p.g);
    for (int32_t r = 0; r < rows; r += MR)
        tiles += key_range<kDecTile>(p, s, r / int32_t(p.g), (min(rows, r + MR) - 1) / int32_t(p.g) + 1).tiles;
    return tiles * p.Hkv;
}

// Sum over the block, and the sum over the threads before this one.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sh, int64_t& before) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t inc = v;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (int(lane) >= o) inc += x;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = inc;
    __syncthreads();
    int64_t total = 0;
    before = inc - v;
    for (uint32_t w = 0; w < kDecWarps; ++w) {
        if (w < warp) before += sh[w];
        total += sh[w];
    }
    return total;
}

// Writes one row's results: out = o / l and lse (base 2: m2 + log2 l).
template <class T>
__device__ __forceinline__ void store_pair(const AttnParams& p, int32_t token, uint32_t head, uint32_t d, float x,
                                           float y) {
    *reinterpret_cast<uint32_t*>(p.out + int64_t(token) * p.o_ts + int64_t(head) * p.o_hs + d) = T::pack(x, y);
}

// The kernel. Items are (sequence, tile of 16 * MT rows, kv head); rows are
// (token, head of the group), so that all heads that share a key read it once.
// Each item's slots are cut into units of 64; the units of all items, in
// order, are cut evenly over the CTAs, so that long and short sequences fill
// the GPU alike. A CTA's four warps take 16 slots of a unit each, with rings,
// sums and maxima of their own (no barrier in the loop), and join at the end of
// the item. An item cut over several CTAs is joined, in the order of its
// pieces, by the CTA that arrives last.
template <class T, int D, int MT>
__global__ void __launch_bounds__(kDecThreads, kDecCtasPerSm) attn_decode_kernel(const AttnParams p) {
    constexpr int MR = 16 * MT, KS = D / 16, PIECES = D / 8, RPI = 32 / PIECES, ITERS = kDecKeys / RPI;
    constexpr uint32_t kStage = kDecKeys * D * 2 * 2;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* ring = smem;
    uint8_t* qs = smem + dec_ring(D);
    int64_t* scan = reinterpret_cast<int64_t*>(qs + MR * D * 2);
    int64_t* pick = scan + 8;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t g = int32_t(p.g);

    // total units, and the sequence in which this CTA begins
    int64_t U = 0;
    for (uint32_t b0 = 0; b0 < p.B; b0 += kDecThreads) {
        const uint32_t b = b0 + tid;
        int64_t before;
        U += block_scan(b < p.B ? seq_units<MR>(p, load_seq(p, b)) : 0, scan, before);
    }
    if (!U) return;
    const int64_t G = min(int64_t(gridDim.x), U);
    if (int64_t(blockIdx.x) >= G) return;
    const int64_t cta = blockIdx.x, u_end = cut_begin(U, G, cta + 1);
    int64_t u = cut_begin(U, G, cta), seq_base = 0;
    const int64_t u_begin = u;
    uint32_t b = 0;
    {
        int64_t base = 0;
        for (uint32_t b0 = 0; b0 < p.B; b0 += kDecThreads) {
            const uint32_t bb = b0 + tid;
            const int64_t v = bb < p.B ? seq_units<MR>(p, load_seq(p, bb)) : 0;
            int64_t before;
            const int64_t total = block_scan(v, scan, before);
            if (u < base + total) {
                if (u >= base + before && u < base + before + v) {
                    pick[0] = bb;
                    pick[1] = base + before;
                }
                __syncthreads();
                b = uint32_t(pick[0]);
                seq_base = pick[1];
                break;
            }
            base += total;
        }
    }
    SeqRange s = load_seq(p, b);
    int32_t r0 = 0, rows = s.nq * g;
    int64_t tile_base = seq_base;  // first unit of row tile r0
    KeyRange kr = key_range<kDecTile>(p, s, 0, (min(rows, MR) - 1) / g + 1);

    while (u < u_end) {
        // the item of unit u
        while (u >= tile_base + int64_t(kr.tiles) * p.Hkv || r0 >= rows) {
            if (r0 < rows) {
                tile_base += int64_t(kr.tiles) * p.Hkv;
                r0 += MR;
            }
            while (r0 >= rows) {  // u < U: a later sequence has rows
                s = load_seq(p, ++b);
                r0 = 0;
                rows = s.nq * g;
            }
            kr = key_range<kDecTile>(p, s, r0 / g, (min(rows, r0 + MR) - 1) / g + 1);
        }
        const int32_t h = int32_t((u - tile_base) / kr.tiles);
        const int64_t item = tile_base + int64_t(h) * kr.tiles;
        const int32_t j0 = int32_t(u - item);
        const int32_t steps = int32_t(min(u_end, item + kr.tiles) - u);
        const int32_t R = min(MR, rows - r0);

        // queries to shared memory, zero rows past R
        __syncthreads();  // earlier item's shared memory is no longer read
        for (uint32_t i = tid; i < uint32_t(MR * PIECES); i += kDecThreads) {
            const uint32_t row = i / PIECES, piece = i % PIECES;
            const int32_t rr = r0 + int32_t(row);
            const bool on = int32_t(row) < R;
            const int32_t t = on ? rr / g : 0, hh = on ? h * g + rr % g : 0;
            cp16(smem_u32(qs) + swz<D>(row, piece), p.q + int64_t(s.q0 + t) * p.q_ts + int64_t(hh) * p.q_hs + piece * 8,
                 on);
        }
        cp_commit();

        int32_t pos[MT][2];  // slot of the token of this lane's rows (-1: no row)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int32_t row = mt * 16 + int32_t(lane >> 2) + 8 * i;
                pos[mt][i] = row < R ? s.f + (r0 + row) / g : -1;
            }
        const int32_t pos_lo = s.f + r0 / g, pos_hi = s.f + (r0 + R - 1) / g;

        // page indices: lane i holds the page of step base + i
        const int32_t* trow = p.table + int64_t(b) * p.table_s;
        auto page_of = [&](int32_t step) -> int32_t {
            if (step >= steps) return 0;
            const int32_t k0 = tile_at(kr, j0 + step) * kDecTile + int32_t(warp) * kDecKeys;
            if (!((k0 < kr.hi && k0 + kDecKeys > kr.lo) || k0 < kr.sink)) return 0;
            const int32_t id = trow[k0 >> p.pshift];
            if (uint32_t(id) >= p.pages) {
                if (p.err) atomicOr(p.err, kErrPage);
                return -1;
            }
            return id;
        };
        int32_t ids = page_of(int32_t(lane)), ids_next = page_of(int32_t(lane) + 32);
        const uint32_t wring = smem_u32(ring) + warp * (kDecStages * kStage);
        const uint32_t my_piece = lane % PIECES, my_row = lane / PIECES;
        int32_t id_base = 0;
        auto id_at = [&](int32_t step) -> int32_t {
            if (step >= id_base + 32) {
                id_base += 32;
                ids = ids_next;
                ids_next = page_of(id_base + 32 + int32_t(lane));
            }
            return __shfl_sync(0xffffffffu, ids, step - id_base);
        };
        auto load = [&](int32_t step) {
            if (step < steps) {
                const int32_t id = id_at(step);
                const int32_t k0 = tile_at(kr, j0 + step) * kDecTile + int32_t(warp) * kDecKeys;
                const uint32_t dst = wring + uint32_t(step % kDecStages) * kStage;
                const int64_t off = int64_t(k0 & int32_t(p.P - 1));
                const uint16_t* kb = p.k_pages + int64_t(max(id, 0)) * p.kp_ps + off * p.kp_ss + int64_t(h) * p.kp_hs;
                const uint16_t* vb = p.v_pages + int64_t(max(id, 0)) * p.vp_ps + off * p.vp_ss + int64_t(h) * p.vp_hs;
#pragma unroll
                for (int i = 0; i < ITERS; ++i) {
                    const int32_t row = i * RPI + int32_t(my_row), key = k0 + row;
                    const bool fresh = p.fused && key >= s.f;
                    const bool on = ((key < kr.hi && key >= kr.lo) || key < kr.sink) && (fresh || id >= 0);
                    const int64_t tok = int64_t(s.q0) + key - s.f;
                    const uint16_t* ks = fresh && on ? p.k_new + tok * p.kn_ts + int64_t(h) * p.kn_hs
                                                     : on ? kb + row * p.kp_ss : p.k_pages;
                    const uint16_t* vs = fresh && on ? p.v_new + tok * p.vn_ts + int64_t(h) * p.vn_hs
                                                     : on ? vb + row * p.vp_ss : p.v_pages;
                    cp16(dst + swz<D>(row, my_piece), ks + my_piece * 8, on);
                    cp16(dst + kDecKeys * D * 2 + swz<D>(row, my_piece), vs + my_piece * 8, on);
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < kDecStages - 1; ++i) load(i);
        cp_wait<kDecStages - 1>();
        __syncthreads();  // queries in shared memory

        float o[MT][2 * KS][4], m[MT][2], l[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int n = 0; n < 2 * KS; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
        }

        for (int32_t step = 0; step < steps; ++step) {
            cp_wait<kDecStages - 2>();
            __syncwarp();
            const int32_t k0 = tile_at(kr, j0 + step) * kDecTile + int32_t(warp) * kDecKeys;
            const uint32_t ks = wring + uint32_t(step % kDecStages) * kStage, vs = ks + kDecKeys * D * 2;
            // S = Q K^T
            float sc[MT][2][4] = {};
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                uint32_t bf[4];
                ldsm4(bf, ks + swz<D>((lane & 7u) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1u)));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    uint32_t af[4];
                    ldsm4(af, smem_u32(qs) + swz<D>(mt * 16 + (lane & 15u), kk * 2 + (lane >> 4)));
                    T::mma(sc[mt][0], af, bf[0], bf[1]);
                    T::mma(sc[mt][1], af, bf[2], bf[3]);
                }
            }
            const bool full = k0 + kDecKeys - 1 <= pos_lo && R == MR &&
                              (!p.window || int64_t(k0) > int64_t(pos_hi) - int64_t(p.window));
            if (!full) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!sees(p, pos[mt][e >> 1], k0 + nt * 8 + int32_t(lane & 3u) * 2 + (e & 1)))
                                sc[mt][nt][e] = -INFINITY;
            }
            if (p.logits) {
                float* lg = p.logits + ((int64_t(b) * p.Hkv + h) * p.wlen) * p.rows;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int32_t row = mt * 16 + int32_t(lane >> 2) + 8 * (e >> 1);
                            const int32_t key = k0 + nt * 8 + int32_t(lane & 3u) * 2 + (e & 1);
                            if (row < R && key < kr.hi) lg[int64_t(key) * p.rows + r0 + row] = sc[mt][nt][e] * p.c;
                        }
            }
            // running maximum, probabilities and sums
            uint32_t ph[MT][4], pl[MT][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                float nm[2], base[2], al[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float x = fmaxf(fmaxf(sc[mt][0][2 * i], sc[mt][0][2 * i + 1]),
                                    fmaxf(sc[mt][1][2 * i], sc[mt][1][2 * i + 1]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                    nm[i] = fmaxf(m[mt][i], x);
                    base[i] = nm[i] == -INFINITY ? 0.f : nm[i] * p.c;
                    al[i] = ex2(m[mt][i] * p.c - base[i]);
                }
                if (__any_sync(0xffffffffu, nm[0] > m[mt][0] || nm[1] > m[mt][1])) {
#pragma unroll
                    for (int n = 0; n < 2 * KS; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[mt][n][e] *= al[e >> 1];
                    l[mt][0] *= al[0];
                    l[mt][1] *= al[1];
                    m[mt][0] = nm[0];
                    m[mt][1] = nm[1];
                }
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float a = ex2(fmaf(sc[mt][nt][2 * i], p.c, -base[i]));
                        const float c = ex2(fmaf(sc[mt][nt][2 * i + 1], p.c, -base[i]));
                        l[mt][i] += a + c;
                        // A fragment: registers (row, row + 8) x (keys 0-7, 8-15)
                        ph[mt][nt * 2 + i] = T::pack(a, c);
                        float ha, hc;
                        T::unpack(ph[mt][nt * 2 + i], ha, hc);
                        pl[mt][nt * 2 + i] = T::pack(a - ha, c - hc);
                    }
            }
            // O += P V. P enters as its 16-bit rounding plus the 16-bit rounding
            // of what that leaves: the tensor cores are far from busy here, and
            // the sum keeps about twice the bits.
#pragma unroll
            for (int n = 0; n < KS; ++n) {
                uint32_t vf[4];
                ldsm4t(vf, vs + swz<D>((lane & 7u) + (((lane >> 3) & 1u) << 3), n * 2 + (lane >> 4)));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    T::mma(o[mt][2 * n], ph[mt], vf[0], vf[1]);
                    T::mma(o[mt][2 * n + 1], ph[mt], vf[2], vf[3]);
                    T::mma(o[mt][2 * n], pl[mt], vf[0], vf[1]);
                    T::mma(o[mt][2 * n + 1], pl[mt], vf[2], vf[3]);
                }
            }
            // the new tokens' keys and values go to their slots
            if (p.fused && k0 + kDecKeys > s.f && k0 < s.n) {
                const int32_t id = trow[k0 >> p.pshift];
                if (uint32_t(id) < p.pages) {
#pragma unroll
                    for (int i = 0; i < ITERS; ++i) {
                        const int32_t row = i * RPI + int32_t(my_row), key = k0 + row;
                        if (key >= s.f && key < s.n) {
                            const int64_t at = key & int32_t(p.P - 1);
                            const uint32_t o16 = swz<D>(row, my_piece);
                            const uint8_t* kk = ring + (ks - smem_u32(ring)) + o16;
                            const uint8_t* vv = ring + (vs - smem_u32(ring)) + o16;
                            *reinterpret_cast<uint4*>(p.k_pages + int64_t(id) * p.kp_ps + at * p.kp_ss +
                                                      int64_t(h) * p.kp_hs + my_piece * 8) =
                                *reinterpret_cast<const uint4*>(kk);
                            *reinterpret_cast<uint4*>(p.v_pages + int64_t(id) * p.vp_ps + at * p.vp_ss +
                                                      int64_t(h) * p.vp_hs + my_piece * 8) =
                                *reinterpret_cast<const uint4*>(vv);
                        }
                    }
                }
            }
            __syncwarp();
            load(step + kDecStages - 1);
        }
        cp_wait<0>();
        __syncthreads();

        // join the warps through the ring's shared memory
        float* so = reinterpret_cast<float*>(ring);  // [4][MR][D]
        float* sm = so + kDecWarps * MR * D;          // [4][MR] maxima, base 2
        float* sl = sm + kDecWarps * MR;              // [4][MR] sums
        static_assert(kDecWarps * MR * (D + 2) * 4 <= int(dec_ring(D)), "the join fits the ring");
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = l[mt][i];
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                const uint32_t row = mt * 16 + (lane >> 2) + 8 * i;
                if ((lane & 3u) == 0) {
                    sm[warp * MR + row] = m[mt][i] * p.c;
                    sl[warp * MR + row] = x;
                }
#pragma unroll
                for (int n = 0; n < 2 * KS; ++n)
                    *reinterpret_cast<float2*>(so + (warp * MR + row) * D + n * 8 + (lane & 3u) * 2) =
                        make_float2(o[mt][n][2 * i], o[mt][n][2 * i + 1]);
            }
        __syncthreads();
        const bool whole = j0 == 0 && steps == kr.tiles;
        float* slot = p.part + (2 * cta + (u == u_begin ? 0 : 1)) * int64_t(MR * (D + 2));
        for (uint32_t i = tid; i < uint32_t(R * (D / 2)); i += kDecThreads) {
            const uint32_t row = i / (D / 2), d = (i % (D / 2)) * 2;
            float mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) mx = fmaxf(mx, sm[w * MR + row]);
            float x = 0.f, y = 0.f, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kDecWarps; ++w) {
                const float f = mx == -INFINITY ? 0.f : ex2(sm[w * MR + row] - mx);
                const float2 v = *reinterpret_cast<const float2*>(so + (w * MR + row) * D + d);
                x = fmaf(f, v.x, x);
                y = fmaf(f, v.y, y);
                sum = fmaf(f, sl[w * MR + row], sum);
            }
            if (whole) {
                const int32_t rr = r0 + int32_t(row), token = s.q0 + rr / g;
                const uint32_t head = uint32_t(h * g + rr % g);
                const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
                store_pair<T>(p, token, head, d, x * inv, y * inv);
                if (d == 0 && p.lse)
                    p.lse[int64_t(token) * p.Hq + head] = sum == 0.f ? -INFINITY : (mx + lg2(sum)) * kLn2;
            } else {
                *reinterpret_cast<float2*>(slot + row * D + d) = make_float2(x, y);
                if (d == 0) {
                    slot[MR * D + row] = mx;
                    slot[MR * D + MR + row] = sum;
                }
            }
        }
        if (!whole) {
            const int64_t c0 = cut_owner(U, G, item), c1 = cut_owner(U, G, item + kr.tiles - 1);
            __threadfence();
            __syncthreads();
            if (tid == 0) pick[0] = atomicAdd(p.count + c0, 1u) == uint32_t(c1 - c0);
            __syncthreads();
            if (pick[0]) {
                __threadfence();
                if (tid == 0) p.count[c0] = 0;
                auto piece = [&](int64_t c) {
                    return p.part + (2 * c + (c == c0 && cut_begin(U, G, c0) != item ? 1 : 0)) * int64_t(MR * (D + 2));
                };
                for (uint32_t i = tid; i < uint32_t(R * (D / 2)); i += kDecThreads) {
                    const uint32_t row = i / (D / 2), d = (i % (D / 2)) * 2;
                    float mx = -INFINITY;
                    for (int64_t c = c0; c <= c1; ++c) mx = fmaxf(mx, __ldcg(piece(c) + MR * D + row));
                    float x = 0.f, y = 0.f, sum = 0.f;
                    for (int64_t c = c0; c <= c1; ++c) {
                        const float* ps = piece(c);
                        const float f = mx == -INFINITY ? 0.f : ex2(__ldcg(ps + MR * D + row) - mx);
                        const float2 v = __ldcg(reinterpret_cast<const float2*>(ps + row * D + d));
                        x = fmaf(f, v.x, x);
                        y = fmaf(f, v.y, y);
                        sum = fmaf(f, __ldcg(ps + MR * D + MR + row), sum);
                    }
                    const int32_t rr = r0 + int32_t(row), token = s.q0 + rr / g;
                    const uint32_t head = uint32_t(h * g + rr % g);
                    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : NAN;
                    store_pair<T>(p, token, head, d, x * inv, y * inv);
                    if (d == 0 && p.lse)
                        p.lse[int64_t(token) * p.Hq + head] = sum == 0.f ? -INFINITY : (mx + lg2(sum)) * kLn2;
                }
            }
        }
        u += steps;
    }
}

// New keys and values to their slots, for calls whose rows need several tiles.
__global__ void __launch_bounds__(256) attn_append_kernel(const AttnParams p) {
    const SeqRange s = load_seq(p, blockIdx.x);
    const uint32_t pieces = p.D / 8, per_token = p.Hkv * pieces;
    const int32_t t_end = min(s.nq, int32_t(blockIdx.y + 1) * 16);
    for (int32_t t = int32_t(blockIdx.y) * 16; t < t_end; ++t) {
        const int32_t slot = s.f + t;
        if (slot < 0) continue;
        const int32_t id = p.table[int64_t(blockIdx.x) * p.table_s + (slot >> p.pshift)];
        if (uint32_t(id) >= p.pages) {
            if (p.err) atomicOr(p.err, kErrPage);
            continue;
        }
        const int64_t at = slot & int32_t(p.P - 1), tok = s.q0 + t;
        for (uint32_t i = threadIdx.x; i < per_token; i += blockDim.x) {
            const int64_t h = i / pieces, e = (i % pieces) * 8;
            *reinterpret_cast<uint4*>(p.k_pages + int64_t(id) * p.kp_ps + at * p.kp_ss + h * p.kp_hs + e) =
                *reinterpret_cast<const uint4*>(p.k_new + tok * p.kn_ts + h * p.kn_hs + e);
            *reinterpret_cast<uint4*>(p.v_pages + int64_t(id) * p.vp_ps + at * p.vp_ss + h * p.vp_hs + e) =
                *reinterpret_cast<const uint4*>(p.v_new + tok * p.vn_ts + h * p.vn_hs + e);
        }
    }
}

// weights[b, h, slot] from the stored logits, once the rows' lse are known.
// One thread per slot sums its rows in order. New slots start here (their old
// weight is not read); slots that no row sees keep theirs.
__global__ void __launch_bounds__(256) attn_weights_kernel(const AttnParams p) {
    __shared__ float lse2[256];
    __shared__ int32_t pos[256];
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
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) {
        cudaGetLastError();
        return 148;
    }
    return uint32_t(sms);
}
uint32_t dec_grid() {
    const uint32_t g = sm_count() * kDecCtasPerSm;
    return g < kMaxCtas ? g : kMaxCtas;
}
// rows that one item of the decode kernel takes (two 16-row MMA tiles hold
// more rows per key read; one keeps twice the registers for latency)
uint32_t dec_mt(const ls_b200_attention_args& a) {
    return uint64_t(a.max_q) * (a.q_heads / a.kv_heads) <= 16 ? 1 : 2;
}

// Rows of a sequence and kv head beyond which the call goes to the 128-row
// tensor-core tiles of ls_attention_chunk.cu.
constexpr uint64_t kChunkRows = 32;
bool is_chunk(const ls_b200_attention_args& a) {
    const uint32_t g = a.q_heads / a.kv_heads;
    return uint64_t(a.max_q) * g > kChunkRows && g <= 128;
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
    s.lse = s.part + up256(2ull * kMaxCtas * 16 * dec_mt(a) * (a.head_dim + 2) * sizeof(float));
    s.logits = s.lse + (w ? up256(uint64_t(a.tokens) * a.q_heads * sizeof(float)) : 0);
    s.total = s.logits + (w ? up256(uint64_t(a.batch) * a.q_heads * a.weights_length * a.max_q * sizeof(float)) : 0);
    return s;
}

bool stride8(int64_t v) { return v % 8 == 0 && v >= 0; }

// The call's shape: everything that does not depend on pointers.
int check_shape(const ls_b200_attention_args& a) {
    if (a.dtype > LS_B200_BF16 || !a.kv_heads || !a.q_heads || a.q_heads % a.kv_heads || a.q_heads > 65536 ||
        (a.head_dim != 64 && a.head_dim != 128))
        return EINVAL;
    if (a.page_size < 16 || a.page_size > 256 || (a.page_size & (a.page_size - 1))) return EINVAL;
    if (uint64_t(a.table_pages) * a.page_size > 0x7fffff00ull || a.pages > 0x7fffffffu || a.batch > (1u << 22) ||
        a.tokens > 0x7fffff00u || uint64_t(a.max_q) * (a.q_heads / a.kv_heads) > 0x3fffffffull ||
        a.weights_length > 0x7fffff00u || a.window > 0x7fffffffu || a.sinks > 0x7fffffffu)
        return EINVAL;
    if (!(a.scale > 0.f) || std::isinf(a.scale) || a.timeout_ns > kMaxTimeoutNs) return EINVAL;
    return 0;
}

template <class T, int D, int MT>
int launch_decode(const AttnParams& p, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return int(e);
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!bit || !(done.load(std::memory_order_acquire) & bit)) {
        e = cudaFuncSetAttribute(attn_decode_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(dec_smem(D, MT)));
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attn_decode_kernel<T, D, MT>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     int(cudaSharedmemCarveoutMaxShared));
        if (e != cudaSuccess) return int(e);
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    attn_decode_kernel<T, D, MT><<<dec_grid(), kDecThreads, dec_smem(D, MT), s>>>(p);
    return int(cudaGetLastError());
}
template <class T>
int launch_decode(const AttnParams& p, uint32_t mt, cudaStream_t s) {
    if (p.D == 64) return mt == 1 ? launch_decode<T, 64, 1>(p, s) : launch_decode<T, 64, 2>(p, s);
    return mt == 1 ? launch_decode<T, 128, 1>(p, s) : launch_decode<T, 128, 2>(p, s);
}

}  // namespace
}  // namespace lsb

extern "C" {

uint64_t ls_b200_attention_scratch_bytes(const ls_b200_attention_args* a) {
    if (!a || lsb::check_shape(*a)) return 0;
    return lsb::scratch_plan(*a).total;
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
    p.window = a->window, p.sinks = a->sinks, p.wlen = a->weights_length;
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
    const uint32_t mt = dec_mt(*a);
    p.fused = p.k_new && p.rows <= 16 * mt;
    if (p.k_new && !p.fused) {
        attn_append_kernel<<<dim3(p.B, (p.max_q + 15) / 16), 256, 0, s>>>(p);
        if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return int(e);
    }
    const int rc = a->dtype == LS_B200_FP16 ? launch_decode<F16>(p, mt, s) : launch_decode<BF16>(p, mt, s);
    if (rc || !p.weights) return rc;
    attn_weights_kernel<<<p.B * p.Hkv * ((p.wlen + 255) / 256), 256, 0, s>>>(p);
    return int(cudaGetLastError());
}

}  // extern "C"
