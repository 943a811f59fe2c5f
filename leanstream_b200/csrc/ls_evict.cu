// Eviction from a paged key/value cache by accumulated attention weight.
//
// Per sequence and kv head, of n slots `budget` stay: the first `sinks`, the
// last `recent`, and of those between the ones of the largest weight (equal
// weights: the lower slot; NaN counts as the lowest value). What stays keeps its
// order and goes to the slots 0 .. of new pages, so that no row is written
// before it is read, pages that other sequences share stay as they are, and
// every row moves on its own.
//
// Two launches: the selection reads 4 B per slot and writes the kept slots'
// indices, the copy moves 4 * head_dim B per kept slot in and out. Both are
// bound by memory where rows are many and long: 64 rows of 16384 to 32768 slots
// cut to 8192 (549 MB) take 118 us, of which the selection 29. (With the copy in
// the selection's CTAs, one launch: 140 us; too few rows under way at a time.)
#include <cooperative_groups.h>
#include <stdint.h>

#include <cerrno>

#include "ls_attention.h"
#include "ls_tc.h"

namespace lsb {
namespace {

namespace cg = cooperative_groups;

constexpr int kShort = 4096;  // slots that one CTA holds in registers
constexpr int kCluster = 8;   // CTAs of a longer row
constexpr int kCopyRows = 4;  // rows that a thread has under way

struct EvictParams {
    const uint16_t* k_pages;
    const uint16_t* v_pages;
    uint16_t* k_new;
    uint16_t* v_new;
    const int32_t* table;
    const int32_t* kv_len;
    const int32_t* new_table;
    const float* weights;
    float* new_weights;
    int32_t* kept;
    int32_t* new_len;
    uint32_t* err;
    int64_t kp_ps, kp_ss, kp_hs, vp_ps, vp_ss, vp_hs, table_s, new_table_s, w_ss, w_hs;
    uint32_t B, Hkv, D, P, pshift, pages, tpages, wlen, budget, sinks, recent;
};

__device__ __forceinline__ int32_t evict_len(const EvictParams& p, uint32_t b) {
    const int32_t n = p.kv_len[b];
    if (n >= 0 && uint64_t(n) <= uint64_t(p.tpages) << p.pshift && uint32_t(n) <= p.wlen) return n;
    if (p.err) atomicOr(p.err, kErrLength);
    return 0;
}

// Unsigned keys in the order of the weights: NaN with -inf, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float w) {
    const uint32_t u = __float_as_uint(isnan(w) ? -INFINITY : w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the block of a pair of 16-bit counts, and of the threads before.
template <int kWarps>
__device__ __forceinline__ uint32_t select_scan(uint32_t v, uint32_t* sh, uint32_t& before) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (int(lane) >= o) inc += x;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = inc;
    __syncthreads();
    uint32_t total = 0;
    before = inc - v;
    for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) before += sh[w];
        total += sh[w];
    }
    return total;
}

// One cluster of CL CTAs per (sequence, kv head), each CTA a stretch of its
// slots. The budget's smallest kept key is found eight bits at a time from the
// top: a histogram of the keys that share the bits found so far, summed over
// the cluster through distributed shared memory. Then every CTA counts what it
// keeps, and writes it from where the CTAs before it end. A stretch of up to
// kShort slots stays in registers; longer ones are read again from L2 by each
// step. (One CTA per row took 108 us for 64 rows of up to 32768 slots.)
template <int CL, int kThreads>
__global__ void __launch_bounds__(kThreads) evict_select_kernel(const EvictParams p) {
    constexpr int kSelThreads = kThreads, kSelWarps = kThreads / 32, kPiece = kShort;
    constexpr int kOwn = kPiece / kThreads;  // consecutive slots of a thread in a piece
    __shared__ uint32_t hist[2][256];
    __shared__ uint32_t total[256], scan[kSelWarps], found[2], counts[2];
    tc::after_start();
    const uint32_t row = blockIdx.x / CL, rank = CL > 1 ? blockIdx.x % CL : 0;
    const uint32_t b = row / p.Hkv, h = row % p.Hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t n = evict_len(p, b);
    const float* w = p.weights + int64_t(b) * p.w_ss + int64_t(h) * p.w_hs;
    int32_t* kept = p.kept + int64_t(row) * p.budget;
    float* nw = p.new_weights ? p.new_weights + int64_t(row) * p.budget : nullptr;
    if (h == 0 && rank == 0 && tid == 0) p.new_len[b] = min(n, int32_t(p.budget));
    if (n <= int32_t(p.budget)) {
        for (uint32_t j = rank * kSelThreads + tid; j < p.budget; j += CL * kSelThreads) {
            kept[j] = int32_t(j) < n ? int32_t(j) : -1;
            if (nw) nw[j] = int32_t(j) < n ? w[j] : 0.f;
        }
        return;  // (the whole cluster)
    }
    auto cluster = cg::this_cluster();
    const int32_t lo = int32_t(p.sinks), hi = n - int32_t(p.recent);
    const int32_t stretch = (n + CL - 1) / CL, first = min(n, int32_t(rank) * stretch), end = min(n, first + stretch);
    const bool held = stretch <= kPiece;
    float v[kOwn];
    auto read = [&](int32_t i0) {  // this thread's slots of the piece from i0
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
            const int32_t i = i0 + int32_t(tid) * kOwn + e;
            v[e] = i < end ? w[i] : 0.f;
        }
    };
    if (held) read(first);
    uint32_t need = p.budget - p.sinks - p.recent;  // slots to take between
    const bool any = need != 0;
    uint32_t prefix = 0, mask = 0;
    if (any) {
#pragma unroll 1
        for (int step = 0; step < 4; ++step) {
            const int shift = 24 - 8 * step;
            uint32_t* const own = hist[step & 1];
            if (tid < 256) own[tid] = 0;
            __syncthreads();
            for (int32_t i0 = first; i0 < end; i0 += kPiece) {
                if (!held) read(i0);
#pragma unroll
                for (int e = 0; e < kOwn; ++e) {
                    const int32_t i = i0 + int32_t(tid) * kOwn + e;
                    const uint32_t k = order_key(v[e]);
                    if (i >= lo && i < hi && i < end && (k & mask) == prefix)
                        atomicAdd(own + ((k >> shift) & 255u), 1u);
                }
            }
            if constexpr (CL > 1) cluster.sync();
            else __syncthreads();
            if (tid < 256) {  // a thread per digit adds up the cluster's
                uint32_t c[CL];
                uint32_t sum = 0;
#pragma unroll
                for (int r = 0; r < CL; ++r) c[r] = CL > 1 ? cluster.map_shared_rank(own, r)[tid] : own[tid];
#pragma unroll
                for (int r = 0; r < CL; ++r) sum += c[r];
                total[tid] = sum;
            }
            __syncthreads();
            if (warp == 0) {  // the digit in which the need-th largest key lies; lane: eight digits
                uint32_t c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += c[i] = total[255 - (lane * 8 + i)];
                uint32_t inc = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
                    if (int(lane) >= o) inc += x;
                }
                uint32_t before = inc - sum;
                if (before < need && need <= inc) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (before < need && need <= before + c[i]) {
                            found[0] = 255 - (lane * 8 + i);
                            found[1] = need - before;
                        }
                        before += c[i];
                    }
                }
            }
            __syncthreads();  // (the other histogram is next: nobody reads this one by the time it is cleared again)
            prefix |= found[0] << shift;
            mask |= 255u << shift;
            need = found[1];
        }
    }
    // prefix is the smallest kept key, of which the first `need` are kept.
    // Low half: slots kept for certain, high half: slots with that key.
    auto counts_of = [&](int32_t i0) {
        uint32_t c = 0;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
            const int32_t i = i0 + int32_t(tid) * kOwn + e;
            const uint32_t k = order_key(v[e]);
            const bool between = i >= lo && i < hi;
            if (i < end) c += (!between || (any && k > prefix)) ? 1u : any && k == prefix ? 1u << 16 : 0u;
        }
        return c;
    };
    uint32_t at = 0, ties = 0, before;
    if constexpr (CL > 1) {  // what the CTAs before this one keep
        uint32_t sure = 0, equal = 0;
        for (int32_t i0 = first; i0 < end; i0 += kPiece) {
            if (!held) read(i0);
            const uint32_t c = select_scan<kSelWarps>(counts_of(i0), scan, before);
            sure += c & 0xffffu;
            equal += c >> 16;
        }
        if (tid == 0) counts[0] = sure, counts[1] = equal;
        cluster.sync();
        for (uint32_t r = 0; r < rank; ++r) {
            at += cluster.map_shared_rank(counts, r)[0];
            ties += cluster.map_shared_rank(counts, r)[1];
        }
        at += min(ties, need);
    }
    for (int32_t i0 = first; i0 < end; i0 += kPiece) {
        if (!held) read(i0);
        const uint32_t c = counts_of(i0), sum = select_scan<kSelWarps>(c, scan, before);
        uint32_t t = ties + (before >> 16);  // slots with the smallest key before this thread's
        uint32_t pos = at + (before & 0xffffu) + (min(t, need) - min(ties, need));
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
            const int32_t i = i0 + int32_t(tid) * kOwn + e;
            const uint32_t k = order_key(v[e]);
            const bool between = i >= lo && i < hi, tie = between && any && k == prefix;
            const bool keep = i < end && (!between || (any && k > prefix) || (tie && t < need));
            if (i < end && tie) ++t;
            if (keep) {
                kept[pos] = i;
                if (nw) nw[pos] = v[e];
                ++pos;
            }
        }
        at += (sum & 0xffffu) + (min(ties + (sum >> 16), need) - min(ties, need));
        ties += sum >> 16;
    }
    if (CL > 1) cluster.sync();  // the others have read this CTA's shared memory
}

// Kept rows to the new pages: 16 bytes of a key and of a value per thread and
// row, kCopyRows rows under way at a time. 64 rows of 8192 kept slots: 89 us, 6.1
// TB/s in and out.
__global__ void __launch_bounds__(256) evict_copy_kernel(const EvictParams p) {
    tc::after_wait();
    const uint32_t pieces = p.D / 8, rows = 256 / pieces;  // rows of the block at a time
    const uint32_t chunks = (p.budget + rows * kCopyRows - 1) / (rows * kCopyRows);
    const uint32_t bh = blockIdx.x / chunks, b = bh / p.Hkv, h = bh % p.Hkv;
    const uint32_t j0 = blockIdx.x % chunks * (rows * kCopyRows) + threadIdx.x / pieces;
    const int64_t e = (threadIdx.x % pieces) * 8;
    int32_t i[kCopyRows], from[kCopyRows], to[kCopyRows];
#pragma unroll
    for (int x = 0; x < kCopyRows; ++x) {
        const uint32_t j = j0 + x * rows;
        i[x] = j < p.budget ? p.kept[int64_t(bh) * p.budget + j] : -1;
    }
#pragma unroll
    for (int x = 0; x < kCopyRows; ++x)
        if (i[x] >= 0) {
            from[x] = p.table[int64_t(b) * p.table_s + (i[x] >> p.pshift)];
            to[x] = p.new_table[int64_t(b) * p.new_table_s + ((j0 + x * rows) >> p.pshift)];
            if (uint32_t(from[x]) >= p.pages || uint32_t(to[x]) >= p.pages) {
                if (p.err) atomicOr(p.err, kErrPage);
                i[x] = -1;
            }
        }
    uint4 k[kCopyRows], v[kCopyRows];
#pragma unroll
    for (int x = 0; x < kCopyRows; ++x)
        if (i[x] >= 0) {
            const int64_t si = i[x] & int32_t(p.P - 1);
            const uint16_t* kf = p.k_pages + from[x] * p.kp_ps + si * p.kp_ss + h * p.kp_hs + e;
            const uint16_t* vf = p.v_pages + from[x] * p.vp_ps + si * p.vp_ss + h * p.vp_hs + e;
            k[x] = __ldcs(reinterpret_cast<const uint4*>(kf));
            v[x] = __ldcs(reinterpret_cast<const uint4*>(vf));
        }
#pragma unroll
    for (int x = 0; x < kCopyRows; ++x)
        if (i[x] >= 0) {
            const int64_t sj = (j0 + x * rows) & (p.P - 1);
            *reinterpret_cast<uint4*>(p.k_new + to[x] * p.kp_ps + sj * p.kp_ss + h * p.kp_hs + e) = k[x];
            *reinterpret_cast<uint4*>(p.v_new + to[x] * p.vp_ps + sj * p.vp_ss + h * p.vp_hs + e) = v[x];
        }
}

template <int CL, int kThreads>
cudaError_t launch_select(const EvictParams& p, cudaStream_t s) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CL;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.B * p.Hkv * CL);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, evict_select_kernel<CL, kThreads>, p);
}

}  // namespace
}  // namespace lsb

extern "C" int ls_b200_evict_cache(const ls_b200_evict_args* a, void* stream) {
    using namespace lsb;
    if (!a || !a->kv_heads || a->kv_heads > 65536 || (a->head_dim != 64 && a->head_dim != 128) || a->page_size < 16 ||
        a->page_size > 256 || (a->page_size & (a->page_size - 1)) || a->batch > (1u << 22) || !a->budget ||
        uint64_t(a->sinks) + a->recent > a->budget || uint64_t(a->table_pages) * a->page_size > kMaxSlots ||
        a->weights_length > kMaxSlots || a->pages > 0x7fffffffu ||
        uint64_t(a->new_table_pages) * a->page_size < a->budget || a->budget > kMaxSlots)
        return EINVAL;
    if (!a->batch) return 0;
    if (!a->k_pages || !a->v_pages || !a->page_table || !a->new_table || !a->kv_len || !a->weights || !a->kept ||
        !a->new_len || !a->pages || !a->table_pages)
        return EINVAL;
    for (const int64_t v :
         {a->k_page_stride, a->k_slot_stride, a->k_head_stride, a->v_page_stride, a->v_slot_stride, a->v_head_stride})
        if (v % 8 || v < 0) return EINVAL;
    if ((reinterpret_cast<uintptr_t>(a->k_pages) & 15u) || (reinterpret_cast<uintptr_t>(a->v_pages) & 15u))
        return EINVAL;
    EvictParams p{};
    p.k_pages = p.k_new = static_cast<uint16_t*>(a->k_pages);
    p.v_pages = p.v_new = static_cast<uint16_t*>(a->v_pages);
    p.table = a->page_table, p.kv_len = a->kv_len, p.new_table = a->new_table;
    p.weights = a->weights, p.new_weights = a->new_weights, p.kept = a->kept, p.new_len = a->new_len, p.err = a->error;
    p.kp_ps = a->k_page_stride, p.kp_ss = a->k_slot_stride, p.kp_hs = a->k_head_stride;
    p.vp_ps = a->v_page_stride, p.vp_ss = a->v_slot_stride, p.vp_hs = a->v_head_stride;
    p.table_s = a->table_stride, p.new_table_s = a->new_table_stride;
    p.w_ss = a->weights_sequence_stride, p.w_hs = a->weights_head_stride;
    p.B = a->batch, p.Hkv = a->kv_heads, p.D = a->head_dim, p.P = a->page_size, p.pages = a->pages;
    while ((1u << p.pshift) < p.P) ++p.pshift;
    p.tpages = a->table_pages, p.wlen = a->weights_length, p.budget = a->budget, p.sinks = a->sinks;
    p.recent = a->recent;
    const uint32_t per_block = 256 / (p.D / 8) * kCopyRows, chunks = (p.budget + per_block - 1) / per_block;
    if (uint64_t(p.B) * p.Hkv * (chunks > 8 ? chunks : 8) > 0x7fffffffull) return EINVAL;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // A cluster per row where a row may be longer than one CTA holds; of narrow
    // CTAs while they hold their stretch (four fit an SM: 64 rows of up to 32768
    // slots 29 us against 38), of wide ones where they read it again (8 rows of
    // 131072 slots 39 us against 56).
    cudaError_t e = p.wlen <= uint32_t(kShort)              ? launch_select<1, 512>(p, s)
                    : p.wlen <= uint32_t(kCluster * kShort) ? launch_select<kCluster, 256>(p, s)
                                                            : launch_select<kCluster, 512>(p, s);
    if (e == cudaSuccess) e = tc::launch_after(evict_copy_kernel, p.B * p.Hkv * chunks, 256, 0, s, p);
    return int(e);
}
