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
// bound by memory.
#include <stdint.h>

#include <cerrno>

#include "ls_attention.h"
#include "ls_tc.h"

namespace lsb {
namespace {

constexpr int kSelThreads = 1024;

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

// One CTA per (sequence, kv head). The budget's smallest kept key is found
// eight bits at a time from the top (a histogram of the keys that share the
// bits found so far), then the kept slots are written in order.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
    __shared__ uint32_t hist[256], warp_gt[32], warp_eq[32], found[2];
    tc::after_start();
    const uint32_t b = blockIdx.x / p.Hkv, h = blockIdx.x % p.Hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t n = evict_len(p, b);
    const float* w = p.weights + int64_t(b) * p.w_ss + int64_t(h) * p.w_hs;
    int32_t* kept = p.kept + int64_t(blockIdx.x) * p.budget;
    float* nw = p.new_weights ? p.new_weights + int64_t(blockIdx.x) * p.budget : nullptr;
    if (h == 0 && tid == 0) p.new_len[b] = min(n, int32_t(p.budget));
    if (n <= int32_t(p.budget)) {
        for (uint32_t j = tid; j < p.budget; j += kSelThreads) {
            kept[j] = int32_t(j) < n ? int32_t(j) : -1;
            if (nw) nw[j] = int32_t(j) < n ? w[j] : 0.f;
        }
        return;
    }
    const int32_t lo = int32_t(p.sinks), hi = n - int32_t(p.recent);
    uint32_t need = p.budget - p.sinks - p.recent;  // slots to take between
    uint32_t prefix = 0, mask = 0;
    if (need) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int32_t i = lo + int32_t(tid); i < hi; i += kSelThreads) {
                const uint32_t k = order_key(w[i]);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (warp == 0) {  // the digit in which the need-th largest key lies
                uint32_t own = 0;
                for (int i = 0; i < 8; ++i) own += hist[255 - (lane * 8 + i)];
                uint32_t inc = own;
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t x = __shfl_up_sync(0xffffffffu, inc, o);
                    if (int(lane) >= o) inc += x;
                }
                uint32_t before = inc - own;
                if (before < need && need <= inc) {
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t d = 255 - (lane * 8 + i);
                        if (need <= before + hist[d]) {
                            found[0] = d;
                            found[1] = need - before;
                            break;
                        }
                        before += hist[d];
                    }
                }
            }
            __syncthreads();
            prefix |= found[0] << shift;
            mask |= 255u << shift;
            need = found[1];
        }
    }
    const bool any = p.budget > p.sinks + p.recent;
    // prefix is the smallest kept key, of which the first `need` are kept
    uint32_t at = 0, ties = 0;
    for (int32_t i0 = 0; i0 < n; i0 += kSelThreads) {
        const int32_t i = i0 + int32_t(tid);
        bool gt = i < n && (i < lo || i >= hi), eq = false;
        float v = 0.f;
        if (i < n) v = w[i];
        if (any && i >= lo && i < hi) {
            const uint32_t k = order_key(v);
            gt = k > prefix;
            eq = k == prefix;
        }
        const uint32_t me = __ballot_sync(0xffffffffu, eq), below = (1u << lane) - 1;
        if (lane == 0) warp_eq[warp] = __popc(me);
        __syncthreads();
        uint32_t before = ties, all = 0;
        for (uint32_t x = 0; x < 32; ++x) {
            if (x < warp) before += warp_eq[x];
            all += warp_eq[x];
        }
        const bool keep = gt || (eq && before + __popc(me & below) < need);
        ties += all;
        const uint32_t mk = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) warp_gt[warp] = __popc(mk);
        __syncthreads();
        uint32_t pos = at, total = 0;
        for (uint32_t x = 0; x < 32; ++x) {
            if (x < warp) pos += warp_gt[x];
            total += warp_gt[x];
        }
        pos += __popc(mk & below);
        if (keep && pos < p.budget) {
            kept[pos] = i;
            if (nw) nw[pos] = v;
        }
        at += total;
        __syncthreads();
    }
}

// Kept rows to the new pages: 16 bytes of a key and of a value per thread.
__global__ void __launch_bounds__(256) evict_copy_kernel(const EvictParams p) {
    tc::after_wait();
    const uint32_t pieces = p.D / 8, per_block = 256 / pieces;
    const uint32_t chunks = (p.budget + per_block - 1) / per_block;
    const uint32_t bh = blockIdx.x / chunks, b = bh / p.Hkv, h = bh % p.Hkv;
    const uint32_t j = blockIdx.x % chunks * per_block + threadIdx.x / pieces;
    const int64_t e = (threadIdx.x % pieces) * 8;
    if (j >= p.budget) return;
    const int32_t i = p.kept[int64_t(bh) * p.budget + j];
    if (i < 0) return;
    const int32_t from = p.table[int64_t(b) * p.table_s + (i >> p.pshift)];
    const int32_t to = p.new_table[int64_t(b) * p.new_table_s + (j >> p.pshift)];
    if (uint32_t(from) >= p.pages || uint32_t(to) >= p.pages) {
        if (p.err) atomicOr(p.err, kErrPage);
        return;
    }
    const int64_t si = i & int32_t(p.P - 1), sj = j & (p.P - 1);
    const uint4 k = *reinterpret_cast<const uint4*>(p.k_pages + from * p.kp_ps + si * p.kp_ss + h * p.kp_hs + e);
    const uint4 v = *reinterpret_cast<const uint4*>(p.v_pages + from * p.vp_ps + si * p.vp_ss + h * p.vp_hs + e);
    *reinterpret_cast<uint4*>(p.k_new + to * p.kp_ps + sj * p.kp_ss + h * p.kp_hs + e) = k;
    *reinterpret_cast<uint4*>(p.v_new + to * p.vp_ps + sj * p.vp_ss + h * p.vp_hs + e) = v;
}

}  // namespace
}  // namespace lsb

extern "C" int ls_b200_evict_cache(const ls_b200_evict_args* a, void* stream) {
    using namespace lsb;
    if (!a || !a->kv_heads || a->kv_heads > 65536 || (a->head_dim != 64 && a->head_dim != 128) || a->page_size < 16 ||
        a->page_size > 256 || (a->page_size & (a->page_size - 1)) || a->batch > (1u << 22) || !a->budget ||
        uint64_t(a->sinks) + a->recent > a->budget || uint64_t(a->table_pages) * a->page_size > 0x7fffff00ull ||
        a->weights_length > 0x7fffff00u || a->pages > 0x7fffffffu ||
        uint64_t(a->new_table_pages) * a->page_size < a->budget || a->budget > 0x7fffff00u)
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
    const uint32_t per_block = 256 / (p.D / 8), chunks = (p.budget + per_block - 1) / per_block;
    if (uint64_t(p.B) * p.Hkv * chunks > 0x7fffffffull) return EINVAL;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    evict_select_kernel<<<p.B * p.Hkv, kSelThreads, 0, s>>>(p);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return int(e);
    return int(tc::launch_after(evict_copy_kernel, p.B * p.Hkv * chunks, 256, 0, s, p));
}
