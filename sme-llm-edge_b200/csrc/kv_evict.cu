// kv_evict.cu -- requests of the paged cache that keep their first, their last
// and their heaviest tokens (specdec_kv_evict_pages).
//
// Three launches:
//   select  a CTA for each request: the request is checked, the `keep` tokens
//           that stay are found (a radix select over the weights' 32-bit keys,
//           ties to the lower slot) and listed in order, with the first slot
//           that another token moves into and the pages that have to be replaced
//           because others hold them;
//   tables  one CTA: all requests' errors, free pages for those replaced, then
//           tables, lengths and reference counts;
//   move    a CTA for each (request, layer, K or V of a head), and for each head
//           of the weights: rows move up in place.
//
// In place: token j of those that stay comes from slot kept[j] >= j, so what a
// chunk of tokens is written over has been read once the chunk itself is in
// registers.  The bytes of the tokens that move bound long requests, latency
// short ones.
#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace specdec {

constexpr int kEvictThreads = 1024, kEvictWarps = kEvictThreads / 32;
constexpr int kMoveThreads = 256;

struct EvictReq {
    int bad;   // an argument is not in order
    int gone;  // tokens leave
    int hole;  // first slot that another token moves into (keep: none)
    int need;  // pages to replace
    int from;  // first slot that is written
};

struct EvictArgs {
    int32_t* tables;
    int32_t* nblk;
    int32_t* len;
    int32_t* ref;
    int num_blocks, max_reqs, max_bpr, bs;
    const int32_t* reqs;
    int n, keep, first, last;
    float* w;
    int wheads, ldw;
    int32_t* kept;  // the caller's, may be null
    int32_t* status;
    // workspace
    int32_t* go;       // 1: the move may run
    EvictReq* req;     // [n]
    uint32_t* keys;    // [n][slots]
    int32_t* list;     // [n][list_len] tokens that stay
    int32_t* old;      // [n][max_bpr] pages before; ~page: to be replaced
    int32_t* fresh;    // free pages taken
    int list_len;
    size_t slots;
};

// Exclusive sum over the CTA; every thread gets the total.
__device__ int evict_scan(int v, int* sh, int* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) sh[w] = x;
    __syncthreads();
    int s = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    *total = __shfl_sync(0xffffffffu, s, 31);
    const int before = __shfl_sync(0xffffffffu, s, max(0, w - 1));
    return (w ? before : 0) + x - v;
}

// Order-preserving key of a token's weight: the heads' sum in 64 bits, rounded
// once (so that its order does not hang on the order of the sum), -0 as 0, NaN
// above all.
__device__ __forceinline__ uint32_t evict_key(const float* w, int heads, size_t ldw) {
    double s = 0.0;
    for (int h = 0; h < heads; ++h) s += (double)w[h * ldw];
    const float f = (float)s + 0.0f;
    return f != f ? 0xFFFFFFFFu : logit_key(f);
}

__global__ void __launch_bounds__(kEvictThreads) kv_evict_select_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ int sh[kEvictWarps], hist[256], pick[2], hole_s, need_s;
    const int i = blockIdx.x, tid = threadIdx.x;
    const int r = a.reqs[i];
    bool bad = r < 0 || r >= a.max_reqs;
    int nb = -1, L = 0;
    if (!bad) {
        nb = a.nblk[r];
        L = a.len[r];
        bad = nb < 0 || nb > a.max_bpr || L < 0 || L > (long long)nb * a.bs || L > a.ldw;
    }
    for (int j = tid; j < a.n; j += kEvictThreads) bad |= j != i && a.reqs[j] == r;
    bad = __syncthreads_or(bad);
    if (!bad) {
        for (int d = tid; d < nb; d += kEvictThreads) {
            const int p = a.tables[(size_t)r * a.max_bpr + d];
            bad |= p < 0 || p >= a.num_blocks;
        }
        bad = __syncthreads_or(bad);
    }
    const bool gone = !bad && L > a.keep;
    int32_t* user = a.kept ? a.kept + (size_t)i * a.keep : nullptr;
    if (!gone) {
        if (user)
            for (int j = tid; j < a.keep; j += kEvictThreads) user[j] = !bad && j < L ? j : -1;
        if (tid == 0) a.req[i] = {bad, 0, a.keep, 0, a.keep};
        return;
    }
    int32_t* list = a.list + (size_t)i * a.list_len;
    uint32_t* keys = a.keys + (size_t)i * a.slots;
    const int lo = a.first, hi = L - a.last, want = a.keep - a.first - a.last;  // the others: slots lo .. hi - 1
    for (int j = lo + tid; j < hi; j += kEvictThreads)
        keys[j] = evict_key(a.w + (size_t)r * a.wheads * a.ldw + j, a.wheads, a.ldw);
    // the smallest key that stays, and how many of it
    uint32_t tau = 0;
    int ties = want;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int j = lo + tid; j < hi; j += kEvictThreads) {
            const uint32_t k = keys[j];
            if (shift == 24 || (k >> (shift + 8)) == (tau >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        int tot;
        const int c = tid < 256 ? hist[255 - tid] : 0;
        const int above = evict_scan(c, sh, &tot);
        if (c && above < ties && above + c >= ties) {
            pick[0] = 255 - tid;
            pick[1] = above;
        }
        __syncthreads();
        if (want > 0) {
            tau |= (uint32_t)pick[0] << shift;
            ties -= pick[1];
        }
        __syncthreads();
    }
    if (tid == 0) {
        hole_s = a.keep;
        need_s = 0;
    }
    __syncthreads();
    // the list: the thread's slots are neighbours, tile by tile
    int out = 0, taken = 0, hole = a.keep;
    for (int t0 = 0; t0 < L; t0 += 4 * kEvictThreads) {
        int stay[4], tie[4], nt = 0, ns = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = t0 + 4 * tid + u;
            const bool other = j >= lo && j < hi;
            const uint32_t k = other && want > 0 ? keys[j] : 0;
            tie[u] = other && want > 0 && k == tau;
            stay[u] = j < L && (!other || (want > 0 && k > tau));
            nt += tie[u];
        }
        int tot;
        int before = taken + evict_scan(nt, sh, &tot);
        taken += tot;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (tie[u] && before++ < ties) stay[u] = 1;
            ns += stay[u];
        }
        int place = out + evict_scan(ns, sh, &tot);
        out += tot;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (!stay[u]) continue;
            const int j = t0 + 4 * tid + u;
            list[place] = j;
            if (user) user[place] = j;
            if (j != place) hole = min(hole, place);
            ++place;
        }
    }
    if (hole < a.keep) atomicMin(&hole_s, hole);
    __syncthreads();
    hole = hole_s;
    const int d0 = hole / a.bs, d1 = (a.keep + a.bs - 1) / a.bs;
    int need = 0;
    int32_t* old = a.old + (size_t)i * a.max_bpr;
    for (int d = tid; d < nb; d += kEvictThreads) {
        const int p = a.tables[(size_t)r * a.max_bpr + d];
        const bool swap = hole < a.keep && d >= d0 && d < d1 && a.ref[p] > 1;
        old[d] = swap ? ~p : p;
        need += swap;
    }
    if (need) atomicAdd(&need_s, need);
    __syncthreads();
    if (tid == 0) {
        const bool first_page = hole < a.keep && old[d0] < 0;  // (written by some thread before the barrier)
        a.req[i] = {0, 1, hole, need_s, first_page ? d0 * a.bs : hole};
    }
}

__global__ void __launch_bounds__(kEvictThreads) kv_evict_tables_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ int sh[kEvictWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    bool bad = false;
    int need = 0;
    for (int i = tid; i < a.n; i += kEvictThreads) {
        bad |= a.req[i].bad != 0;
        need += a.req[i].need;
    }
    bad = __syncthreads_or(bad);
    int total;
    (void)evict_scan(need, sh, &total);
    if (bad) {
        if (tid == 0) {
            *a.go = 0;
            *a.status = SPECDEC_EINVAL;
        }
        return;
    }
    if (total > 0) {  // the lowest free pages, in order
        int got = 0;
        for (int b0 = 0; b0 < a.num_blocks && got < total; b0 += kEvictThreads) {
            const int b = b0 + tid;
            const int is_free = b < a.num_blocks && a.ref[b] == 0;
            int tot;
            const int before = got + evict_scan(is_free, sh, &tot);
            if (is_free && before < total) a.fresh[before] = b;
            got += tot;
        }
        if (got < total) {
            if (tid == 0) {
                *a.go = 0;
                *a.status = SPECDEC_ENOMEM;
            }
            return;
        }
    }
    __syncthreads();
    // a warp for each request
    const int pages = (a.keep + a.bs - 1) / a.bs;
    for (int i = warp; i < a.n; i += kEvictWarps) {
        if (!a.req[i].gone) continue;
        const int r = a.reqs[i], nb = a.nblk[r];
        int at = 0;  // fresh pages of the requests before
        for (int k = lane; k < i; k += 32) at += a.req[k].need;
        at = warp_sum(at);
        const int32_t* old = a.old + (size_t)i * a.max_bpr;
        int32_t* tab = a.tables + (size_t)r * a.max_bpr;
        for (int d0 = 0; d0 < nb; d0 += 32) {
            const int d = d0 + lane, p = d < nb ? old[d] : 0;
            const bool swap = d < nb && p < 0;
            const uint32_t m = __ballot_sync(0xffffffffu, swap);
            if (swap) {
                const int f = a.fresh[at + __popc(m & ((1u << lane) - 1))];
                tab[d] = f;
                a.ref[f] = 1;
                atomicSub(&a.ref[~p], 1);
            } else if (d < nb && d >= pages) {
                tab[d] = -1;
                atomicSub(&a.ref[p], 1);
            }
            at += __popc(m);
        }
        __syncwarp();
        if (lane == 0) {
            a.nblk[r] = pages;
            a.len[r] = a.keep;
        }
    }
    if (tid == 0) {
        *a.go = 1;
        *a.status = SPECDEC_OK;
    }
}

// x < 2 * Hkv: K or V of a head of layer y; above: a head of the weights.
__global__ void __launch_bounds__(kMoveThreads) kv_evict_move_kernel(const __grid_constant__ EvictArgs a, __half* kv,
                                                                     size_t layer_stride, int Hkv, int hd, int planes) {
    const int i = blockIdx.z, x = blockIdx.x, tid = threadIdx.x;
    if (!*a.go) return;
    const EvictReq q = a.req[i];
    if (!q.gone) return;
    const int r = a.reqs[i];
    const int32_t* list = a.list + (size_t)i * a.list_len;
    if (x >= planes) {
        if (blockIdx.y) return;
        float* w = a.w + ((size_t)r * a.wheads + (x - planes)) * a.ldw;
        for (int j0 = q.hole; j0 < a.keep; j0 += 4 * kMoveThreads) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = j0 + u * kMoveThreads + tid;
                if (j < a.keep) v[u] = w[list[j]];
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = j0 + u * kMoveThreads + tid;
                if (j < a.keep) w[j] = v[u];
            }
        }
        __syncthreads();
        for (int j = a.keep + tid; j < a.ldw; j += kMoveThreads) w[j] = 0.f;
        return;
    }
    if (q.hole >= a.keep) return;
    const int32_t* old = a.old + (size_t)i * a.max_bpr;
    const int32_t* tab = a.tables + (size_t)r * a.max_bpr;
    const int pieces = hd / 8, per = kMoveThreads / pieces, e = tid % pieces, t = tid / pieces;
    __half* base = kv + layer_stride * blockIdx.y + (size_t)x * 16 * hd + 8 * e;
    const size_t page = (size_t)2 * Hkv * 16 * hd;
    for (int j0 = q.from; j0 < a.keep; j0 += 4 * per) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = j0 + u * per + t;
            if (t < per && j < a.keep) {
                const int s = list[j], p = old[s >> 4];
                v[u] = *reinterpret_cast<const uint4*>(base + page * (p < 0 ? ~p : p) + (s & 15) * hd);
            }
        }
        __syncthreads();  // what these tokens are written over has been read
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = j0 + u * per + t;
            if (t < per && j < a.keep) *reinterpret_cast<uint4*>(base + page * tab[j >> 4] + (j & 15) * hd) = v[u];
        }
    }
}

static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }
static int evict_list_len(int keep, size_t slots) { return (int)std::min<size_t>((size_t)keep, slots); }

size_t kv_evict_workspace(int max_bpr, int block_size, int n, int keep) {
    const size_t slots = (size_t)max_bpr * block_size, N = (size_t)n;
    return 256 + up256(N * sizeof(EvictReq)) + up256(N * slots * 4) + up256(N * evict_list_len(keep, slots) * 4) +
           up256(N * max_bpr * 4) + up256(N * max_bpr * 4);
}

int kv_evict_launch(const KVState& st, const int32_t* reqs, int n, int keep, int first, int last, float* weights,
                    int wheads, int ldw, __half* kv, int layers, size_t layer_stride, int Hkv, int hd, int32_t* kept,
                    int32_t* status, void* ws, cudaStream_t s) {
    EvictArgs a = {};
    a.tables = st.tables;
    a.nblk = st.nblk;
    a.len = st.len;
    a.ref = st.ref;
    a.num_blocks = st.num_blocks;
    a.max_reqs = st.max_reqs;
    a.max_bpr = st.max_bpr;
    a.bs = st.block_size;
    a.reqs = reqs;
    a.n = n;
    a.keep = keep;
    a.first = first;
    a.last = last;
    a.w = weights;
    a.wheads = wheads;
    a.ldw = ldw;
    a.kept = kept;
    a.status = status;
    a.slots = (size_t)st.max_bpr * st.block_size;
    a.list_len = evict_list_len(keep, a.slots);
    char* w = static_cast<char*>(ws);
    a.go = reinterpret_cast<int32_t*>(w);
    w += 256;
    a.req = reinterpret_cast<EvictReq*>(w);
    w += up256((size_t)n * sizeof(EvictReq));
    a.keys = reinterpret_cast<uint32_t*>(w);
    w += up256((size_t)n * a.slots * 4);
    a.list = reinterpret_cast<int32_t*>(w);
    w += up256((size_t)n * a.list_len * 4);
    a.old = reinterpret_cast<int32_t*>(w);
    w += up256((size_t)n * st.max_bpr * 4);
    a.fresh = reinterpret_cast<int32_t*>(w);
    kv_evict_select_kernel<<<n, kEvictThreads, 0, s>>>(a);
    SD_LAUNCH_CHECK("kv_evict_select_kernel");
    kv_evict_tables_kernel<<<1, kEvictThreads, 0, s>>>(a);
    SD_LAUNCH_CHECK("kv_evict_tables_kernel");
    const int planes = layers > 0 ? 2 * Hkv : 0;
    const dim3 grid((unsigned)(planes + wheads), (unsigned)std::max(1, layers), (unsigned)n);
    kv_evict_move_kernel<<<grid, kMoveThreads, 0, s>>>(a, kv, layer_stride, Hkv, hd, planes);
    SD_LAUNCH_CHECK("kv_evict_move_kernel");
    return SPECDEC_OK;
}

int kv_evict_check(const char* who, int max_reqs, int n, int keep, int first, int last, const float* weights, int wheads,
                   int ldw) {
    const std::string w(who);
    SD_CHECK(n >= 0 && n <= max_reqs && n <= 65535, SPECDEC_EINVAL, w + ": 0 to max_reqs requests, at most 65535");
    SD_CHECK(keep >= 1 && first >= 0 && last >= 0 && first <= keep && last <= keep - first, SPECDEC_EINVAL,
             w + ": keep at least one token, and at least the first and the last");
    SD_CHECK(n == 0 || weights, SPECDEC_EINVAL, w + ": null argument");
    SD_CHECK(wheads >= 1 && wheads <= 1024 && ldw >= 1, SPECDEC_EINVAL, w + ": 1 to 1024 heads of weights, ldw at least 1");
    return SPECDEC_OK;
}

}  // namespace specdec

using namespace specdec;

extern "C" size_t specdec_kv_evict_pages_workspace_bytes(int num_blocks, int max_reqs, int max_blocks, int n, int keep) {
    if (num_blocks <= 0 || max_reqs <= 0 || max_blocks <= 0 || n < 0 || keep < 1) return 0;
    return kv_evict_workspace(max_blocks, 16, n, keep);
}

extern "C" int specdec_kv_evict_pages(int32_t* tables, int32_t* n_blocks, int32_t* lens, int32_t* refcounts,
                                      int num_blocks, int max_reqs, int max_blocks, const int32_t* reqs, int n,
                                      int keep, int first, int last, float* weights, int weight_heads, int ldw,
                                      uint16_t* kv, int layers, size_t layer_stride, int n_kv_heads, int head_dim,
                                      int32_t* kept, int32_t* status, void* workspace, size_t workspace_bytes,
                                      void* stream) {
    SD_CHECK(tables && n_blocks && lens && refcounts && status && (n <= 0 || reqs), SPECDEC_EINVAL,
             "kv_evict_pages: null argument");
    SD_CHECK(num_blocks > 0 && max_reqs > 0 && max_blocks > 0 && max_blocks <= (1 << 26), SPECDEC_EINVAL,
             "kv_evict_pages: bad sizes");
    int rc = kv_evict_check("kv_evict_pages", max_reqs, n, keep, first, last, weights, weight_heads, ldw);
    if (!rc) rc = kv_fork_check_pool("kv_evict_pages", kv, layers, layer_stride, num_blocks, n_kv_heads, head_dim);
    if (rc) return rc;
    SD_CHECK(workspace && workspace_bytes >= kv_evict_workspace(max_blocks, 16, n, keep) &&
                 (reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
             SPECDEC_EINVAL, "kv_evict_pages: workspace too small or not 16-byte aligned");
    const struct {
        const void* p;
        const char* what;
    } given[] = {{tables, "kv_evict_pages: tables"},
                 {n_blocks, "kv_evict_pages: n_blocks"},
                 {lens, "kv_evict_pages: lens"},
                 {refcounts, "kv_evict_pages: refcounts"},
                 {status, "kv_evict_pages: status"},
                 {workspace, "kv_evict_pages: the workspace"},
                 {n ? (const void*)reqs : tables, "kv_evict_pages: reqs"},
                 {n ? (const void*)weights : tables, "kv_evict_pages: weights"},
                 {kept && n ? (const void*)kept : tables, "kv_evict_pages: kept"},
                 {layers ? (const void*)kv : tables, "kv_evict_pages: the pool"}};
    for (const auto& g : given)
        if ((rc = check_on_device(g.p, g.what))) return rc;
    cudaStream_t s = as_stream(stream);
    if (n == 0) {
        SD_CUDA(cudaMemsetAsync(status, 0, sizeof(int32_t), s));
        return SPECDEC_OK;
    }
    KVState st = {};
    st.num_blocks = num_blocks;
    st.block_size = 16;
    st.max_reqs = max_reqs;
    st.max_bpr = max_blocks;
    st.tables = tables;
    st.nblk = n_blocks;
    st.len = lens;
    st.ref = refcounts;
    return kv_evict_launch(st, reqs, n, keep, first, last, weights, weight_heads, ldw, reinterpret_cast<__half*>(kv),
                           layers, layer_stride, n_kv_heads, head_dim, kept, status, workspace, s);
}
