// kv_evict.cu -- requests of the paged cache that keep their first, their last
// and their heaviest tokens (specdec_kv_evict_pages).
//
// Three steps:
//   select  a CTA for each request: the request is checked, the `keep` tokens
//           that stay are found (the smallest of their weights' 32-bit keys, bits
//           from the top; ties to the lower slot) and listed in order, with the
//           first slot that another token moves into and the pages that have to be
//           replaced because others hold them;
//   tables  one CTA: all requests' errors, free pages for those replaced, then
//           tables, lengths and reference counts;
//   move    a CTA for each (request, layer, K or V of a head), and for each head
//           of the weights: rows move up in place.
// Up to 8 requests are selected by the CTAs of one cluster, whose first goes on
// with the tables: two launches.
//
// In place: token j of those that stay comes from slot kept[j] >= j, so what a
// chunk of tokens is written over has been read once the chunk itself is in
// registers.  The bytes of the tokens that move bound long requests, latency
// short ones.
#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace specdec {

constexpr int kEvictThreads = 1024, kEvictWarps = kEvictThreads / 32;  // of a CTA at most
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
template <int THREADS>
__device__ __forceinline__ int evict_scan(int v, int* sh, int* total) {
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
    int s = lane < THREADS / 32 ? sh[lane] : 0;
#pragma unroll
    for (int o = 1; o < THREADS / 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    *total = __shfl_sync(0xffffffffu, s, THREADS / 32 - 1);
    const int before = __shfl_sync(0xffffffffu, s, max(0, w - 1));
    return (w ? before : 0) + x - v;
}

// Order-preserving key of a token's weight: the heads' sum in 64 bits, rounded
// once (so that its order does not hang on the order of the sum), -0 as 0, NaN
// above all.
__device__ __forceinline__ uint32_t evict_key(double sum) {
    const float f = (float)sum + 0.0f;
    return f != f ? 0xFFFFFFFFu : logit_key(f);
}

constexpr int kEvictKeys = 8;  // of a thread, where a request's stay in registers
constexpr int kEvictCluster = 8;

struct EvictShared {
    int scan[kEvictWarps], hist[256], pick[2], hole, need;
    uint32_t count[2][kEvictWarps];
};

// The smallest key that stays, and how many of it: `want` of the keys, the largest
// first; 0 is no key.  From registers, two bits at a time: one barrier a round (a
// histogram of 256 digits has most of a request's keys in a few bins).
template <int THREADS>
__device__ __forceinline__ uint32_t evict_threshold(EvictShared& sh, const uint32_t (&k)[kEvictKeys], int want, int* ties) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    uint32_t tau = 0;
    int left = want;
    for (int shift = 30; shift >= 0; shift -= 2) {
        // keys with digits 3, 2, 1 under the bits known: 10 bits each (256 of a warp at most)
        uint32_t c = 0;
        const uint32_t known = tau >> shift;
#pragma unroll
        for (int u = 0; u < kEvictKeys; ++u) {
            const uint32_t d = min((k[u] >> shift) - known, 4u);
            uint32_t one;  // (shl gives 0 from 32 on; digit 0 counts into the two bits above)
            asm("shl.b32 %0, 1, %1;" : "=r"(one) : "r"(30u - 10u * d));
            c += one;
        }
        c = __reduce_add_sync(0xffffffffu, c);
        uint32_t* row = sh.count[(shift >> 1) & 1];
        if (lane == 0) row[w] = c;
        __syncthreads();
        const uint32_t x = lane < THREADS / 32 ? row[lane] : 0;
        const uint32_t hi = __reduce_add_sync(0xffffffffu, (x & 1023u) | ((x >> 10) & 1023u) << 16);
        const int c3 = (int)(hi & 0xFFFFu), c2 = (int)(hi >> 16), c1 = (int)__reduce_add_sync(0xffffffffu, (x >> 20) & 1023u);
        uint32_t digit = 3;
        if (left > c3) {
            left -= c3;
            digit = 2;
            if (left > c2) {
                left -= c2;
                digit = 1;
                if (left > c1) {
                    left -= c1;
                    digit = 0;
                }
            }
        }
        tau |= digit << shift;
    }
    *ties = left;
    return tau;
}

template <int THREADS>
__device__ __forceinline__ void evict_select(const EvictArgs& a, EvictShared& sh, int i) {
    const int tid = threadIdx.x;
    const int r = a.reqs[i];
    bool bad = r < 0 || r >= a.max_reqs;
    int nb = -1, L = 0;
    if (!bad) {
        nb = a.nblk[r];
        L = a.len[r];
        bad = nb < 0 || nb > a.max_bpr || L < 0 || L > (long long)nb * a.bs || L > a.ldw;
    }
    const bool sound = !bad;
    for (int j = tid; j < a.n; j += THREADS) bad |= j != i && a.reqs[j] == r;
    if (sound)
        for (int d = tid; d < nb; d += THREADS) {
            const int p = a.tables[(size_t)r * a.max_bpr + d];
            bad |= p < 0 || p >= a.num_blocks;
        }
    if (tid == 0) {
        sh.hole = a.keep;
        sh.need = 0;
    }
    // (the weights are on their way before all checks are known)
    const int lo = a.first, hi = L - a.last, want = a.keep - a.first - a.last;  // the others: slots lo .. hi - 1
    const float* w = a.w + (size_t)(sound ? r : 0) * a.wheads * a.ldw;
    const bool small = L <= kEvictKeys * THREADS;
    const int j0 = kEvictKeys * tid;
    uint32_t k[kEvictKeys], real = 0;
    if (sound && L > a.keep && small && want > 0) {
        double sum[kEvictKeys];
#pragma unroll
        for (int u = 0; u < kEvictKeys; ++u) {
            sum[u] = 0.0;
            if (j0 + u >= lo && j0 + u < hi) real |= 1u << u;
        }
        if (real) {
            // whole 32-byte runs where they are aligned, so that all heads' loads go out together
            const bool wide = (a.ldw & 3) == 0 && (reinterpret_cast<uintptr_t>(a.w) & 15) == 0 && j0 + kEvictKeys <= a.ldw;
            if (wide) {
#pragma unroll 4
                for (int h = 0; h < a.wheads; ++h) {
                    const float4* src = reinterpret_cast<const float4*>(w + (size_t)h * a.ldw + j0);
                    const float4 x = src[0], y = src[1];
                    sum[0] += x.x, sum[1] += x.y, sum[2] += x.z, sum[3] += x.w;
                    sum[4] += y.x, sum[5] += y.y, sum[6] += y.z, sum[7] += y.w;
                }
            } else {
                for (int h = 0; h < a.wheads; ++h)
#pragma unroll
                    for (int u = 0; u < kEvictKeys; ++u) sum[u] += w[(size_t)h * a.ldw + min(j0 + u, a.ldw - 1)];
            }
        }
#pragma unroll
        for (int u = 0; u < kEvictKeys; ++u) k[u] = (real >> u) & 1u ? evict_key(sum[u]) : 0u;
    }
    bad = __syncthreads_or(bad);
    const bool gone = !bad && L > a.keep;
    int32_t* user = a.kept ? a.kept + (size_t)i * a.keep : nullptr;
    if (!gone) {
        if (user)
            for (int j = tid; j < a.keep; j += THREADS) user[j] = !bad && j < L ? j : -1;
        if (tid == 0) a.req[i] = {bad, 0, a.keep, 0, a.keep};
        return;
    }
    int32_t* list = a.list + (size_t)i * a.list_len;
    int hole = a.keep, tot;
    if (small) {
        uint32_t tau = 0xFFFFFFFFu;
        int ties = 0;
        if (want > 0) tau = evict_threshold<THREADS>(sh, k, want, &ties);
        uint32_t stay = 0, tie = 0;
#pragma unroll
        for (int u = 0; u < kEvictKeys; ++u) {
            const int j = j0 + u;
            const bool other = j >= lo && j < hi;
            if (j < L && !other) stay |= 1u << u;
            if (other && want > 0) {
                if (k[u] > tau) stay |= 1u << u;
                if (k[u] == tau) tie |= 1u << u;
            }
        }
        // both sums in one, 16 bits each (8192 slots at most)
        const int before = evict_scan<THREADS>(__popc(stay) | __popc(tie) << 16, sh.scan, &tot);
        int ahead = before & 0xFFFF, tied = before >> 16;
#pragma unroll
        for (int u = 0; u < kEvictKeys; ++u) {
            const int place = ahead + min(tied, ties), j = j0 + u;
            const bool is_tie = (tie >> u) & 1u, is_in = ((stay >> u) & 1u) || (is_tie && tied < ties);
            if (is_in) {
                list[place] = j;
                if (user) user[place] = j;
                if (j != place) hole = min(hole, place);
            }
            ahead += (stay >> u) & 1u;
            tied += is_tie;
        }
    } else {
        uint32_t* keys = a.keys + (size_t)i * a.slots;
        for (int j = lo + tid; j < hi; j += THREADS) {
            double sum = 0.0;
#pragma unroll 4
            for (int h = 0; h < a.wheads; ++h) sum += w[(size_t)h * a.ldw + j];
            keys[j] = evict_key(sum);
        }
        uint32_t tau = 0;
        int ties = want;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) sh.hist[tid] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += THREADS) {
                const uint32_t x = keys[j];
                if (shift == 24 || (x >> (shift + 8)) == (tau >> (shift + 8))) atomicAdd(&sh.hist[(x >> shift) & 255], 1);
            }
            __syncthreads();
            const int c = tid < 256 ? sh.hist[255 - tid] : 0;
            const int above = evict_scan<THREADS>(c, sh.scan, &tot);
            if (c && above < ties && above + c >= ties) {
                sh.pick[0] = 255 - tid;
                sh.pick[1] = above;
            }
            __syncthreads();
            if (want > 0) {
                tau |= (uint32_t)sh.pick[0] << shift;
                ties -= sh.pick[1];
            }
            __syncthreads();
        }
        // the list: the thread's slots are neighbours, tile by tile
        int out = 0, taken = 0;
        for (int t0 = 0; t0 < L; t0 += 4 * THREADS) {
            int stay[4], tie[4], nt = 0, ns = 0;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = t0 + 4 * tid + u;
                const bool other = j >= lo && j < hi;
                const uint32_t x = other && want > 0 ? keys[j] : 0;
                tie[u] = other && want > 0 && x == tau;
                stay[u] = j < L && (!other || (want > 0 && x > tau));
                nt += tie[u];
            }
            int before = taken + evict_scan<THREADS>(nt, sh.scan, &tot);
            taken += tot;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (tie[u] && before++ < ties) stay[u] = 1;
                ns += stay[u];
            }
            int place = out + evict_scan<THREADS>(ns, sh.scan, &tot);
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
    }
    if (hole < a.keep) atomicMin(&sh.hole, hole);
    __syncthreads();
    hole = sh.hole;
    const int d0 = hole / a.bs, d1 = (a.keep + a.bs - 1) / a.bs;
    int need = 0;
    int32_t* old = a.old + (size_t)i * a.max_bpr;
    for (int d = tid; d < nb; d += THREADS) {
        const int p = a.tables[(size_t)r * a.max_bpr + d];
        const bool swap = hole < a.keep && d >= d0 && d < d1 && a.ref[p] > 1;
        old[d] = swap ? ~p : p;
        need += swap;
    }
    if (need) atomicAdd(&sh.need, need);
    __syncthreads();
    if (tid == 0) {
        const bool first_page = hole < a.keep && old[d0] < 0;  // (written by some thread before the barrier)
        a.req[i] = {0, 1, hole, sh.need, first_page ? d0 * a.bs : hole};
    }
}

template <int THREADS>
__device__ __forceinline__ void evict_tables(const EvictArgs& a, int* sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    bool bad = false;
    int need = 0;
    for (int i = tid; i < a.n; i += THREADS) {
        bad |= a.req[i].bad != 0;
        need += a.req[i].need;
    }
    bad = __syncthreads_or(bad);
    int total;
    (void)evict_scan<THREADS>(need, sh, &total);
    if (bad) {
        if (tid == 0) {
            *a.go = 0;
            *a.status = SPECDEC_EINVAL;
        }
        return;
    }
    if (total > 0) {  // the lowest free pages, in order
        int got = 0;
        for (int b0 = 0; b0 < a.num_blocks && got < total; b0 += THREADS) {
            const int b = b0 + tid;
            const int is_free = b < a.num_blocks && a.ref[b] == 0;
            int tot;
            const int before = got + evict_scan<THREADS>(is_free, sh, &tot);
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
    for (int i = warp; i < a.n; i += THREADS / 32) {
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

// PHASE 0: both steps of up to kEvictCluster requests, by a cluster (CTAS > 1) or a CTA; 1 and 2: one of them.
template <int PHASE, int CTAS, int THREADS>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS)
    kv_evict_plan_kernel(const __grid_constant__ EvictArgs a) {
    __shared__ EvictShared sh;
    pdl_trigger();
    if constexpr (PHASE == 2) pdl_wait();
    if (PHASE < 2 && (int)blockIdx.x < a.n) evict_select<THREADS>(a, sh, blockIdx.x);
    if constexpr (PHASE == 0) {
        if constexpr (CTAS > 1) cluster_sync_all();
        else __syncthreads();
    }
    if (PHASE != 1 && blockIdx.x == 0) evict_tables<THREADS>(a, sh.scan);
}

// x < 2 * Hkv: K or V of a head of layer y; above: a head of the weights.
__global__ void __launch_bounds__(kMoveThreads) kv_evict_move_kernel(const __grid_constant__ EvictArgs a, __half* kv,
                                                                     size_t layer_stride, int Hkv, int hd, int planes) {
    const int i = blockIdx.z, x = blockIdx.x, tid = threadIdx.x;
    pdl_wait();
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
    cudaLaunchConfig_t cfg = {};
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    // No more threads than the tables' slots need: a barrier of 32 warps takes twice one of 8.
    const int threads = a.slots <= 256 * kEvictKeys ? 256 : a.slots <= 512 * kEvictKeys ? 512 : kEvictThreads;
    const int kind = n == 1 ? 0 : n <= kEvictCluster ? 1 : 2;
#define EVICT_PLAN(t)                                                                    \
    (kind == 0 ? kv_evict_plan_kernel<0, 1, t>                                           \
               : kind == 1 ? kv_evict_plan_kernel<0, kEvictCluster, t> : kv_evict_plan_kernel<1, 1, t>)
    const auto plan = threads == 256 ? EVICT_PLAN(256) : threads == 512 ? EVICT_PLAN(512) : EVICT_PLAN(kEvictThreads);
#undef EVICT_PLAN
    plan<<<kind == 1 ? kEvictCluster : n, threads, 0, s>>>(a);
    SD_LAUNCH_CHECK("kv_evict_plan_kernel");
    if (kind == 2) {
        cfg.gridDim = dim3(1);
        cfg.blockDim = dim3(kEvictThreads);
        SD_CUDA(cudaLaunchKernelEx(&cfg, kv_evict_plan_kernel<2, 1, kEvictThreads>, a));
    }
    const int planes = layers > 0 ? 2 * Hkv : 0;
    cfg.gridDim = dim3((unsigned)(planes + wheads), (unsigned)std::max(1, layers), (unsigned)n);
    cfg.blockDim = dim3(kMoveThreads);
    SD_CUDA(cudaLaunchKernelEx(&cfg, kv_evict_move_kernel, a, kv, layer_stride, Hkv, hd, planes));
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
