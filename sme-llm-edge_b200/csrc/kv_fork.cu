// kv_fork.cu -- requests of the paged cache that become copies of others.
//
// A fork shares the source's whole blocks by reference count and copies the
// used rows of its block in use, in every layer, into a block of the copy's
// own (the lowest free ones, in the order of the call); the blocks that the
// copy's slot held before are released first.  Either all forks of a call
// happen or none.
//
// Two launches: the tables by one CTA or one cluster of 8 (the phases need a
// barrier, not a grid: the tables of 48 copies of 1500 tokens are 4,500 entries),
// then the copies by one CTA for each (copy, layer).  Bound by latency for few
// copies and by the copies' bytes for many: only the rows in use move, each as
// runs of 16 * head_dim bytes or more.
#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace specdec {

constexpr int kForkSmall = 2048;  // table entries and blocks of a call that one CTA works on
constexpr int kForkCtas = 8, kForkThreads = 512, kForkWarps = kForkThreads / 32;

struct ForkArgs {
    int32_t* tables;
    int32_t* nblk;
    int32_t* len;
    int32_t* ref;
    int num_blocks, max_reqs, max_bpr, block_size;
    const int32_t* src;
    const int32_t* dst;
    int n;
    int32_t* status;
    // workspace
    int32_t* head;   // [64]: c error seen by CTA c, 8 pairs to copy, 16 + c free blocks counted by CTA c
    int32_t* refw;   // [num_blocks] reference counts in the making
    int32_t* rank;   // [n] copies before this one that need a block
    int32_t* fresh;  // [n] blocks for them
    int32_t* pair;   // [n][3] block to read, block to write, rows
};

// The next free slots of a CTA-wide exclusive sum; every thread gets the total.
__device__ int fork_scan(int v, int* sh, int* total) {
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
    int before = 0, t = 0;
    for (int i = 0; i < kForkWarps; ++i) {
        if (i == w) before = t;
        t += sh[i];
    }
    *total = t;
    return before + x - v;
}

template <int CTAS>
__device__ __forceinline__ void fork_sync() {
    if constexpr (CTAS > 1) cluster_sync_all();
    else __syncthreads();
}

template <int CTAS>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(kForkThreads) kv_fork_kernel(ForkArgs a) {
    __shared__ int sh[kForkWarps], ranks[kForkThreads];
    const int cta = blockIdx.x, tid = threadIdx.x;
    const int gt = cta * kForkThreads + tid, stride = CTAS * kForkThreads;
    const int bs = a.block_size;
    // Every check of the arguments reads what the call does not change yet, so one
    // barrier stands between the checks and the first change; refw is a copy.
    // Ids in range, targets distinct and no sources, sources with a table that
    // holds their tokens.  A group of the cluster's warps to each copy (one copy
    // after the other in a CTA took most of 23 us for 48).
    const int warps = CTAS * kForkWarps, gw = gt >> 5, lane = tid & 31;
    const int group = max(1, warps / max(1, a.n)), groups = warps / group;
    const int mine = gw / group, part = gw % group * 32 + lane, step = group * 32;
    const int first = mine < groups ? mine : a.n;
    auto leave = [&](int code) {
        if (cta == 0 && tid == 0) *a.status = code;
    };
    // A call waits for its loads, one round behind the other, far longer than it
    // computes: what does not depend on one another is loaded together, and what a
    // group knows of its first copy (most often its only one) it keeps.
    struct Copy {
        int s, d, have, L, old;  // source, target, source's blocks and tokens, target's blocks
    };
    auto ids_ok = [&](int s, int d) { return s >= 0 && s < a.max_reqs && d >= 0 && d < a.max_reqs; };
    auto load = [&](int i) {
        Copy c = {a.src[i], a.dst[i], -1, 0, -1};
        if (ids_ok(c.s, c.d)) {
            c.have = a.nblk[c.s];
            c.L = a.len[c.s];
            c.old = a.nblk[c.d];
        }
        return c;
    };
    const int scan_s = tid < a.n ? a.src[tid] : -1, ref0 = gt < a.num_blocks ? a.ref[gt] : 0;
    Copy kept = {-1, -1, -1, 0, -1};
    if (first < a.n) kept = load(first);
    const int scan_L = scan_s >= 0 && scan_s < a.max_reqs ? a.len[scan_s] : 0;
    auto copy = [&](int i) { return i == first ? kept : load(i); };
    bool bad = false;
    for (int i = first; i < a.n; i += groups) {
        const Copy c = copy(i);
        if (!ids_ok(c.s, c.d)) {
            bad = true;
            continue;
        }
        const int use = c.L < 0 ? 0 : (int)(((long long)c.L + bs - 1) / bs);
        const bool fits = c.have >= 0 && c.have <= a.max_bpr && c.old <= a.max_bpr && c.L >= 0 && use <= c.have;
        bad |= !fits;
        for (int j = part; j < a.n; j += step) {
            const int e = a.dst[j];
            bad |= e == c.s || (e == c.d && j != i);
        }
        if (fits)
            for (int j = part; j < use; j += step) {
                const int p = a.tables[(size_t)c.s * a.max_bpr + j];
                bad |= p < 0 || p >= a.num_blocks;
            }
    }
    // the copies that need a block, in order (every CTA counts; CTA 0 writes the ranks behind the first 512)
    int need = 0;
    for (int i0 = 0; i0 < a.n; i0 += kForkThreads) {
        const int i = i0 + tid;
        const int s = i0 == 0 ? scan_s : (i < a.n ? a.src[i] : -1);
        const int t = s >= 0 && s < a.max_reqs && (i0 == 0 ? scan_L : a.len[s]) % bs != 0;
        int tot;
        const int before = fork_scan(t, sh, &tot), r = t ? need + before : -1;
        if (i0 == 0) ranks[tid] = r;
        else if (cta == 0 && i < a.n) a.rank[i] = r;
        need += tot;
    }
    bad = __syncthreads_or(bad);
    if (tid == 0) a.head[cta] = bad;
    if (gt == 0) a.head[kForkCtas] = 0;  // pairs to copy
    for (int i = gt; i < a.num_blocks; i += stride) a.refw[i] = i == gt ? ref0 : a.ref[i];
    fork_sync<CTAS>();
    int any = 0;
    for (int c = 0; c < CTAS; ++c) any |= __ldcg(&a.head[c]);
    if (any) return leave(SPECDEC_EINVAL);
    // the targets' old blocks are released
    for (int i = first; i < a.n; i += groups) {
        const Copy c = copy(i);
        for (int j = part; j < c.old; j += step) {
            const int p = a.tables[(size_t)c.d * a.max_bpr + j];
            if (p >= 0 && p < a.num_blocks) atomicSub(&a.refw[p], 1);
        }
    }
    fork_sync<CTAS>();
    // the lowest free blocks: each CTA takes a range, its threads neighbouring pieces of it
    const int per_cta = (a.num_blocks + CTAS - 1) / CTAS;
    const int b0 = min(a.num_blocks, cta * per_cta), b1 = min(a.num_blocks, b0 + per_cta);
    const int per = (b1 - b0 + kForkThreads - 1) / kForkThreads;
    const int lo = min(b1, b0 + tid * per), hi = min(b1, lo + per);
    int cnt = 0;
    for (int b = lo; b < hi; ++b) cnt += __ldcg(&a.refw[b]) == 0;
    int here;
    int before = fork_scan(cnt, sh, &here);
    if (tid == 0) a.head[16 + cta] = here;
    fork_sync<CTAS>();
    int total = 0;
    for (int c = 0; c < CTAS; ++c) {
        const int x = __ldcg(&a.head[16 + c]);
        if (c < cta) before += x;
        total += x;
    }
    if (total < need) return leave(SPECDEC_ENOMEM);
    if (before < need)
        for (int b = lo; b < hi && before < need; ++b)
            if (__ldcg(&a.refw[b]) == 0) a.fresh[before++] = b;
    fork_sync<CTAS>();
    // tables, lengths and counts of the copies
    for (int i = first; i < a.n; i += groups) {
        const Copy c = copy(i);
        const int s = c.s, d = c.d, L = c.L, whole = L / bs, r = i < kForkThreads ? ranks[i] : __ldcg(&a.rank[i]);
        const int page = r >= 0 ? __ldcg(&a.fresh[r]) : -1;
        int32_t* to = a.tables + (size_t)d * a.max_bpr;
        const int32_t* from = a.tables + (size_t)s * a.max_bpr;
        for (int j = part; j < a.max_bpr; j += step) {
            int p = -1;
            if (j < whole) {
                p = from[j];
                atomicAdd(&a.refw[p], 1);
            } else if (j == whole) {
                p = page;
            }
            to[j] = p;
        }
        if (part == 0) {
            a.len[d] = L;
            a.nblk[d] = whole + (r >= 0);
            if (r >= 0) {
                a.refw[page] = 1;
                a.pair[3 * r] = from[whole];
                a.pair[3 * r + 1] = page;
                a.pair[3 * r + 2] = L % bs;
            }
        }
    }
    fork_sync<CTAS>();
    for (int i = gt; i < a.num_blocks; i += stride) a.ref[i] = __ldcg(&a.refw[i]);
    if (gt == 0) {
        a.head[kForkCtas] = need;
        *a.status = SPECDEC_OK;
    }
}

// One CTA copies the rows in use of one block in one layer: for K and V and
// each head a run of rows * hd halves.
__global__ void __launch_bounds__(256) kv_fork_copy_kernel(const int32_t* head, const int32_t* pair, __half* kv,
                                                           size_t layer_stride, int Hkv, int hd) {
    pdl_wait();
    const int i = blockIdx.x;
    if (i >= head[kForkCtas]) return;
    const int rows = pair[3 * i + 2], run = rows * hd / 8, total = 2 * Hkv * run;  // 16-byte pieces
    const size_t block = (size_t)2 * Hkv * 16 * hd;
    const uint4* src = reinterpret_cast<const uint4*>(kv + layer_stride * blockIdx.y + block * pair[3 * i]);
    uint4* dst = reinterpret_cast<uint4*>(kv + layer_stride * blockIdx.y + block * pair[3 * i + 1]);
    const int plane = 2 * hd;  // 16 rows of hd halves in 16-byte pieces
    for (int x0 = threadIdx.x; x0 < total; x0 += 4 * 256) {
        uint4 v[4];
        int at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int x = x0 + 256 * u;
            at[u] = x < total ? x / run * plane + x % run : -1;
            if (at[u] >= 0) v[u] = src[at[u]];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (at[u] >= 0) dst[at[u]] = v[u];
    }
}

size_t kv_fork_workspace(int num_blocks, int n) { return sizeof(int32_t) * (64 + (size_t)num_blocks + 5 * (size_t)n); }

int kv_fork_launch(const KVState& st, const int32_t* src, const int32_t* dst, int n, __half* kv, int layers,
                   size_t layer_stride, int Hkv, int hd, int32_t* status, void* ws, cudaStream_t s) {
    ForkArgs a = {};
    a.tables = st.tables;
    a.nblk = st.nblk;
    a.len = st.len;
    a.ref = st.ref;
    a.num_blocks = st.num_blocks;
    a.max_reqs = st.max_reqs;
    a.max_bpr = st.max_bpr;
    a.block_size = st.block_size;
    a.src = src;
    a.dst = dst;
    a.n = n;
    a.status = status;
    a.head = static_cast<int32_t*>(ws);
    a.refw = a.head + 64;
    a.rank = a.refw + st.num_blocks;
    a.fresh = a.rank + n;
    a.pair = a.fresh + n;
    // Few entries: one CTA, whose barriers cost little (4 copies of 205 tokens in a pool of 256 blocks: 8.0 us a call,
    // a cluster 10.6; 8 of 1500 in 2048: 11.7 and 11.9; 16 of 1500 in 4096: 15.4 and 12.2).
    if ((long long)n * st.max_bpr + st.num_blocks <= kForkSmall) kv_fork_kernel<1><<<1, kForkThreads, 0, s>>>(a);
    else kv_fork_kernel<kForkCtas><<<kForkCtas, kForkThreads, 0, s>>>(a);
    SD_LAUNCH_CHECK("kv_fork_kernel");
    if (kv && layers > 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)n, (unsigned)layers);
        cfg.blockDim = dim3(256);
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        SD_CUDA(cudaLaunchKernelEx(&cfg, kv_fork_copy_kernel, (const int32_t*)a.head, (const int32_t*)a.pair, kv,
                                   layer_stride, Hkv, hd));
    }
    return SPECDEC_OK;
}

int kv_fork_check_pool(const char* who, const void* kv, int layers, size_t layer_stride, int num_blocks, int Hkv, int hd) {
    const std::string w(who);
    SD_CHECK(layers >= 0 && layers <= 65535, SPECDEC_EINVAL, w + ": 0 to 65535 layers");
    if (layers == 0) return SPECDEC_OK;
    SD_CHECK(kv && (reinterpret_cast<uintptr_t>(kv) & 15) == 0, SPECDEC_EINVAL,
             w + ": the pool must be given and 16-byte aligned");
    SD_CHECK(Hkv > 0 && Hkv <= 1024 && hd > 0 && hd <= 1024 && hd % 8 == 0, SPECDEC_EINVAL, w + ": bad head shape");
    SD_CHECK(layer_stride % 8 == 0 && layer_stride >= (size_t)num_blocks * 2 * Hkv * 16 * hd, SPECDEC_EINVAL,
             w + ": layer stride below the pool of a layer, or not a multiple of 8");
    return SPECDEC_OK;
}

}  // namespace specdec

using namespace specdec;

extern "C" size_t specdec_kv_fork_pages_workspace_bytes(int num_blocks, int max_reqs, int n) {
    if (num_blocks <= 0 || max_reqs <= 0 || n < 0) return 0;
    return kv_fork_workspace(num_blocks, n);
}

extern "C" int specdec_kv_fork_pages(int32_t* tables, int32_t* n_blocks, int32_t* lens, int32_t* refcounts,
                                     int num_blocks, int max_reqs, int max_blocks, const int32_t* src,
                                     const int32_t* dst, int n, uint16_t* kv, int layers, size_t layer_stride,
                                     int n_kv_heads, int head_dim, int32_t* status, void* workspace,
                                     size_t workspace_bytes, void* stream) {
    SD_CHECK(tables && n_blocks && lens && refcounts && status && (n == 0 || (src && dst)), SPECDEC_EINVAL,
             "kv_fork_pages: null argument");
    SD_CHECK(num_blocks > 0 && max_reqs > 0 && max_blocks > 0 && max_blocks <= (1 << 26) && n >= 0 && n <= max_reqs,
             SPECDEC_EINVAL, "kv_fork_pages: bad sizes (at most max_reqs copies)");
    int rc = kv_fork_check_pool("kv_fork_pages", kv, layers, layer_stride, num_blocks, n_kv_heads, head_dim);
    if (rc) return rc;
    SD_CHECK(workspace && workspace_bytes >= kv_fork_workspace(num_blocks, n) &&
                 (reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
             SPECDEC_EINVAL, "kv_fork_pages: workspace too small or not 4-byte aligned");
    cudaStream_t s = as_stream(stream);
    const struct {
        const void* p;
        const char* what;
    } given[] = {{tables, "kv_fork_pages: tables"},
                 {n_blocks, "kv_fork_pages: n_blocks"},
                 {lens, "kv_fork_pages: lens"},
                 {refcounts, "kv_fork_pages: refcounts"},
                 {status, "kv_fork_pages: status"},
                 {workspace, "kv_fork_pages: the workspace"},
                 {n ? src : tables, "kv_fork_pages: src"},
                 {n ? dst : tables, "kv_fork_pages: dst"},
                 {layers ? (const void*)kv : tables, "kv_fork_pages: the pool"}};
    for (const auto& g : given)
        if ((rc = check_on_device(g.p, g.what))) return rc;
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
    return kv_fork_launch(st, src, dst, n, reinterpret_cast<__half*>(kv), layers, layer_stride, n_kv_heads, head_dim,
                          status, workspace, s);
}
