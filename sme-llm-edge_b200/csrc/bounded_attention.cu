// bounded_attention.cu -- causal attention of packed rows over the paged pool
// that sees a window and the first tokens (specdec_attention_window), or that
// adds up what weight each slot received (specdec_attention_accumulate).
//
// With x = q.k / sqrt(hd) over the slots that a row sees, m = max x:
//   l = sum e^(x - m),  out = sum e^(x - m) v / l,  weights[slot] += e^(x - m) / l.
#include <algorithm>

#include "common.cuh"
#include "internal.h"

namespace specdec {

constexpr int kBoundMaxSeqs = 1024;

struct BoundArgs {
    const __half* q;
    int ldq;
    const __half* kv;
    int num_blocks, Hkv, Hq, G;
    const int32_t* tables;
    int max_blocks;
    const int32_t* ctx_len;
    const int32_t* row_off;
    int B, T, window, sinks;
    float* weights;
    int ldw;
    __half* out;
    int ldo;
    float2* ml;  // [T][Hq] a row's largest x and sum (accumulate)
    float scale;
};

struct BoundRow {
    int b, slot, last;  // sequence (-1: none), the row's slot, last slot that exists for it
};
__device__ __forceinline__ BoundRow bound_row(const BoundArgs& a, int r) {
    int lo = 0, hi = a.B;  // first sequence whose end is past the row
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.row_off[mid + 1] > r) hi = mid;
        else lo = mid + 1;
    }
    if (lo >= a.B || a.row_off[lo] > r) return {-1, 0, 0};
    const int slot = max(0, min(a.ctx_len[lo], 1 << 30)) + r - max(0, a.row_off[lo]);
    return {lo, slot, min(slot, a.max_blocks * 16 - 1)};
}
__device__ __forceinline__ const __half* bound_slot(const BoundArgs& a, int b, int slot, int plane, int kvh, int hd) {
    const int p = a.tables[(size_t)b * a.max_blocks + (slot >> 4)];
    const int page = p < 0 || p >= a.num_blocks ? 0 : p;
    return a.kv + ((((size_t)page * 2 + plane) * a.Hkv + kvh) * 16 + (slot & 15)) * hd;
}

// A warp for each row and query head.
template <int HD>
__global__ void __launch_bounds__(256) bound_rows_kernel(const __grid_constant__ BoundArgs a) {
    constexpr int W = HD / 32;
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int r = (int)(w / a.Hq), head = (int)(w % a.Hq);
    if (r >= a.T) return;
    const BoundRow row = bound_row(a, r);
    if (row.b < 0) return;
    const int kvh = head / a.G;
    float q[W], o[W], bad[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
        q[e] = __half2float(a.q[(size_t)r * a.ldq + (size_t)head * HD + lane * W + e]) * a.scale;
        o[e] = bad[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int from = max(0, row.slot - a.window + 1), first = min(a.sinks, from);
    for (int j = first > 0 ? 0 : from; j <= row.last; j = j + 1 == first ? from : j + 1) {
        const __half* k = bound_slot(a, row.b, j, 0, kvh, HD) + lane * W;
        const __half* v = bound_slot(a, row.b, j, 1, kvh, HD) + lane * W;
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < W; ++e) x = fmaf(q[e], __half2float(k[e]), x);
        x = warp_sum(x);
        const float top = x > m || x != x ? x : m;
        const float sub = top == -INFINITY ? 0.f : top;
        const float f = expf(m - sub), p = expf(x - sub);
        m = top;
        l = l * f + p;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const float y = __half2float(v[e]);
            if (isfinite(y)) o[e] = o[e] * f + p * y;
            else {
                o[e] *= f;
                bad[e] += y;  // reaches the row whatever its weight
            }
        }
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        float y = o[e] * inv;
        if (fabsf(y) > 65504.f) y = copysignf(65504.f, y);
        a.out[(size_t)r * a.ldo + (size_t)head * HD + lane * W + e] = __float2half_rn(y == y && bad[e] != 0.f ? bad[e] : y);
    }
    if (a.ml && lane == 0) a.ml[(size_t)r * a.Hq + head] = make_float2(m, l);
}

// A warp for each slot of a sequence's KV head.
template <int HD>
__global__ void __launch_bounds__(256) bound_weights_kernel(const __grid_constant__ BoundArgs a) {
    constexpr int W = HD / 32;
    const int lane = threadIdx.x & 31, b = blockIdx.z, kvh = blockIdx.y;
    const int j = blockIdx.x * 8 + (threadIdx.x >> 5);
    const int r0 = max(0, min(a.row_off[b], a.T)), r1 = max(r0, min(a.row_off[b + 1], a.T));
    const int ctx = max(0, min(a.ctx_len[b], 1 << 30));
    if (j >= a.max_blocks * 16 || j >= ctx + (r1 - r0)) return;
    const __half* k = bound_slot(a, b, j, 0, kvh, HD) + lane * W;
    float kf[W], sum = 0.f;
#pragma unroll
    for (int e = 0; e < W; ++e) kf[e] = __half2float(k[e]);
    for (int r = max(r0, r0 + j - ctx); r < r1; ++r)
        for (int g = 0; g < a.G; ++g) {
            const int head = kvh * a.G + g;
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < W; ++e)
                x = fmaf(__half2float(a.q[(size_t)r * a.ldq + (size_t)head * HD + lane * W + e]) * a.scale, kf[e], x);
            x = warp_sum(x);
            const float2 ml = a.ml[(size_t)r * a.Hq + head];
            sum += ml.y > 0.f || ml.y != ml.y ? expf(x - ml.x) / ml.y : 0.f;
        }
    if (lane == 0) a.weights[((size_t)b * a.Hkv + kvh) * a.ldw + j] += sum;
}

static int check_bound(const char* who, const void* q, int ldq, const void* kv, const void* out, int ldo, int num_blocks,
                       int Hkv, int HD, const void* tables, int max_blocks, const void* ctx_len, const void* row_off,
                       int B, int T, int Hq) {
    const std::string w(who);
    SD_CHECK(B == 0 || T == 0 || (q && kv && tables && ctx_len && row_off && out), SPECDEC_EINVAL, w + ": null argument");
    SD_CHECK(HD == 64 || HD == 128, SPECDEC_EINVAL, w + ": head_dim must be 64 or 128");
    SD_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 128 && Hq <= 1024, SPECDEC_EINVAL,
             w + ": bad head counts (at most 1024 query heads, 128 for each KV head)");
    SD_CHECK(num_blocks > 0 && max_blocks > 0 && max_blocks <= (1 << 26), SPECDEC_EINVAL, w + ": empty block pool or table");
    SD_CHECK(B >= 0 && B <= kBoundMaxSeqs, SPECDEC_EINVAL, w + ": 0 to 1024 sequences");
    SD_CHECK(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
             SPECDEC_EINVAL, w + ": q, KV pool and out must be 16-byte aligned");
    SD_CHECK(ldq >= Hq * HD && ldq % 8 == 0 && ldo >= Hq * HD && ldo % 8 == 0, SPECDEC_EINVAL,
             w + ": row strides hold all heads and are multiples of 8");
    return SPECDEC_OK;
}
static int check_bound_memory(const char* who, const void* q, const void* kv, const void* out, const void* tables,
                              const void* ctx_len, const void* row_off, const void* ws) {
    const std::string w(who);
    const struct {
        const void* p;
        const char* what;
    } given[] = {{q, ": q"}, {kv, ": the KV pool"}, {out, ": out"}, {tables, ": tables"}, {ctx_len, ": ctx_len"},
                 {row_off, ": row_off"}, {ws, ": the workspace"}};
    int rc;
    for (const auto& g : given)
        if ((rc = check_on_device(g.p, (w + g.what).c_str()))) return rc;
    return SPECDEC_OK;
}

}  // namespace specdec

using namespace specdec;

static int launch_bound(const BoundArgs& a, int HD, cudaStream_t s) {
    const unsigned grid = (unsigned)(((long long)a.T * a.Hq + 7) / 8);
    if (HD == 128) bound_rows_kernel<128><<<grid, 256, 0, s>>>(a);
    else bound_rows_kernel<64><<<grid, 256, 0, s>>>(a);
    SD_LAUNCH_CHECK("bound_rows_kernel");
    if (a.weights) {
        const dim3 g2((unsigned)(2 * (size_t)a.max_blocks), (unsigned)a.Hkv, (unsigned)a.B);
        if (HD == 128) bound_weights_kernel<128><<<g2, 256, 0, s>>>(a);
        else bound_weights_kernel<64><<<g2, 256, 0, s>>>(a);
        SD_LAUNCH_CHECK("bound_weights_kernel");
    }
    return SPECDEC_OK;
}

extern "C" size_t specdec_attention_window_workspace_bytes(int B, int T, int n_q_heads, int n_kv_heads, int head_dim,
                                                           int max_blocks) {
    if (B <= 0 || T <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || max_blocks <= 0) return 0;
    return 256;
}

extern "C" int specdec_attention_window(const uint16_t* q, int ldq, const uint16_t* kv_layer, int num_blocks,
                                        int n_kv_heads, int head_dim, const int32_t* tables, int max_blocks,
                                        const int32_t* ctx_len, const int32_t* row_off, int B, int T, int n_q_heads,
                                        int window, int sinks, uint16_t* out, int ldo, void* workspace,
                                        size_t workspace_bytes, void* stream) {
    const char* who = "attention_window";
    int rc = check_bound(who, q, ldq, kv_layer, out, ldo, num_blocks, n_kv_heads, head_dim, tables, max_blocks, ctx_len,
                         row_off, B, T, n_q_heads);
    if (rc) return rc;
    SD_CHECK(T >= 0 && T <= (1 << 24), SPECDEC_EINVAL, "attention_window: 0 to 2^24 rows");
    SD_CHECK(window >= 1 && sinks >= 0, SPECDEC_EINVAL, "attention_window: a window of at least one slot, sinks not negative");
    if (B == 0 || T == 0) return SPECDEC_OK;
    SD_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 31) == 0 &&
                 workspace_bytes >= specdec_attention_window_workspace_bytes(B, T, n_q_heads, n_kv_heads, head_dim, max_blocks),
             SPECDEC_EINVAL, "attention_window: workspace too small or not 32-byte aligned");
    if ((rc = check_bound_memory(who, q, kv_layer, out, tables, ctx_len, row_off, workspace))) return rc;
    BoundArgs a = {};
    a.q = reinterpret_cast<const __half*>(q);
    a.ldq = ldq;
    a.kv = reinterpret_cast<const __half*>(kv_layer);
    a.num_blocks = num_blocks;
    a.Hkv = n_kv_heads;
    a.Hq = n_q_heads;
    a.G = n_q_heads / n_kv_heads;
    a.tables = tables;
    a.max_blocks = max_blocks;
    a.ctx_len = ctx_len;
    a.row_off = row_off;
    a.B = B;
    a.T = T;
    a.window = window;
    a.sinks = sinks;
    a.out = reinterpret_cast<__half*>(out);
    a.ldo = ldo;
    a.scale = (float)(1.0 / sqrt((double)head_dim));
    return launch_bound(a, head_dim, as_stream(stream));
}

extern "C" size_t specdec_attention_accumulate_workspace_bytes(int B, int T, int n_q_heads, int n_kv_heads,
                                                               int head_dim, int max_blocks) {
    if (B <= 0 || T <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || max_blocks <= 0) return 0;
    return (size_t)T * n_q_heads * sizeof(float2);
}

extern "C" int specdec_attention_accumulate(const uint16_t* q, int ldq, const uint16_t* kv_layer, int num_blocks,
                                            int n_kv_heads, int head_dim, const int32_t* tables, int max_blocks,
                                            const int32_t* ctx_len, const int32_t* row_off, int B, int T, int n_q_heads,
                                            float* weights, int ldw, uint16_t* out, int ldo, void* workspace,
                                            size_t workspace_bytes, void* stream) {
    const char* who = "attention_accumulate";
    int rc = check_bound(who, q, ldq, kv_layer, out, ldo, num_blocks, n_kv_heads, head_dim, tables, max_blocks, ctx_len,
                         row_off, B, T, n_q_heads);
    if (rc) return rc;
    SD_CHECK(T >= 0 && T <= 65536 && n_q_heads / n_kv_heads <= 32, SPECDEC_EINVAL,
             "attention_accumulate: 0 to 65536 rows, at most 32 query heads for each KV head");
    SD_CHECK(B == 0 || T == 0 || weights, SPECDEC_EINVAL, "attention_accumulate: null argument");
    SD_CHECK(max_blocks <= (1 << 26) && ldw >= 16LL * max_blocks && ldw % 4 == 0 &&
                 (reinterpret_cast<uintptr_t>(weights) & 15) == 0,
             SPECDEC_EINVAL, "attention_accumulate: weights 16-byte aligned, ldw a multiple of 4 that holds max_blocks * 16 slots");
    if (B == 0 || T == 0) return SPECDEC_OK;
    SD_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 31) == 0 &&
                 workspace_bytes >=
                     specdec_attention_accumulate_workspace_bytes(B, T, n_q_heads, n_kv_heads, head_dim, max_blocks),
             SPECDEC_EINVAL, "attention_accumulate: workspace too small or not 32-byte aligned");
    if ((rc = check_bound_memory(who, q, kv_layer, out, tables, ctx_len, row_off, workspace))) return rc;
    if ((rc = check_on_device(weights, "attention_accumulate: weights"))) return rc;
    BoundArgs a = {};
    a.q = reinterpret_cast<const __half*>(q);
    a.ldq = ldq;
    a.kv = reinterpret_cast<const __half*>(kv_layer);
    a.num_blocks = num_blocks;
    a.Hkv = n_kv_heads;
    a.Hq = n_q_heads;
    a.G = n_q_heads / n_kv_heads;
    a.tables = tables;
    a.max_blocks = max_blocks;
    a.ctx_len = ctx_len;
    a.row_off = row_off;
    a.B = B;
    a.T = T;
    a.window = 1 << 30;
    a.weights = weights;
    a.ldw = ldw;
    a.out = reinterpret_cast<__half*>(out);
    a.ldo = ldo;
    a.ml = static_cast<float2*>(workspace);
    a.scale = (float)(1.0 / sqrt((double)head_dim));
    return launch_bound(a, head_dim, as_stream(stream));
}
