// prompt_attention.cu -- attention of packed prompt rows, and of verify rows
// whose sequences share a prefix, over paged fp16 KV (sm_100a).
//
// First form: one warp per (query row, head); the lanes split the head
// dimension and walk the visible keys with an online base-2 softmax.
#include "common.cuh"
#include "internal.h"

namespace specdec {

constexpr int kRowsMaxSeqs = 4096;

struct RowAttnArgs {
    const __half* q;
    int ldq;
    const __half* kv;
    int num_blocks, Hkv, Hq, G;
    const int32_t* tables;
    int max_blocks;
    const int32_t* ctx_len;
    const int32_t* row_off;  // null: R rows for every sequence
    const uint64_t* mask;    // null: causal
    int B, T, R;
    __half* out;
    int ldo;
    float scale_log2;
};

template <int HD>
__global__ void __launch_bounds__(128) row_attention_kernel(RowAttnArgs a) {
    constexpr int E = HD / 32;
    const long long id = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (id >= (long long)a.T * a.Hq) return;
    const int t = (int)(id / a.Hq), h = (int)(id % a.Hq), kvh = h / a.G;
    int b, i, n;
    if (a.row_off) {
        int lo = 0, hi = a.B;  // first sequence whose end is past t
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (a.row_off[mid + 1] > t) hi = mid;
            else lo = mid + 1;
        }
        b = lo;
        if (b >= a.B || t < a.row_off[b]) return;  // a row of no sequence
        i = t - a.row_off[b];
        n = a.row_off[b + 1] - a.row_off[b];
    } else {
        b = t / a.R;
        i = t % a.R;
        n = a.R;
    }
    const int ctx = max(0, a.ctx_len[b]);
    const long long cap = (long long)a.max_blocks * 16;
    const int L = (int)min((long long)ctx + n, cap);
    const uint64_t bits = a.mask ? a.mask[i] : 0;
    float q[E], o[E];
    const __half* qp = a.q + (size_t)t * a.ldq + (size_t)h * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = __half2float(qp[e]) * a.scale_log2;
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < L; ++j) {
        const bool seen = j < ctx || (a.mask ? (j - ctx < 64 && ((bits >> (j - ctx)) & 1)) : j - ctx <= i);
        if (!seen) continue;
        int blk = a.tables[(size_t)b * a.max_blocks + j / 16];
        if (blk < 0 || blk >= a.num_blocks) blk = 0;  // a malformed table reads block 0, never out of range
        const __half* kp = a.kv + ((((size_t)blk * 2) * a.Hkv + kvh) * 16 + j % 16) * HD + lane * E;
        const __half* vp = kp + (size_t)a.Hkv * 16 * HD;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += q[e] * __half2float(kp[e]);
        s = warp_sum(s);
        const float mn = fmaxf(m, s);
        const float w = exp2f(m - mn), p = exp2f(s - mn);
        l = l * w + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * w + p * __half2float(vp[e]);
        m = mn;
    }
    __half* op = a.out + (size_t)t * a.ldo + (size_t)h * HD + lane * E;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < E; ++e) op[e] = __float2half_rn(o[e] * inv);
}

static int launch_rows(const RowAttnArgs& a, int HD, cudaStream_t s) {
    const long long warps = (long long)a.T * a.Hq;
    const unsigned grid = (unsigned)((warps + 3) / 4);
    if (HD == 128) row_attention_kernel<128><<<grid, 128, 0, s>>>(a);
    else row_attention_kernel<64><<<grid, 128, 0, s>>>(a);
    SD_LAUNCH_CHECK("row_attention_kernel");
    return SPECDEC_OK;
}

// The checks that both entry points share.
static int check_rows(const char* who, const void* q, const void* kv, const void* out, int num_blocks, int Hkv, int HD,
                      int max_blocks, int B, int Hq) {
    const std::string w(who);
    SD_CHECK(HD == 64 || HD == 128, SPECDEC_EINVAL, w + ": head_dim must be 64 or 128");
    SD_CHECK(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 128 && Hq <= 1024, SPECDEC_EINVAL,
             w + ": bad head counts (at most 1024 query heads, 128 for each KV head)");
    SD_CHECK(num_blocks > 0 && max_blocks > 0 && max_blocks <= (1 << 26), SPECDEC_EINVAL,
             w + ": empty block pool or table");
    SD_CHECK(B >= 0 && B <= kRowsMaxSeqs, SPECDEC_EINVAL, w + ": 0 to 4096 sequences");
    SD_CHECK(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv) | reinterpret_cast<uintptr_t>(out)) &
              15) == 0,
             SPECDEC_EINVAL, w + ": q, KV pool and out must be 16-byte aligned");
    return SPECDEC_OK;
}

}  // namespace specdec

using namespace specdec;

extern "C" size_t specdec_attention_prompt_workspace_bytes(int B, int T, int n_q_heads, int n_kv_heads, int head_dim,
                                                           int max_blocks) {
    (void)B, (void)T, (void)n_q_heads, (void)n_kv_heads, (void)head_dim, (void)max_blocks;
    return 0;
}

extern "C" int specdec_attention_prompt(const uint16_t* q, int ldq, const uint16_t* kv_layer, int num_blocks,
                                        int n_kv_heads, int head_dim, const int32_t* tables, int max_blocks,
                                        const int32_t* ctx_len, const int32_t* row_off, int B, int T, int n_q_heads,
                                        uint16_t* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
    SD_CHECK(q && kv_layer && tables && ctx_len && row_off && out, SPECDEC_EINVAL, "attention_prompt: null argument");
    int rc = check_rows("attention_prompt", q, kv_layer, out, num_blocks, n_kv_heads, head_dim, max_blocks, B,
                        n_q_heads);
    if (rc) return rc;
    SD_CHECK(T >= 0 && T <= (1 << 24), SPECDEC_EINVAL, "attention_prompt: 0 to 2^24 rows");
    SD_CHECK(ldq >= n_q_heads * head_dim && ldq % 8 == 0 && ldo >= n_q_heads * head_dim && ldo % 8 == 0,
             SPECDEC_EINVAL, "attention_prompt: row strides hold all heads and are multiples of 8");
    (void)workspace;
    (void)workspace_bytes;
    if (B == 0 || T == 0) return SPECDEC_OK;
    RowAttnArgs a = {};
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
    a.out = reinterpret_cast<__half*>(out);
    a.ldo = ldo;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
    return launch_rows(a, head_dim, as_stream(stream));
}

extern "C" size_t specdec_attention_shared_prefix_workspace_bytes(int B, int R, int n_groups, int n_q_heads,
                                                                  int n_kv_heads, int head_dim, int max_blocks) {
    (void)B, (void)R, (void)n_groups, (void)n_q_heads, (void)n_kv_heads, (void)head_dim, (void)max_blocks;
    return 0;
}

extern "C" int specdec_attention_shared_prefix(const uint16_t* q, const uint16_t* kv_layer, int num_blocks,
                                               int n_kv_heads, int head_dim, const int32_t* tables, int max_blocks,
                                               const int32_t* ctx_len, const uint64_t* mask, const int32_t* group_off,
                                               const int32_t* shared_blocks, int n_groups, int B, int R, int n_q_heads,
                                               uint16_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    SD_CHECK(q && kv_layer && tables && ctx_len && mask && out && (n_groups == 0 || (group_off && shared_blocks)),
             SPECDEC_EINVAL, "attention_shared_prefix: null argument");
    int rc = check_rows("attention_shared_prefix", q, kv_layer, out, num_blocks, n_kv_heads, head_dim, max_blocks, B,
                        n_q_heads);
    if (rc) return rc;
    SD_CHECK(R >= 1 && R <= 64, SPECDEC_EINVAL, "attention_shared_prefix: 1 to 64 rows");
    SD_CHECK(n_groups >= 0 && n_groups <= B, SPECDEC_EINVAL, "attention_shared_prefix: 0 to B groups");
    (void)workspace;
    (void)workspace_bytes;
    if (B == 0) return SPECDEC_OK;
    RowAttnArgs a = {};
    a.q = reinterpret_cast<const __half*>(q);
    a.ldq = n_q_heads * head_dim;
    a.kv = reinterpret_cast<const __half*>(kv_layer);
    a.num_blocks = num_blocks;
    a.Hkv = n_kv_heads;
    a.Hq = n_q_heads;
    a.G = n_q_heads / n_kv_heads;
    a.tables = tables;
    a.max_blocks = max_blocks;
    a.ctx_len = ctx_len;
    a.mask = mask;
    a.B = B;
    a.R = R;
    a.T = B * R;
    a.out = reinterpret_cast<__half*>(out);
    a.ldo = a.ldq;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
    return launch_rows(a, head_dim, as_stream(stream));
}
