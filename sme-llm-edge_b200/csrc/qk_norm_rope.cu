// qk_norm_rope.cu -- queries and keys of packed rows normed per head and
// rotated, keys and values into their pages: what stands between the fused QKV
// projection and the attention calls (specdec_qk_norm_rope_kv).
//
// For each head x of q and k, in 32 bits and rounded to fp16 once:
//   y = x / sqrt(mean(x^2) + eps) * w
//   (y_d, y_{d + r/2}) -> (y_d c_d - y_{d + r/2} s_d, y_{d + r/2} c_d + y_d s_d), d < r/2
// A row's values are read once and written once; HBM bounds many rows, the chain
// bounds -> sequence -> page number -> store a few.
//
// head_dim / 8 lanes hold a head, and 2 (head_dim 128) or 4 heads are in a warp.  A
// lane holds four values and the other halves of their pairs (8 of the rest where
// a head turns in part): only the sum of squares crosses lanes.
#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace specdec {

constexpr int kNormMaxSeqs = 1024;
constexpr int kNormWarps = 4;

struct NormArgs {
    const void* qkv;
    int ld;
    const float* qw;
    const float* kw;
    float eps;
    const float* cos_t;
    const float* sin_t;
    int max_pos, half;  // half: pairs of a head that rotate
    const int32_t* pos;
    __half* kv;
    int num_blocks, Hkv, Hq;
    const int32_t* tables;
    int max_blocks;
    const int32_t* ctx_len;
    const int32_t* row_off;
    int B, T;
    __half* q_out;
    int ldq;
    int parts;  // warps of a row
};

// The sequence of packed row r, -1 where it has none: bounds in two rounds of 32.
__device__ __forceinline__ int norm_sequence(const NormArgs& a, int r) {
    const int lane = threadIdx.x & 31, step = (a.B + 31) / 32;
    auto below = [&](int b) { return b < a.B && a.row_off[b + 1] <= r; };  // sequence b ends before the row
    const int c = __popc(__ballot_sync(0xffffffffu, (lane + 1) * step <= a.B && below((lane + 1) * step - 1)));
    const int b = c * step + __popc(__ballot_sync(0xffffffffu, lane < step && below(c * step + lane)));
    return b < a.B && a.row_off[b] <= r ? b : -1;
}

// Four values at lo and four at hi, as they lie in memory.
template <typename In>
struct NormRaw;
template <>
struct NormRaw<float> {
    float4 u, v;
    __device__ __forceinline__ void load(const float* src, int lo, int hi) {
        u = __ldcs(reinterpret_cast<const float4*>(src + lo));
        v = __ldcs(reinterpret_cast<const float4*>(src + hi));
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
        x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    }
};
template <>
struct NormRaw<__half> {
    uint2 u, v;
    __device__ __forceinline__ void load(const __half* src, int lo, int hi) {
        u = __ldcs(reinterpret_cast<const uint2*>(src + lo));
        v = __ldcs(reinterpret_cast<const uint2*>(src + hi));
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t h[4] = {u.x, u.y, v.x, v.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
            x[2 * e] = f.x, x[2 * e + 1] = f.y;
        }
    }
};
__device__ __forceinline__ void norm_load4(const float* src, float* x) {
    const float4 u = *reinterpret_cast<const float4*>(src);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
}

// U: head groups that a warp has in flight at a time (their loads go out together, before the row's place is looked up).
template <int HD, typename In, int U, int MINB>
__global__ void __launch_bounds__(32 * kNormWarps, MINB) qk_norm_rope_kernel(const __grid_constant__ NormArgs a) {
    constexpr int LPH = HD / 8, HS = 32 / LPH;  // lanes of a head, heads of a group
    const int lane = threadIdx.x & 31, sub = lane / LPH, l = lane % LPH;
    // this lane's values: d .. d + 3 and their pairs, or 8 of those that do not turn
    const int pairs = a.half / 4;  // lanes that turn
    const bool turns = l < pairs;
    const int lo = turns ? 4 * l : 2 * a.half + 8 * (l - pairs), hi = turns ? lo + a.half : lo + 4;
    const long long w = (long long)blockIdx.x * kNormWarps + (threadIdx.x >> 5);
    const int r = a.parts == 1 ? (int)w : (int)(w / a.parts), part = (int)(w - (long long)r * a.parts);
    if (r >= a.T) return;
    const int heads = a.Hq + 2 * a.Hkv;
    const In* row = static_cast<const In*>(a.qkv) + (size_t)r * a.ld;
    NormRaw<In> raw[U];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int u = 0; u < U; ++u)  // (behind the last head: the last one again)
            raw[u].load(row + (size_t)min(h0 + u * a.parts * HS + sub, heads - 1) * HD, lo, hi);
    };
    fetch(part * HS);
    const int b = norm_sequence(a, r);
    if (b < 0) return;
    const int slot = max(0, min(a.ctx_len[b], 1 << 30)) + (r - max(0, a.row_off[b]));
    const int page = slot < a.max_blocks * 16 ? a.tables[(size_t)b * a.max_blocks + (slot >> 4)] : -1;
    const bool paged = page >= 0 && page < a.num_blocks;
    float c[4], s[4];
    if (turns) {
        const int p = max(0, min(a.pos ? a.pos[r] : slot, a.max_pos - 1));
        norm_load4(a.cos_t + (size_t)p * a.half + lo, c);
        norm_load4(a.sin_t + (size_t)p * a.half + lo, s);
    }
    __half* kv = a.kv + ((size_t)max(page, 0) * 2 * a.Hkv * 16 + (slot & 15)) * HD;
    for (int h0 = part * HS; h0 < heads; h0 += U * a.parts * HS) {
        if (h0 > part * HS) fetch(h0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * a.parts * HS + sub;
            const bool real = h < heads, is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hkv;
            float x[8], sum = 0.f;
            raw[u].get(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
            for (int o = LPH / 2; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float* norm = is_q ? a.qw : is_k ? a.kw : nullptr;
            if (norm) {
                float g[8];
                norm_load4(norm + lo, g);
                norm_load4(norm + hi, g + 4);
                const float inv = rsqrtf(sum * (1.0f / HD) + a.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * g[e];
            }
            if (turns && (is_q || is_k)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y = x[e], z = x[e + 4];
                    x[e] = y * c[e] - z * s[e];
                    x[e + 4] = z * c[e] + y * s[e];
                }
            }
            uint2 out[2];
            __half2* o2 = reinterpret_cast<__half2*>(out);
#pragma unroll
            for (int e = 0; e < 4; ++e) o2[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
            // a query head; or in [K|V][kv head][16][HD], K's heads and then V's
            __half* dst = is_q ? a.q_out + (size_t)r * a.ldq + (size_t)h * HD : kv + (size_t)(h - a.Hq) * 16 * HD;
            if (real && (is_q || paged)) {
                *reinterpret_cast<uint2*>(dst + lo) = out[0];
                *reinterpret_cast<uint2*>(dst + hi) = out[1];
            }
        }
    }
}

}  // namespace specdec

using namespace specdec;

extern "C" int specdec_qk_norm_rope_kv(const void* qkv, int qkv_f16, int ldqkv, const float* q_norm,
                                       const float* k_norm, float eps, const float* cos_t, const float* sin_t,
                                       int max_pos, int rot_dim, const int32_t* pos, uint16_t* kv_layer, int num_blocks,
                                       int n_kv_heads, int head_dim, const int32_t* tables, int max_blocks,
                                       const int32_t* ctx_len, const int32_t* row_off, int B, int T, int n_q_heads,
                                       uint16_t* q_out, int ldq, void* stream) {
    const char* who = "qk_norm_rope_kv";
    const std::string w(who);
    const bool empty = B == 0 || T == 0;  // an empty call's tensors may have no memory
    SD_CHECK(empty || (qkv && kv_layer && tables && ctx_len && row_off && q_out && (rot_dim == 0 || (cos_t && sin_t))),
             SPECDEC_EINVAL, w + ": null argument");
    SD_CHECK(qkv_f16 == 0 || qkv_f16 == 1, SPECDEC_EINVAL, w + ": qkv_f16 is 0 (fp32) or 1 (fp16)");
    SD_CHECK(head_dim == 64 || head_dim == 128, SPECDEC_EINVAL, w + ": head_dim must be 64 or 128");
    SD_CHECK(n_kv_heads > 0 && n_q_heads > 0 && n_q_heads % n_kv_heads == 0 && n_q_heads <= 1024, SPECDEC_EINVAL,
             w + ": bad head counts (at most 1024 query heads)");
    SD_CHECK(num_blocks > 0 && max_blocks > 0 && max_blocks <= (1 << 26), SPECDEC_EINVAL, w + ": empty block pool or table");
    SD_CHECK(B >= 0 && B <= kNormMaxSeqs && T >= 0 && T <= (1 << 24), SPECDEC_EINVAL,
             w + ": 0 to 1024 sequences and 0 to 2^24 rows");
    SD_CHECK(rot_dim >= 0 && rot_dim <= head_dim && rot_dim % 16 == 0 && (rot_dim == 0 || max_pos > 0), SPECDEC_EINVAL,
             w + ": rot_dim is a multiple of 16 up to head_dim, with a table of at least one position");
    SD_CHECK(eps >= 0.f && eps < INFINITY, SPECDEC_EINVAL, w + ": eps must be finite and not negative");
    const int per16 = qkv_f16 ? 8 : 4;
    SD_CHECK(ldqkv >= (n_q_heads + 2 * n_kv_heads) * head_dim && ldqkv % per16 == 0 && ldq >= n_q_heads * head_dim &&
                 ldq % 8 == 0,
             SPECDEC_EINVAL, w + ": row strides hold all heads and are multiples of 16 bytes");
    SD_CHECK(((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(kv_layer) |
               reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(q_norm) |
               reinterpret_cast<uintptr_t>(k_norm) | reinterpret_cast<uintptr_t>(cos_t) |
               reinterpret_cast<uintptr_t>(sin_t)) &
              15) == 0,
             SPECDEC_EINVAL, w + ": qkv, norms, cos / sin tables, KV pool and q_out must be 16-byte aligned");
    if (empty) return SPECDEC_OK;
    const struct {
        const void* p;
        const char* what;
    } given[] = {{qkv, "qk_norm_rope_kv: qkv"},
                 {kv_layer, "qk_norm_rope_kv: the KV pool"},
                 {q_out, "qk_norm_rope_kv: q_out"},
                 {tables, "qk_norm_rope_kv: tables"},
                 {ctx_len, "qk_norm_rope_kv: ctx_len"},
                 {row_off, "qk_norm_rope_kv: row_off"},
                 {q_norm ? q_norm : qkv, "qk_norm_rope_kv: q_norm"},
                 {k_norm ? k_norm : qkv, "qk_norm_rope_kv: k_norm"},
                 {rot_dim ? (const void*)cos_t : qkv, "qk_norm_rope_kv: cos_t"},
                 {rot_dim ? (const void*)sin_t : qkv, "qk_norm_rope_kv: sin_t"},
                 {pos && rot_dim ? (const void*)pos : qkv, "qk_norm_rope_kv: pos"}};
    int rc;
    for (const auto& g : given)
        if ((rc = check_on_device(g.p, g.what))) return rc;
    NormArgs a = {};
    a.qkv = qkv;
    a.ld = ldqkv;
    a.qw = q_norm;
    a.kw = k_norm;
    a.eps = eps;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.max_pos = max_pos;
    a.half = rot_dim / 2;
    a.pos = pos;
    a.kv = reinterpret_cast<__half*>(kv_layer);
    a.num_blocks = num_blocks;
    a.Hkv = n_kv_heads;
    a.Hq = n_q_heads;
    a.tables = tables;
    a.max_blocks = max_blocks;
    a.ctx_len = ctx_len;
    a.row_off = row_off;
    a.B = B;
    a.T = T;
    a.q_out = reinterpret_cast<__half*>(q_out);
    a.ldq = ldq;
    // Few rows: a warp for each head group, so that a row's chain of look-ups is all there is (160 rows of 32/8 heads of
    // 128, fp32: 3.7 us, a warp for the whole row 16.6).  Many: four groups in flight, four times, at 28 warps of an SM
    // (8 x 2501 such rows 117 us, 0.96 of the copy rate; 16 groups in flight or more warps of fewer registers 120 to 148).
    const int groups = ((n_q_heads + 2 * n_kv_heads) * head_dim + 255) / 256;
    const bool many = (long long)T * groups > 148LL * 64 * 4;
    // (eight times where that still fills the SMs: a row's look-ups are made by fewer warps)
    const int groups_of_warp = (long long)T * groups >= 148LL * 28 * 32 ? 32 : 16;
    a.parts = many ? (groups + groups_of_warp - 1) / groups_of_warp : groups;
    const long long warps = (long long)T * a.parts;
    const dim3 grid((unsigned)((warps + kNormWarps - 1) / kNormWarps)), block(32 * kNormWarps);
    cudaStream_t s = as_stream(stream);
#define NORM_LAUNCH(hd, type)                                          \
    do {                                                                         \
        if (many) qk_norm_rope_kernel<hd, type, 4, 7><<<grid, block, 0, s>>>(a); \
        else qk_norm_rope_kernel<hd, type, 1, 8><<<grid, block, 0, s>>>(a);      \
    } while (0)
    if (head_dim == 128) {
        if (qkv_f16) NORM_LAUNCH(128, __half);
        else NORM_LAUNCH(128, float);
    } else {
        if (qkv_f16) NORM_LAUNCH(64, __half);
        else NORM_LAUNCH(64, float);
    }
#undef NORM_LAUNCH
    SD_LAUNCH_CHECK("qk_norm_rope_kernel");
    return SPECDEC_OK;
}
