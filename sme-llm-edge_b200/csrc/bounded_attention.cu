// bounded_attention.cu -- causal attention of packed rows over the paged pool
// that sees a window and the first tokens (specdec_attention_window), or that
// adds up what weight each slot received (specdec_attention_accumulate).
//
// With x = q.k / sqrt(hd) over the slots that a row sees, m = max x:
//   l = sum e^(x - m),  out = sum e^(x - m) v / l,  weights[slot] += e^(x - m) / l.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <climits>

#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace specdec {

constexpr int kBoundMaxSeqs = 1024;
constexpr int kBoundSlots = (1 << 30) + (1 << 24);  // contexts and rows of a call at most

// ------------------------------------------------------------------ few rows
//
// A warp works for itself: it streams pages (16 tokens of one KV head, K and V
// together, one TMA request) through a ring of its own, so no barrier of the CTA
// stands between its loads and its arithmetic.  The call's pages, in the order
// (sequence, tile of rows, KV head, page), are cut into ranges, one for each warp,
// so ragged lengths balance by themselves.  SMs do not get equal shares of the
// memory's rate, so in long calls a fifth of the pages is left for a second wave
// of CTAs, which start where the first ones end early.  A tile is as many whole
// tokens as fit into 8 * NT rows (row = token * G + g).  For a page
//   S^T [16 keys][rows] = K Q^T,  P = 2^(S' - m),  O^T [hd][rows] += V^T P
// in mma.sync of 16 x 8 x 16: 16 keys of 8 rows are 4 FLOP for each byte of the
// cache, far from what the tensor cores of either kind can do, and the fragments
// stay in registers (128 rows of tensor memory for 4 to 32 real ones would not).
// The reference m of a row is 11 below its largest score at the time it was set and
// follows only when a score is more than 15 above it, so most pages move nothing
// and need no maximum across lanes.  P, rounded to fp16 for the product, is 2^15 at
// most, and weights keep their 11 bits down to 2^-25 of the largest (2^-29 where m
// is as high as it can be).  m, sums and O are fp32.
//
// Ranges that a warp shares with others leave unnormalised O with (m, l); they
// are joined in their order.
constexpr int kFewWarps = 4;       // of a CTA
constexpr int kFewMaxSms = 148;    // SMs for which there are ranges
constexpr int kFewMaxRows = 32;    // rows of a tile
// CTAs of an SM, and waves of them at most.  Registers allow three of one tile of 8 rows; pieces of more than 16 rows cost
// more than the wave gains.
__host__ __device__ constexpr int few_resident(int NT) { return NT == 1 ? 3 : 2; }
__host__ __device__ constexpr int few_waves(int NT) { return NT <= 2 ? 2 : 1; }
constexpr int kFewMinPages = 4;    // of a range
constexpr float kFewLift = 11.0f, kFewTop = 15.0f;
constexpr float kFewNone = -3e38f;  // m of a row that has seen no slot: below all scores
constexpr float kFewMax = 65504.0f;

struct FewArgs {
    const __half* q;
    int ldq;
    const __half* kv;
    int num_blocks, Hkv, Hq, G, tpt;  // tpt: tokens of a tile
    const int32_t* tables;
    int max_blocks, slots_max;
    const int32_t* ctx_len;
    const int32_t* row_off;
    int B, T, window, sinks;
    int least, most;  // sequences of up to `least` and of more than `most` rows are left out
    float* weights;
    int ldw;
    __half* out;
    int ldo;
    float scale_log2;
    int ctas, waves;    // CTAs of a wave (ranges)
    int wave_pages;     // pages of a warp from which there is a second wave
    int chunk, chunks;  // pages of a piece, pieces of a table at most (chunk 0: ranges)
    // workspace
    long long* pre;     // [B + 1] pages before sequence b
    int32_t* np;        // [B] pages of each (tile, head) of sequence b
    int32_t* runs;      // [B + 1] runs of 128 slots before sequence b (weights)
    // ranges; or [T][Hq][chunks] and [T][Hq][chunks][hd]
    float2* pml;        // [ranges][2][rows] m, l of a piece (l < 0: it met an infinity or NaN of V): of the range's
    float* po;          // [ranges][2][rows][hd]  first pages, or of later ones
    float2* ml;         // [T][Hq] m, 1 / l (weights)
    float* scores;      // [T][Hkv][slots_max][G] (weights)
    DeviceStatus* status;
};

struct FewSeq {
    int lo, n, ctx;
    int np;  // pages of each of its (tile, head)
};
__device__ __forceinline__ FewSeq few_seq(const FewArgs& a, int b) {
    FewSeq s;
    s.np = 0;
    s.lo = max(0, min(a.row_off[b], a.T));
    s.n = max(s.lo, min(a.row_off[b + 1], a.T)) - s.lo;
    if (s.n <= a.least || s.n > a.most) s.n = 0;
    s.ctx = max(0, min(a.ctx_len[b], 1 << 30));
    return s;
}
// Pages of a sequence's tile at most.
__device__ __forceinline__ int few_pages(const FewArgs& a, const FewSeq& s) {
    const int last = (min(s.ctx + s.n, a.slots_max) + 15) >> 4;
    const long long most = ((long long)min(a.sinks, a.slots_max) + 15) / 16 + ((long long)a.window + a.tpt - 2) / 16 + 2;
    return max(1, (int)min((long long)last, most));
}

// What tile `tile` of a sequence reads: pages 0 .. sinkp - 1 of its table, and
// from there on page v + gap.
struct FewTile {
    int tokens, row, p0;  // its tokens, first packed row, first row's slot
    int np, sinkp, gap;
};
__device__ __forceinline__ FewTile few_tile(const FewArgs& a, const FewSeq& s, int tile) {
    FewTile t;
    const int i0 = tile * a.tpt;
    t.tokens = min(a.tpt, s.n - i0);
    t.row = s.lo + i0;
    t.p0 = s.ctx + i0;
    const int end = min(t.p0 + t.tokens, a.slots_max);
    const int wp = max(0, t.p0 - a.window + 1) >> 4, last = (end + 15) >> 4;
    t.sinkp = (min(a.sinks, end) + 15) >> 4;
    t.gap = max(0, wp - t.sinkp);
    t.np = t.gap ? t.sinkp + max(0, last - wp) : last;
    return t;
}

// A warp's way through the pages of its range.
struct FewWalk {
    long long u, hi;    // next page of the call, end of the range
    int b, tile, kvh;
    int v, ve;          // pages of the tile still to come
    long long begun;    // the segment's first page of the call
    bool whole;         // the segment is all of the tile's pages
    FewTile t;
};
// To the next segment; false: the range is done.
__device__ __forceinline__ bool few_next(const FewArgs& a, const long long* pre, const FewSeq* seqs, FewWalk& w) {
    if (w.u >= w.hi) return false;
    int lo = 0, hi = a.B;  // last sequence with pre <= u
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= w.u) lo = mid;
        else hi = mid;
    }
    w.b = lo;
    const long long local = w.u - pre[lo];
    const FewSeq s = seqs[lo];
    const int n = s.np, pair = n < 1 ? 0 : local >> 31 ? (int)(local / n) : (int)local / n;
    w.v = (int)(local - (long long)pair * n);
    w.tile = pair / a.Hkv;
    w.kvh = pair - w.tile * a.Hkv;
    w.t = few_tile(a, s, w.tile);
    w.begun = w.u;
    const int take = (int)min((long long)(n - w.v), w.hi - w.u);
    w.u += take;
    w.ve = min(w.v + take, w.t.np);
    w.whole = w.v == 0 && w.ve == w.t.np;
    return true;
}

__device__ __forceinline__ void few_mma(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void few_ldm(uint32_t (&x)[4], uint32_t addr) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t few_turn(uint32_t x) {  // an 8 x 8 tile of halves, transposed
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float few_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float few_max(float x, float y) {  // NaN if one is
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}

// Sets the columns of a row in which it sees an infinity or a NaN of V: no weight
// is 0 by the definition, so they reach the row whatever the weight.  A warp for
// each row and head.
template <int HD>
__device__ __noinline__ void few_nonfinite(const FewArgs& a, int b, int p, int kvh, __half* dst) {
    constexpr int W = HD / 32;
    const int lane = threadIdx.x & 31, last = min(p, a.slots_max - 1);
    const int from = max(0, p - a.window + 1), first = min(a.sinks, from);
    float bad[W] = {};
    bool any = false;
    for (int j = first > 0 ? 0 : from; j <= last; j = j + 1 == first ? from : j + 1) {
        const int x = a.tables[(size_t)b * a.max_blocks + (j >> 4)], page = x < 0 || x >= a.num_blocks ? 0 : x;
        const __half* v = a.kv + ((((size_t)page * 2 + 1) * a.Hkv + kvh) * 16 + (j & 15)) * HD + lane * W;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const float y = __half2float(v[e]);
            if (!isfinite(y)) {
                bad[e] += y;
                any = true;
            }
        }
    }
    if (any)
#pragma unroll
        for (int e = 0; e < W; ++e)
            if (bad[e] != 0.f) dst[lane * W + e] = __float2half_rn(bad[e]);
}

template <int HD, int NT>
struct FewCfg {
    static constexpr int PAGE = 64 * HD;                 // bytes of a page's K and V of a head
    // Pages in flight of a warp: 64 single tokens on 4096 (8 heads of 128, tables of 2048 pages) take 181 us with two in
    // each warp of three CTAs of an SM, 184 with three in each of two CTAs, 186 with two.
    static constexpr int RING = (HD == 128 ? 1 : 2) * (NT == 1 ? 2 : 3);
    static constexpr size_t smem(int B) {
        return 1024 + (size_t)kFewWarps * RING * PAGE + kFewWarps * RING * 8 + (size_t)(B + 1) * 8 + (size_t)B * sizeof(FewSeq) + 16;
    }
};
static_assert(FewCfg<64, 2>::smem(kBoundMaxSeqs) <= 232448, "shared memory of a CTA");

// Pages before each sequence, by every CTA for itself from the lengths in device
// memory (so a captured call serves other lengths); CTA 0 leaves them for the
// kernels that follow.
__device__ __forceinline__ long long few_plan(const FewArgs& a, long long* pre, FewSeq* seqs, bool acc) {
    __shared__ long long wsum[kFewWarps];
    __shared__ int csum[kFewWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (a.B + 32 * kFewWarps - 1) / (32 * kFewWarps);
    const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
    long long x = 0;
    int c = 0;
    for (int b = b0; b < b1; ++b) {
        FewSeq s = few_seq(a, b);
        const int n = s.np = few_pages(a, s);
        seqs[b] = s;
        const long long all = (long long)((s.n + a.tpt - 1) / a.tpt) * a.Hkv * n;
        pre[b] = all;
        x += all;
        if (acc && s.n > 0) c += a.Hkv * ((n + 7) / 8);
    }
    const long long mine = x;
    const int cmine = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        const int d = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) {
            x += y;
            c += d;
        }
    }
    if (lane == 31) {
        wsum[warp] = x;
        csum[warp] = c;
    }
    __syncthreads();
    long long before = 0, total = 0;
    int cbefore = 0, ctotal = 0;
    for (int w = 0; w < kFewWarps; ++w) {
        if (w == warp) {
            before = total;
            cbefore = ctotal;
        }
        total += wsum[w];
        ctotal += csum[w];
    }
    before += x - mine;
    cbefore += c - cmine;
    for (int b = b0; b < b1; ++b) {
        const long long all = pre[b];
        pre[b] = before;
        if (blockIdx.x == 0) {
            a.pre[b] = before;
            a.np[b] = seqs[b].np;
            if (acc) {
                a.runs[b] = cbefore;
                if (all > 0) cbefore += a.Hkv * ((seqs[b].np + 7) / 8);
            }
        }
        before += all;
    }
    if (tid == 0) {
        pre[a.B] = total;
        if (blockIdx.x == 0) {
            a.pre[a.B] = total;
            if (acc) a.runs[a.B] = ctotal;
        }
    }
    __syncthreads();
    return total;
}
// How the pages are cut: the first wave's ranges of per0 pages, then those of the second wave of per1.
struct FewCut {
    long long total, from1;
    int warps, per0, per1;  // warps of a wave
    __device__ __forceinline__ FewCut(const FewArgs& a, long long n) : total(n), warps(a.ctas * kFewWarps) {
        const bool both = a.waves > 1 && n >= (long long)a.wave_pages * warps;
        const long long given = both ? n - n / 5 : n;
        per0 = (int)max((long long)kFewMinPages, (given + warps - 1) / warps);
        from1 = min(n, (long long)warps * per0);
        per1 = (int)max((long long)kFewMinPages, (n - from1 + warps - 1) / warps);
    }
    __device__ __forceinline__ long long begin(int r) const {
        return r < warps ? (long long)r * per0 : from1 + (long long)(r - warps) * per1;
    }
    __device__ __forceinline__ long long end(int r) const {
        return r < warps ? min(begin(r) + per0, from1) : min(begin(r) + per1, total);
    }
    __device__ __forceinline__ int of(long long u) const {
        return u < from1 ? (int)(u / per0) : warps + (int)((u - from1) / per1);
    }
};

// What a warp holds of a tile: its queries as MMA fragments (lane 4 g + t4: row g), each row's m and partial sums, O.
template <int HD, int NT, bool ACC>
struct FewWork {
    static constexpr int KS = HD / 16, NH = HD / 64;
    uint32_t qf[NT][KS][2];
    int slot_of[NT][2];  // slots of this lane's rows 2 t4, 2 t4 + 1 (of those behind the tile: the last one's)
    float m[NT][2], l[NT][2], o[KS][NT][4];
    float* score[NT];  // of this lane's rows at its slot of a page
    FewTile t;
    int kvh, rows, p1;
    bool bad;  // an infinity or a NaN of V was left out

    __device__ __forceinline__ float* score_at(const FewArgs& a, int row) const {
        const int tok = row / a.G;
        return a.scores + ((size_t)(t.row + tok) * a.Hkv + kvh) * a.slots_max * a.G + (row - tok * a.G);
    }
    __device__ __forceinline__ void begin(const FewArgs& a, const FewTile& tile, int head) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
        t = tile;
        kvh = head;
        rows = t.tokens * a.G;
        p1 = t.p0 + t.tokens - 1;
        bad = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = 8 * n + g;
            const bool real = row < rows;
            const int tok = real ? row / a.G : 0;
            const __half* src = a.q + (size_t)(t.row + tok) * a.ldq + (size_t)(kvh * a.G + (real ? row - tok * a.G : 0)) * HD + 2 * t4;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                qf[n][k][0] = real ? *reinterpret_cast<const uint32_t*>(src + 16 * k) : 0u;
                qf[n][k][1] = real ? *reinterpret_cast<const uint32_t*>(src + 16 * k + 8) : 0u;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                slot_of[n][e] = t.p0 + min(t.tokens - 1, (8 * n + 2 * t4 + e) / a.G);
                m[n][e] = kFewNone;
                l[n][e] = 0.f;
            }
            if constexpr (ACC) score[n] = score_at(a, 8 * n + 2 * t4) + (size_t)g * a.G;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k][n][e] = 0.f;
    }
    // The page in shared memory at sk, whose first slot is s0.
    __device__ __forceinline__ void page(const FewArgs& a, uint32_t sk, int s0) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
        const uint32_t k_row = (uint32_t)(lane & 15), k_chunk = (uint32_t)(lane >> 4);
        const uint32_t v_row = (uint32_t)((lane & 7) + ((lane >> 4) & 1) * 8), v_chunk = (uint32_t)((lane >> 3) & 1);
        const uint32_t sv = sk + NH * 2048;
        // every row sees every slot of the page
        const bool clear = s0 + 15 <= t.p0 && (s0 + 15 < a.sinks || s0 > p1 - a.window);
        float s[NT][4], s2[4] = {0.f, 0.f, 0.f, 0.f};  // one tile of rows: two chains
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t x[4];
            few_ldm<false>(x, sk + (k >> 2) * 2048 + k_row * 128 + (((2 * (k & 3) + k_chunk) ^ (k_row & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) few_mma(NT == 1 && (k & 1) ? s2 : s[n], x, qf[n][k][0], qf[n][k][1]);
        }
        if constexpr (NT == 1)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0][e] += s2[e];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] = __fmul_rn(s[n][e], a.scale_log2);  // (rounded by itself: the largest less m is exact)
                if (!clear) {
                    const int slot = s0 + g + 8 * (e >> 1), p = slot_of[n][e & 1];
                    if (!(slot <= p && (slot < a.sinks || slot > p - a.window))) s[n][e] = -INFINITY;
                }
            }
            if constexpr (ACC) {  // the rows' scores, for their weights once the rows' sums are known
                const int row = 8 * n + 2 * t4;
                float* dst = score[n] + (size_t)s0 * a.G;
                if ((a.G & 1) == 0) {
                    if (row < rows) {
                        *reinterpret_cast<float2*>(dst) = make_float2(s[n][0], s[n][1]);
                        *reinterpret_cast<float2*>(dst + 8 * a.G) = make_float2(s[n][2], s[n][3]);
                    }
                } else {
                    if (row < rows) {
                        dst[0] = s[n][0];
                        dst[8 * a.G] = s[n][2];
                    }
                    if (row + 1 < rows) {
                        float* d1 = score_at(a, row + 1) + (size_t)(s0 + g) * a.G;
                        d1[0] = s[n][1];
                        d1[8 * a.G] = s[n][3];
                    }
                }
            }
            // (also for NaN)
            grow |= !(few_max(s[n][0], s[n][2]) - m[n][0] <= kFewTop) || !(few_max(s[n][1], s[n][3]) - m[n][1] <= kFewTop);
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = few_max(s[n][e], s[n][2 + e]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = few_max(top, __shfl_xor_sync(0xffffffffu, top, d));
                    f[e] = 1.f;
                    if (!(top - m[n][e] <= kFewTop)) {
                        // a NaN or infinite maximum makes every weight, and so the row, NaN; far from 0 the 11 would
                        // be lost in rounding
                        const float now = top < INFINITY ? (fabsf(top) < 0x1p20f ? top - kFewLift : top)
                                                         : __int_as_float(0x7FC00000);
                        f[e] = m[n][e] == kFewNone ? 0.f : exp2f(m[n][e] - now);
                        m[n][e] = now;
                        l[n][e] *= f[e];
                    }
                }
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[k][n][e] *= f[e & 1];
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = few_exp2(s[n][e] - m[n][e & 1]);
            l[n][0] += y[0] + y[2];
            l[n][1] += y[1] + y[3];
            const __half2 h0 = __floats2half2_rn(y[0], y[1]), h1 = __floats2half2_rn(y[2], y[3]);
            pb[n][0] = few_turn(*reinterpret_cast<const uint32_t*>(&h0));
            pb[n][1] = few_turn(*reinterpret_cast<const uint32_t*>(&h1));
        }
        // V: slots that no row sees may hold anything and become 0; infinities and NaN of slots that some rows see
        // too (0 * NaN would reach the others), and the rows look them up at the end
        uint32_t keep[2] = {0xFFFFFFFFu, 0xFFFFFFFFu}, some[2] = {0u, 0u};
        if (!clear) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int slot = s0 + 2 * t4 + (e & 1) + 8 * (e >> 1);
                const bool any = slot <= p1 && (slot < a.sinks || slot > t.p0 - a.window);
                const bool all = slot <= t.p0 && (slot < a.sinks || slot > p1 - a.window);
                const uint32_t half = e & 1 ? 0xFFFF0000u : 0xFFFFu;
                if (!any) keep[e >> 1] &= ~half;
                else if (!all) some[e >> 1] |= half;
            }
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t x[4];
            few_ldm<true>(x, sv + (k >> 2) * 2048 + v_row * 128 + (((2 * (k & 3) + v_chunk) ^ (v_row & 7)) << 4));
            if (!clear) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] &= keep[e >> 1];
                    uint32_t wild = 0;
                    if ((x[e] & 0x7C00u) == 0x7C00u) wild |= 0xFFFFu;
                    if ((x[e] & 0x7C000000u) == 0x7C000000u) wild |= 0xFFFF0000u;
                    wild &= some[e >> 1];
                    bad |= wild != 0;
                    x[e] &= ~wild;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) few_mma(o[k][n], x, pb[n][0], pb[n][1]);
        }
    }
};

template <int HD, int NT, bool ACC>
__global__ void __launch_bounds__(32 * kFewWarps, few_resident(NT))
    few_rows_kernel(const __grid_constant__ CUtensorMap kvmap, const __grid_constant__ FewArgs a) {
    using C = FewCfg<HD, NT>;
    constexpr int KS = HD / 16, RING = C::RING;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + kFewWarps * RING * C::PAGE);
    long long* pre = reinterpret_cast<long long*>(bars + kFewWarps * RING);
    FewSeq* seqs = reinterpret_cast<FewSeq*>(pre + a.B + 1);
    pdl_trigger();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = s_addr(base + warp * RING * C::PAGE), bar = s_addr(bars + warp * RING);
    if (lane == 0) {
        for (int i = 0; i < RING; ++i) mbar_init(bar + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const long long total = few_plan(a, pre, seqs, ACC);  // ends with a CTA-wide barrier
    const FewCut cut(a, total);
    // neighbouring ranges on different SMs: a call of few ranges has them to itself
    const int wave = blockIdx.x / a.ctas, range = (wave * kFewWarps + warp) * a.ctas + (blockIdx.x - wave * a.ctas);
    const long long u0 = cut.begin(range), u1 = cut.end(range);
    if (u0 >= u1) return;

    // ---- loads: as many pages ahead as the ring holds
    FewWalk ld = {};
    ld.u = u0;
    ld.hi = u1;
    int asked = 0, tb = 0, ent = 0, ent_next = 0;  // pages asked for; table entries tb + lane, tb + 32 + lane
    bool more = true;
    auto entry = [&](int v) -> int {
        if (v >= ld.ve) return 0;
        const int x = a.tables[(size_t)ld.b * a.max_blocks + (v < ld.t.sinkp ? v : v + ld.t.gap)];
        return x < 0 || x >= a.num_blocks ? 0 : x;  // a malformed table reads block 0, never out of range
    };
    auto load = [&]() {
        while (more && ld.v >= ld.ve) {
            more = few_next(a, pre, seqs, ld);
            if (more) {
                tb = ld.v;
                ent = entry(tb + lane);
                ent_next = entry(tb + 32 + lane);
            }
        }
        if (!more) return;
        if (ld.v - tb >= 32) {
            tb += 32;
            ent = ent_next;
            ent_next = entry(tb + 32 + lane);
        }
        const int page = __shfl_sync(0xffffffffu, ent, ld.v - tb);
        if (lane == 0) {
            const uint32_t b = bar + 8 * (asked % RING);
            mbar_expect_tx(b, C::PAGE);
            tma_load_5d(ring + (asked % RING) * C::PAGE, &kvmap, 0, ld.kvh * 16, 0, 0, page, b);
        }
        ++asked;
        ++ld.v;
    };
    for (int i = 0; i < RING; ++i) load();

    // ---- arithmetic
    FewWalk w = {};
    w.u = u0;
    w.hi = u1;
    int done = 0;
    bool ok = true;
    while (ok && few_next(a, pre, seqs, w)) {
        const FewTile& t = w.t;
        const int rows = t.tokens * a.G;
        FewWork<HD, NT, ACC> f;
        f.begin(a, t, w.kvh);
        for (int v = w.v; v < w.ve; ++v) {
            const int at = done % RING;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar + 8 * at, (uint32_t)(done / RING) & 1u)))) break;
            const uint32_t sk = ring + at * C::PAGE;
            const int s0 = 16 * (v < t.sinkp ? v : v + t.gap);
            f.page(a, sk, s0);
            ++done;
            __syncwarp();  // the page has been read
            load();
        }
        if (!ok) break;
        // ---- the segment's rows
        const bool bad = __any_sync(0xffffffffu, f.bad);
        const int piece = 2 * range + (w.begun == u0 ? 0 : 1);
        if (w.v >= w.ve && !w.whole) continue;  // behind the tile's pages
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = f.l[n][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const int row = 8 * n + 2 * t4 + e;
                const bool real = row < rows;
                const int tok = row / a.G, head = w.kvh * a.G + (row - tok * a.G), r = t.row + tok;
                bool wild = bad;
                if (w.whole) {
                    const float inv = sum > 0.f || sum != sum ? 1.0f / sum : 0.f;
                    __half* dst = a.out + (size_t)r * a.ldo + (size_t)head * HD;
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float y = f.o[k][n][e + 2 * h] * inv;
                            wild |= !(fabsf(y) < INFINITY);
                            // (a finite mean that rounding took past fp16's largest)
                            if (real) dst[16 * k + 8 * h + g] = __float2half_rn(y == y ? fminf(fmaxf(y, -kFewMax), kFewMax) : y);
                        }
                    if (ACC && real && g == 0) a.ml[(size_t)r * a.Hq + head] = make_float2(f.m[n][e], inv);
                    const uint32_t look = __ballot_sync(0xffffffffu, real && wild && sum == sum);
                    for (int q = 0; q < 4; ++q) {  // rows that met an infinity or a NaN
                        if (!(look & (0x11111111u << q))) continue;
                        const int row_q = 8 * n + 2 * q + e, tok_q = row_q / a.G, head_q = w.kvh * a.G + (row_q - tok_q * a.G);
                        __syncwarp();
                        few_nonfinite<HD>(a, w.b, t.p0 + tok_q, w.kvh,
                                          a.out + (size_t)(t.row + tok_q) * a.ldo + (size_t)head_q * HD);
                    }
                } else {
                    float* dst = a.po + ((size_t)piece * (8 * NT) + row) * HD;
#pragma unroll
                    for (int k = 0; k < KS; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float y = f.o[k][n][e + 2 * h];
                            wild |= !(fabsf(y) < INFINITY);
                            if (real) dst[16 * k + 8 * h + g] = y;
                        }
                    wild = (__ballot_sync(0xffffffffu, wild) & (0x11111111u << t4)) != 0;
                    if (real && g == 0) a.pml[(size_t)piece * (8 * NT) + row] = make_float2(f.m[n][e], wild ? -sum : sum);
                }
            }
        }
    }
    if (!ok) {
        if (lane == 0) record_timeout(a.status, 40);
        // the copies in flight land before the CTA leaves
        for (int c = done; c < asked; ++c) (void)mbar_wait(bar + 8 * (c % RING), (uint32_t)(c / RING) & 1u);
    }
}

// Chunks: a CTA for each sequence, KV head and run of `chunk` pages, whose warps take
// the pages in turn and join what they have in shared memory.  Where the run is all
// there is the result is final, and the CTA adds up its slots' weights too: one
// launch for short tables.  CTAs come to the SMs as these are free, which evens out
// both ragged lengths and the SMs' shares of the memory's rate (64 single tokens on
// 2000, 8 heads of 128: 96 us, ranges 108).
constexpr int kChunkMost = 128, kChunkLeast = 64;  // pages (four table entries of a lane)
constexpr int kChunkCtas = 4096;                   // of a call at most

template <int HD, int WARPS>
struct ChunkCfg {
    static constexpr int PAGE = 64 * HD, RING = HD == 128 ? 2 : 4;  // a warp's ring holds its rows' O afterwards
    static constexpr size_t smem(int NT) {
        return 1024 + (size_t)WARPS * RING * (PAGE + 8) + (size_t)WARPS * 8 * NT * 8 + 8 * NT * 8;
    }
    static_assert(RING * PAGE >= kFewMaxRows * HD * 4, "a warp's O");
};

template <int HD, int NT, bool ACC, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 8 ? 1 : NT == 1 ? 3 : 2)
    chunk_rows_kernel(const __grid_constant__ CUtensorMap kvmap, const __grid_constant__ FewArgs a) {
    using C = ChunkCfg<HD, WARPS>;
    constexpr int KS = HD / 16, RING = C::RING, W = HD / 32;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + WARPS * RING * C::PAGE);
    float2* pml = reinterpret_cast<float2*>(bars + WARPS * RING);  // [warp][row] m, l (l < 0: look V up again)
    float2* lse = pml + WARPS * 8 * NT;                            // [row] m, 1 / l
    pdl_trigger();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const int kvh = blockIdx.x, b = blockIdx.y, v0 = blockIdx.z * a.chunk;
    const uint32_t ring = s_addr(base + warp * RING * C::PAGE), bar = s_addr(bars + warp * RING);
    const float* own_o = reinterpret_cast<const float*>(base);
    const FewSeq s = few_seq(a, b);
    if (s.n == 0 || (v0 > 0 && v0 >= few_pages(a, s))) return;
    const bool all = (min(s.ctx + s.n, a.slots_max) + 15) >> 4 <= a.chunk;  // no tile of the sequence has another piece
    if (lane == 0) {
        for (int i = 0; i < RING; ++i) mbar_init(bar + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    int asked = 0, done = 0;
    bool ok = true;
    const int tiles = (s.n + a.tpt - 1) / a.tpt;
    for (int tile = 0; tile < tiles; ++tile) {
        const FewTile t = few_tile(a, s, tile);
        if (v0 > 0 && v0 >= t.np) continue;  // (the same for all)
        const int rows = t.tokens * a.G, ve = min(t.np, v0 + a.chunk);
        const bool whole = v0 == 0 && t.np <= a.chunk;
        int ent[kChunkMost / 32];
#pragma unroll
        for (int i = 0; i < kChunkMost / 32; ++i) {
            const int v = v0 + 32 * i + lane;
            ent[i] = v < ve ? a.tables[(size_t)b * a.max_blocks + (v < t.sinkp ? v : v + t.gap)] : 0;
        }
        int next = v0 + warp;  // page to ask for
        auto load = [&]() {
            if (next >= ve) return;
            int page = ent[0];
#pragma unroll
            for (int i = 1; i < kChunkMost / 32; ++i) page = (next - v0) >> 5 == i ? ent[i] : page;
            page = __shfl_sync(0xffffffffu, page, (next - v0) & 31);
            if (page < 0 || page >= a.num_blocks) page = 0;  // a malformed table reads block 0, never out of range
            if (lane == 0) {
                const uint32_t at = bar + 8 * (asked % RING);
                mbar_expect_tx(at, C::PAGE);
                tma_load_5d(ring + (asked % RING) * C::PAGE, &kvmap, 0, kvh * 16, 0, 0, page, at);
            }
            ++asked;
            next += WARPS;
        };
        for (int i = 0; i < RING; ++i) load();
        FewWork<HD, NT, ACC> f;
        f.begin(a, t, kvh);
        for (int v = v0 + warp; v < ve && ok; v += WARPS) {
            const int at = done % RING;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar + 8 * at, (uint32_t)(done / RING) & 1u)))) break;
            f.page(a, ring + at * C::PAGE, 16 * (v < t.sinkp ? v : v + t.gap));
            ++done;
            __syncwarp();  // the page has been read
            load();
        }
        if (!ok) {
            if (lane == 0) record_timeout(a.status, 42);
            // the copies in flight land before anything else is done with their places
            for (int c = done; c < asked; ++c) (void)mbar_wait(bar + 8 * (c % RING), (uint32_t)(c / RING) & 1u);
            done = asked;
        }
        // this warp's part, over its ring
        float* mine = reinterpret_cast<float*>(base + warp * RING * C::PAGE);
        bool wild = f.bad;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = f.l[n][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const int row = 8 * n + 2 * t4 + e;
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float y = f.o[k][n][e + 2 * h];
                        wild |= !(fabsf(y) < INFINITY);
                        mine[row * HD + 16 * k + 8 * h + g] = y;
                    }
                wild = __any_sync(0xffffffffu, wild);
                if (g == 0) pml[warp * 8 * NT + row] = make_float2(f.m[n][e], wild ? -sum : sum);
            }
        __syncthreads();
        // rows of the tile, a warp for each in turn
        for (int row = warp; row < rows; row += WARPS) {
            const int tok = row / a.G, head = kvh * a.G + row - tok * a.G, r = t.row + tok;
            float M = -INFINITY, l = 0.f, y[W] = {};
            bool look = false;
#pragma unroll
            for (int q = 0; q < WARPS; ++q) M = few_max(M, pml[q * 8 * NT + row].x);
#pragma unroll
            for (int q = 0; q < WARPS; ++q) {
                const float2 ml = pml[q * 8 * NT + row];
                look |= !(ml.y >= 0.f);
                const float w = exp2f(ml.x - M);
                if (w == 0.f) continue;  // a part without weight may hold anything
                l += w * fabsf(ml.y);
                const float* src = own_o + q * (RING * C::PAGE / 4) + row * HD + lane * W;
#pragma unroll
                for (int e = 0; e < W; ++e) y[e] += w * src[e];
            }
            if (!whole) {
                const size_t at = ((size_t)r * a.Hq + head) * a.chunks + blockIdx.z;
#pragma unroll
                for (int e = 0; e < W; ++e) a.po[at * HD + lane * W + e] = y[e];
                if (lane == 0) a.pml[at] = make_float2(M, look ? -l : l);
                continue;
            }
            const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
            __half* dst = a.out + (size_t)r * a.ldo + (size_t)head * HD;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const float x = y[e] * inv;
                look |= !(fabsf(x) < INFINITY);
                dst[lane * W + e] = __float2half_rn(x == x ? fminf(fmaxf(x, -kFewMax), kFewMax) : x);
            }
            if (ACC && lane == 0) {
                lse[row] = make_float2(M, inv);
                if (!all) a.ml[(size_t)r * a.Hq + head] = make_float2(M, inv);
            }
            if (__any_sync(0xffffffffu, look) && l == l) {
                __syncwarp();
                few_nonfinite<HD>(a, b, t.p0 + tok, kvh, dst);
            }
        }
        fence_async_smem();  // the rings were written and read here: the next tile's loads come behind it
        __syncthreads();
        if constexpr (ACC) {
            if (all) {
                float* weights = a.weights + ((size_t)b * a.Hkv + kvh) * a.ldw;
                const int end = min(t.p0 + t.tokens, a.slots_max);
                // four slots of a thread at a time, so that their loads are out together
                for (int j0 = threadIdx.x; j0 < end; j0 += 4 * 32 * WARPS) {
                    float sum[4] = {}, was[4] = {};
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (j0 + 32 * WARPS * u < end) was[u] = weights[j0 + 32 * WARPS * u];
                    for (int tok = max(0, j0 - t.p0); tok < t.tokens; ++tok) {
                        const float* src = f.score_at(a, tok * a.G);
                        const float2* y = lse + tok * a.G;
                        const int last = min(t.p0 + tok, end - 1);
                        if ((a.G & 3) == 0) {
                            for (int h = 0; h < a.G; h += 4) {
                                float4 x[4];
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    if (j0 + 32 * WARPS * u <= last)
                                        x[u] = *reinterpret_cast<const float4*>(src + (size_t)(j0 + 32 * WARPS * u) * a.G + h);
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    if (j0 + 32 * WARPS * u <= last)
                                        sum[u] += few_exp2(x[u].x - y[h].x) * y[h].y + few_exp2(x[u].y - y[h + 1].x) * y[h + 1].y +
                                                  few_exp2(x[u].z - y[h + 2].x) * y[h + 2].y + few_exp2(x[u].w - y[h + 3].x) * y[h + 3].y;
                            }
                        } else {
                            for (int h = 0; h < a.G; ++h) {
                                float x[4];
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    if (j0 + 32 * WARPS * u <= last) x[u] = src[(size_t)(j0 + 32 * WARPS * u) * a.G + h];
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    if (j0 + 32 * WARPS * u <= last) sum[u] += few_exp2(x[u] - y[h].x) * y[h].y;
                            }
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (j0 + 32 * WARPS * u < end) weights[j0 + 32 * WARPS * u] = was[u] + sum[u];
                }
            }
        }
    }
}

// out = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p over a row's pieces, in their
// order: a warp for each row and head of up to 8 pieces, else the CTA's WARPS warps
// take pieces in turn and are joined in their order.  ROWS: rows of a CTA, 1 where
// there are few (one token on 65,520: 57 us a call with four rows of a CTA one
// after the other, 48 with one; 91 and 56 in ranges, under a wider table).  Where
// the row belongs is looked up while the kernel before still runs.
template <int HD, int ROWS, int WARPS>
__device__ __forceinline__ void few_merge(const FewArgs& a, int tile_rows, unsigned block) {
    constexpr int W = HD / 32;
    static_assert(ROWS == 1 || ROWS == WARPS, "rows of a CTA");
    __shared__ float sm[WARPS], sl[WARPS], so[WARPS][HD];
    __shared__ int sbad[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long rows = (long long)a.T * a.Hq, first = (long long)ROWS * block;
    struct Row {
        int n, b, p, kvh, row, np, tile, r0;
        long long u0;
        __half* dst;
        size_t at;
    };
    auto find = [&](long long idx) {
        Row x;
        x.n = x.np = x.r0 = 0;
        x.u0 = 0;
        if (idx >= rows) return x;
        const int r = (int)(idx / a.Hq), head = (int)(idx - (long long)r * a.Hq);
        int lo = 0, hi = a.B;  // first sequence whose end is past the row
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.row_off[mid + 1] > r) hi = mid;
            else lo = mid + 1;
        }
        if (lo >= a.B) return x;
        const FewSeq s = few_seq(a, lo);
        const int i = r - s.lo;
        if (i < 0 || i >= s.n) return x;
        x.tile = i / a.tpt;
        x.np = few_tile(a, s, x.tile).np;
        x.b = lo;
        x.p = s.ctx + i;
        x.kvh = head / a.G;
        x.row = (i - x.tile * a.tpt) * a.G + head - x.kvh * a.G;
        x.dst = a.out + (size_t)r * a.ldo + (size_t)head * HD;
        x.at = (size_t)r * a.Hq + head;
        return x;
    };
    Row mine = find(first + (ROWS == 1 ? 0 : warp));
    pdl_wait();
    const FewCut cut(a, a.chunk ? 0 : a.pre[a.B]);
    auto count = [&](Row& x) {  // its pieces
        if (x.np <= 0) return;
        if (a.chunk) {
            x.n = (x.np + a.chunk - 1) / a.chunk;
            return;
        }
        x.u0 = a.pre[x.b] + ((long long)x.tile * a.Hkv + x.kvh) * a.np[x.b];
        x.r0 = cut.of(x.u0);
        x.n = cut.of(x.u0 + x.np - 1) - x.r0 + 1;
    };
    count(mine);
    float m, l, o[W];
    bool bad;
    auto join = [&](const Row& x, int k0, int step) {  // pieces k0, k0 + step, ..
        m = -INFINITY;
        l = 0.f;
        bad = false;
#pragma unroll
        for (int e = 0; e < W; ++e) o[e] = 0.f;
        constexpr int P = 8;
        for (int k = k0; k < x.n; k += P * step) {
            float2 ml[P];
            float v[P][W];
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const bool real = k + u * step < x.n;
                const int range = x.r0 + k + u * step;
                size_t at = 0;
                if (real) at = a.chunk ? x.at * a.chunks + k + u * step
                                       : (size_t)(2 * range + (x.u0 > cut.begin(range) ? 1 : 0)) * tile_rows + x.row;
                ml[u] = real ? a.pml[at] : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int e = 0; e < W; ++e) v[u][e] = real ? a.po[at * HD + lane * W + e] : 0.f;
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                top = few_max(top, ml[u].x);
                bad |= !(ml[u].y >= 0.f);
            }
            const float sub = top == -INFINITY ? 0.f : top;
            const float f = exp2f(m - sub);
            m = top;
            l *= f;
#pragma unroll
            for (int e = 0; e < W; ++e) o[e] *= f;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const float w = exp2f(ml[u].x - sub);
                if (w == 0.f) continue;  // a piece without weight may hold anything
                l += w * fabsf(ml[u].y);
#pragma unroll
                for (int e = 0; e < W; ++e) o[e] += w * v[u][e];
            }
        }
    };
    auto finish = [&](const Row& x) {
        const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const float y = o[e] * inv;
            bad |= !(fabsf(y) < INFINITY);
            x.dst[lane * W + e] = __float2half_rn(y == y ? fminf(fmaxf(y, -kFewMax), kFewMax) : y);
        }
        if (a.ml && lane == 0) a.ml[x.at] = make_float2(m, inv);
        if (__any_sync(0xffffffffu, bad) && l == l) few_nonfinite<HD>(a, x.b, x.p, x.kvh, x.dst);
    };
    if (mine.n > 1 && mine.n <= 8 && (ROWS > 1 || warp == 0)) {
        join(mine, 0, 1);
        finish(mine);
    }
    if (!__syncthreads_or(mine.n > 8)) return;
    for (int k = 0; k < ROWS; ++k) {
        Row x = mine;
        if constexpr (ROWS > 1) {
            x = find(first + k);
            count(x);
        }
        if (x.n <= 8) continue;  // (the same for all)
        join(x, warp, WARPS);
        if (lane == 0) {
            sm[warp] = m;
            sl[warp] = l;
            sbad[warp] = bad;
        }
#pragma unroll
        for (int e = 0; e < W; ++e) so[warp][lane * W + e] = o[e];
        __syncthreads();
        if (warp == 0) {
            float top = sm[0];
            for (int q = 1; q < WARPS; ++q) top = few_max(top, sm[q]);
            const float sub = top == -INFINITY ? 0.f : top;
            m = top;
            l = 0.f;
            bad = false;
#pragma unroll
            for (int e = 0; e < W; ++e) o[e] = 0.f;
            for (int q = 0; q < WARPS; ++q) {
                const float w = exp2f(sm[q] - sub);
                bad |= sbad[q] != 0;
                if (w == 0.f) continue;
                l += w * sl[q];
#pragma unroll
                for (int e = 0; e < W; ++e) o[e] += w * so[q][lane * W + e];
            }
            finish(x);
        }
        __syncthreads();
    }
}

template <int HD, int ROWS, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) few_merge_kernel(const __grid_constant__ FewArgs a, int tile_rows) {
    pdl_trigger();
    few_merge<HD, ROWS, WARPS>(a, tile_rows, blockIdx.x);
}

// A row's weights of up to four slots j + STEP u <= last, added to sum: src its scores [slot][G], ml its heads' (m, 1 / l).
template <int V, int STEP>
__device__ __forceinline__ void few_weigh(const float* src, const float2* ml, int G, int j, int last, float (&sum)[4]) {
    for (int g = 0; g < G; g += V) {
        float x[4][V];
        float2 y[V];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float* at = src + (size_t)(j + STEP * u) * G + g;
            if (j + STEP * u <= last) {
                if constexpr (V == 4) {
                    const float4 f = *reinterpret_cast<const float4*>(at);
                    x[u][0] = f.x, x[u][1] = f.y, x[u][2] = f.z, x[u][3] = f.w;
                } else if constexpr (V == 2) {
                    const float2 f = *reinterpret_cast<const float2*>(at);
                    x[u][0] = f.x, x[u][1] = f.y;
                } else {
                    x[u][0] = *at;
                }
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = ml[g + v];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j + STEP * u <= last)
#pragma unroll
                for (int v = 0; v < V; ++v) sum[u] += few_exp2(x[u][v] - y[v].x) * y[v].y;
    }
}

// weights[b][kvh][j] += sum over the rows that see slot j, and the group's heads,
// of 2^(x - m) / l, from the scores that the attention left.  A warp for 128 slots of
// a head, four a lane; V heads' scores in one load.
template <int V>
__global__ void __launch_bounds__(256) few_weights_kernel(const __grid_constant__ FewArgs a) {
    extern __shared__ int runs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (a.chunk) {  // blocks (1024 slots, KV head, sequence)
        const FewSeq s = few_seq(a, blockIdx.z);
        const int end = min(s.ctx + s.n, a.slots_max);
        // (short sequences: a CTA of the attention has added up its own)
        if (s.n == 0 || (end + 15) >> 4 <= a.chunk || 1024 * (int)blockIdx.x >= end) {
            if ((blockIdx.x | blockIdx.y | blockIdx.z) == 0) pdl_wait();  // who waits for this kernel waits for those before it
            return;
        }
    }
    pdl_wait();
    if (!a.chunk) {
        for (int b = threadIdx.x; b <= a.B; b += 256) runs[b] = a.runs[b];
        __syncthreads();
    }
    const int total = a.chunk ? 8 * (int)(blockIdx.x + 1) : runs[a.B];
    for (int c = blockIdx.x * 8 + warp; c < total; c += gridDim.x * 8) {
        int lo = a.chunk ? (int)blockIdx.z : 0, hi = a.chunk ? lo : a.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (runs[mid] <= c) lo = mid;
            else hi = mid;
        }
        const FewSeq s = few_seq(a, lo);
        int kvh = blockIdx.y, j0 = 128 * c;
        if (!a.chunk) {
            const int per_head = (runs[lo + 1] - runs[lo]) / a.Hkv, local = c - runs[lo];
            kvh = local / per_head;
            j0 = 128 * (local - kvh * per_head);
        }
        const int end = min(min(s.ctx + s.n, a.slots_max), j0 + 128);
        float* dst = a.weights + ((size_t)lo * a.Hkv + kvh) * a.ldw;
        float sum[4] = {}, was[4] = {};
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j0 + 32 * u + lane < end) was[u] = dst[j0 + 32 * u + lane];
        for (int i = max(0, j0 - s.ctx); i < s.n; ++i) {
            const int r = s.lo + i, p = min(s.ctx + i, end - 1);
            const float* src = a.scores + ((size_t)r * a.Hkv + kvh) * a.slots_max * a.G;
            const float2* ml = a.ml + (size_t)r * a.Hq + kvh * a.G;
            few_weigh<V, 32>(src, ml, a.G, j0 + lane, p, sum);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j0 + 32 * u + lane < end) dst[j0 + 32 * u + lane] = was[u] + sum[u];
    }
}

// Behind chunks of up to kFewJoin rows and heads, both in one launch: the rows' pieces
// joined by the first `merges` CTAs, and what the slots of sequences of more than one
// chunk received by the others, 512 slots of a KV head each, which join the rows'
// (m, l) for themselves, so neither waits for the other.  In place of two launches: one
// token of each of 4 sequences on 3000 17.4 -> 15.3 us a call, of 8 on 8192 57.9 -> 54.6.
// The merge's registers leave the weights fewer warps, which costs more where rows are
// many: of 64 on 4096 198.7 -> 200.4, of 148 419.7 -> 439.3, four of each of 64 251 -> 263.
constexpr long long kFewJoin = 1024;
template <int HD, int V>
__global__ void __launch_bounds__(128) few_join_kernel(const __grid_constant__ FewArgs a, int tile_rows, unsigned merges,
                                                       unsigned runs) {
    if (blockIdx.x < merges) {
        few_merge<HD, 1, 4>(a, tile_rows, blockIdx.x);
        return;
    }
    __shared__ float2 lse[64];
    const unsigned w = blockIdx.x - merges;
    const int b = (int)(w / runs / a.Hkv), kvh = (int)(w / runs % a.Hkv), j0 = 512 * (int)(w % runs);
    const FewSeq s = few_seq(a, b);
    const int end = min(s.ctx + s.n, a.slots_max);
    if (s.n == 0 || (end + 15) >> 4 <= a.chunk || j0 >= end) return;  // (one chunk: its CTA has added up its own)
    pdl_wait();
    const int j = j0 + (int)threadIdx.x, tokens = 64 / a.G;
    float* dst = a.weights + ((size_t)b * a.Hkv + kvh) * a.ldw;
    float sum[4] = {}, was[4] = {};
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (j + 128 * u < end) was[u] = dst[j + 128 * u];
    for (int i0 = max(0, j0 - s.ctx); i0 < s.n; i0 += tokens) {
        const int n = min(tokens, s.n - i0);
        __syncthreads();
        if ((int)threadIdx.x < n * a.G) {
            const int tok = i0 + (int)threadIdx.x / a.G, head = kvh * a.G + (int)threadIdx.x % a.G;
            const size_t at = (size_t)(s.lo + tok) * a.Hq + head;
            const int pieces = (few_tile(a, s, tok / a.tpt).np + a.chunk - 1) / a.chunk;
            if (pieces <= 1) {
                lse[threadIdx.x] = a.ml[at];
            } else {
                float m = -INFINITY, l = 0.f;
                for (int k = 0; k < pieces; ++k) m = few_max(m, a.pml[at * a.chunks + k].x);
                for (int k = 0; k < pieces; ++k) {
                    const float2 y = a.pml[at * a.chunks + k];
                    l += exp2f(y.x - m) * fabsf(y.y);
                }
                lse[threadIdx.x] = make_float2(m, l > 0.f || l != l ? 1.0f / l : 0.f);
            }
        }
        __syncthreads();
        for (int i = 0; i < n; ++i)
            few_weigh<V, 128>(a.scores + ((size_t)(s.lo + i0 + i) * a.Hkv + kvh) * a.slots_max * a.G, lse + i * a.G, a.G, j,
                              min(s.ctx + i0 + i, end - 1), sum);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (j + 128 * u < end) dst[j + 128 * u] = was[u] + sum[u];
}

// ------------------------------------------------------------------ many rows
//
// weights[b][kvh][j] += sum over the rows that see slot j, and the group's heads,
// of 2^(x - m) / l, where the rows' (m, 1 / l) are known (the packed-row kernel's):
// the scores are computed again rather than kept, a read of K (256 bytes of a slot
// and head of 128) against one write and one read of 4 bytes for each row.
//   S^T [128 slots][rows] = K Q^T by tcgen05.mma into tensor memory: a lane is a
// slot, so a thread sums its slot's weights over up to 128 rows by itself.  That is
// three instructions a score, half of what the memory takes for K at 64 rows
// (mma.sync fragments, 16 slots a warp, took twice the instructions and 42 us where
// this takes 17).  One CTA for a KV head and run of up to 1024 slots; warps:
//   0-3  sums, 4  MMA issuer, 5  loads (a group's queries, 128-slot tiles of K)
constexpr int kWeighTiles = 8, kWeighThreads = 192, kWeighTmem = 256;

template <int HD>
struct WeighCfg {
    static constexpr int NH = HD / 64, TILE = NH * 16384, RING = HD == 128 ? 2 : 4;
    static constexpr size_t smem = 1024 + (size_t)(1 + RING) * TILE + 128 * 8 + (2 * RING + 6) * 8 + 16;
};

template <int HD>
__global__ void __launch_bounds__(kWeighThreads, 2)
    weigh_rows_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ FewArgs a) {
    using C = WeighCfg<HD>;
    constexpr int NH = C::NH, RING = C::RING;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sQ = base;              // [NH][128 rows][128 B]
    unsigned char* sK = base + C::TILE;    // [RING][NH][128 slots][128 B]
    float2* lse = reinterpret_cast<float2*>(sK + RING * C::TILE);  // [row] m, 1 / l
    uint64_t* k_full = reinterpret_cast<uint64_t*>(lse + 128);
    uint64_t* k_empty = k_full + RING;
    uint64_t* q_full = k_empty + RING;
    uint64_t* q_empty = q_full + 1;
    uint64_t* s_full = q_empty + 1;  // [2] scores landed
    uint64_t* s_free = s_full + 2;   // [2] scores read (4 warps)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_free + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int kvh = blockIdx.x, b = blockIdx.y;
    const FewSeq s = few_seq(a, b);
    const int end = min(s.ctx + s.n, a.slots_max), tiles = (end + 127) >> 7, run = a.chunk, step = gridDim.z * run;
    const int first_tile = blockIdx.z * run;
    if (s.n == 0 || first_tile >= tiles) {
        if ((blockIdx.x | blockIdx.y | blockIdx.z) == 0) pdl_wait();  // who waits for this kernel waits for those before it
        return;
    }
    const int tpt = 128 / a.G, groups = (s.n + tpt - 1) / tpt;  // tokens of a group of rows
    if (threadIdx.x == 0) {
        for (int i = 0; i < RING; ++i) {
            mbar_init(s_addr(&k_full[i]), 1);
            mbar_init(s_addr(&k_empty[i]), 1);
        }
        mbar_init(s_addr(q_full), 1);
        mbar_init(s_addr(q_empty), 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_addr(&s_full[i]), 1);
            mbar_init(s_addr(&s_free[i]), 4);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_slot)),
                     "r"(kWeighTmem));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    auto wait = [&](uint64_t* bar, int turn) -> bool {  // false: it ran out, here or in another role
        const bool ok = __all_sync(0xffffffffu, mbar_wait(s_addr(bar), (uint32_t)turn & 1u)) != 0;
        if (!ok && lane == 0) {
            *abort_flag = 1;
            record_timeout(a.status, 41);
        }
        return ok && !__any_sync(0xffffffffu, *abort_flag != 0);
    };
    // every role goes through the groups, and in each through the CTA's tiles
    if (warp == 5) {
        int kc = 0, qc = 0;
        bool ok = true;
        for (int k = 0; ok && k < groups; ++k) {
            for (int t0 = first_tile; ok && t0 < tiles; t0 += step)
                for (int tile = t0; tile < min(tiles, t0 + run); ++tile) {
                    const int pages = min(8, ((end + 15) >> 4) - 8 * tile), at = kc % RING, turn = kc / RING;
                    int page = 0;
                    if (lane < pages * NH) page = a.tables[(size_t)b * a.max_blocks + 8 * tile + lane / NH];
                    if (page < 0 || page >= a.num_blocks) page = 0;  // a malformed table reads block 0, never out of range
                    if (turn && !(ok = wait(&k_empty[at], turn - 1))) break;
                    if (lane == 0) mbar_expect_tx(s_addr(&k_full[at]), (uint32_t)(pages * NH * 2048));
                    __syncwarp();
                    if (lane < pages * NH)
                        tma_load_5d(s_addr(sK + at * C::TILE + (lane % NH) * 16384 + (lane / NH) * 2048), &kmap, 0, kvh * 16,
                                    lane % NH, 0, page, s_addr(&k_full[at]));
                    ++kc;
                    if (tile == first_tile) {  // the group's queries, behind its first keys
                        if (k && !(ok = wait(q_empty, k - 1))) break;
                        if (lane == 0) {
                            mbar_expect_tx(s_addr(q_full), (uint32_t)(tpt * a.G * 128 * NH));
                            for (int h = 0; h < NH; ++h)
                                tma_load_4d(s_addr(sQ + h * 16384), &qmap, 0, h, kvh * a.G, s.lo + k * tpt, s_addr(q_full));
                        }
                        __syncwarp();
                        ++qc;
                    }
                }
        }
        // the copies in flight land before the CTA leaves
        if (qc) (void)mbar_wait(s_addr(q_full), (uint32_t)(qc - 1) & 1u);
        for (int c = max(0, kc - RING); c < kc; ++c) (void)mbar_wait(s_addr(&k_full[c % RING]), (uint32_t)(c / RING) & 1u);
    } else if (warp == 4) {
        const uint64_t qd = sw128_desc(s_addr(sQ)), kd0 = sw128_desc(s_addr(sK));
        int kc = 0;
        bool ok = true;
        for (int k = 0; ok && k < groups; ++k) {
            const int rows = min(tpt, s.n - k * tpt) * a.G;
            const uint32_t idesc = idesc_f16(128, (rows + 15) & ~15);
            ok = wait(q_full, k);
            for (int t0 = first_tile; ok && t0 < tiles; t0 += step)
                for (int tile = t0; tile < min(tiles, t0 + run); ++tile, ++kc) {
                    const int at = kc % RING, buf = kc & 1;
                    if (!(ok = wait(&k_full[at], kc / RING))) break;
                    if (kc >= 2 && !(ok = wait(&s_free[buf], (kc >> 1) - 1))) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint64_t kd = kd0 + (uint64_t)(at * (C::TILE >> 4));
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk)
                            tc_mma_f16_ss(tmem + buf * 128, kd + (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4),
                                          qd + (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), idesc, kk > 0 ? 1u : 0u);
                        tc_commit(s_addr(&s_full[buf]));
                        tc_commit(s_addr(&k_empty[at]));
                        // (the group's last tile: commits cover all MMAs before them)
                        if (tile + 1 >= min(tiles, t0 + run) && t0 + step >= tiles) tc_commit(s_addr(q_empty));
                    }
                    __syncwarp();
                }
        }
        // every MMA has finished with shared and tensor memory before the CTA leaves
        if (kc > 0) (void)mbar_wait(s_addr(&s_full[(kc - 1) & 1]), (uint32_t)((kc - 1) >> 1) & 1u);
        __syncwarp();
    } else {
        pdl_wait();  // m and l of the rows
        const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
        float* weights = a.weights + ((size_t)b * a.Hkv + kvh) * a.ldw;
        int kc = 0;
        bool ok = true;
        for (int k = 0; k < groups; ++k) {  // (all of them: the four warps meet at the barriers also where one gave up)
            const int tokens = min(tpt, s.n - k * tpt), rows = tokens * a.G, p0 = s.ctx + k * tpt, p1 = p0 + tokens - 1;
            asm volatile("bar.sync 1, 128;" ::: "memory");  // the rows before have been read
            {
                const int c = threadIdx.x, tok = c / a.G;
                float2 y = make_float2(0.f, 0.f);
                if (c < rows) y = __ldcg(a.ml + (size_t)(s.lo + k * tpt + tok) * a.Hq + kvh * a.G + c - tok * a.G);
                if (y.x == -INFINITY) y.x = 0.f;
                lse[c] = y;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int t0 = first_tile; ok && t0 < tiles; t0 += step)
                for (int tile = t0; tile < min(tiles, t0 + run); ++tile, ++kc) {
                    const int buf = kc & 1, j = 128 * tile + threadIdx.x;
                    const bool keeps = j <= p1 && j < end;
                    const float was = keeps ? weights[j] : 0.f;
                    const int from = max(0, j - p0) * a.G;  // the first row that sees this slot
                    const bool clear = 128 * tile + 127 <= p0;
                    if (!(ok = wait(&s_full[buf], kc >> 1))) break;
                    tc_fence_after();
                    float sum[4] = {};
                    const bool here = 128 * tile + 32 * warp <= p1;  // some row sees a slot of this warp
                    if (here) {
                        for (int c0 = 0; c0 < rows; c0 += 32) {
                            uint32_t v[32];
                            __syncwarp();
                            tc_ld_x32(t_lane + buf * 128 + c0, v);
                            tc_wait_ld();
                            if (clear && c0 + 32 <= rows) {
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    const float2 y = lse[c0 + e];
                                    sum[e & 3] = fmaf(few_exp2(__fmul_rn(__uint_as_float(v[e]), a.scale_log2) - y.x), y.y, sum[e & 3]);
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    const float2 y = lse[c0 + e];
                                    const float w = few_exp2(__fmul_rn(__uint_as_float(v[e]), a.scale_log2) - y.x) * y.y;
                                    if (c0 + e >= from && c0 + e < rows) sum[e & 3] += w;
                                }
                            }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_addr(&s_free[buf]));
                    if (keeps) weights[j] = was + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kWeighTmem));
    }
}

// ------------------------------------------------------------------ host side
static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// Pages of a run and runs of a table where every run has a CTA; 0 pages where too
// many of them might be empty (tables far wider than most sequences): ranges, which
// are cut by the lengths in device memory.
struct FewChunks {
    int pages, count;
};
static FewChunks few_chunks(int B, int Hkv, int max_blocks) {
    const long long pairs = (long long)B * Hkv, all = pairs * max_blocks;
    // whole tables where they are short; else runs for two CTAs of each SM
    const int pages = (int)std::min<long long>(kChunkMost, std::max<long long>(kChunkLeast, (all + 2 * kFewMaxSms - 1) / (2 * kFewMaxSms)));
    const int count = (max_blocks + pages - 1) / pages;
    if (pairs * count > kChunkCtas || B > 65535 || count > 65535) return {0, 0};
    return {pages, count};
}
// CTAs of a wave: no more than there can be ranges.
static int few_ctas(int sms, int NT, int T, int Hkv, int max_blocks) {
    const long long ranges = ((long long)T * Hkv * max_blocks + kFewMinPages - 1) / kFewMinPages;
    return (int)std::min<long long>(few_resident(NT) * std::min(sms, kFewMaxSms), ranges);
}
// Weights of few rows keep their scores, up to 1 GiB of them; other calls compute them again.
constexpr size_t kFewScores = (size_t)1 << 30;
static size_t few_scores(int T, int Hq, int max_blocks) { return (size_t)T * Hq * max_blocks * 16 * sizeof(float); }
// Sizes that do not fall where B, T or max_blocks grows.
struct FewSpace {
    size_t pre, np, runs, pml, po, ml, scores, bytes;  // offsets, and all
};
static FewSpace few_space(int B, int T, int Hq, int Hkv, int HD, int max_blocks, bool acc) {
    FewSpace s = {};
    // rows of all pieces: two for each range, of the kernel that has most
    const long long rows = std::min<long long>(kFewMaxRows, ((long long)T * (Hq / Hkv) + 7) / 8 * 8);
    long long most = 0;
    for (int nt = 1; nt <= 4; ++nt)
        most = std::max(most, 2LL * few_waves(nt) * few_ctas(kFewMaxSms, nt, T, Hkv, max_blocks) * kFewWarps * std::min<long long>(8 * nt, rows));
    // or one for each run of a row and head: calls of few rows have at most kFewMaxRows rows for each of a sequence's heads' runs
    const long long runs = std::min<long long>((long long)T * Hq * ((max_blocks + kChunkLeast - 1) / kChunkLeast), (long long)kFewMaxRows * kChunkCtas);
    const size_t pieces = (size_t)std::max(most, runs);
    size_t at = 0;
    auto room = [&](size_t n) {
        const size_t here = at;
        at += up256(n);
        return here;
    };
    s.pre = room((size_t)(B + 1) * 8);
    s.np = room((size_t)B * 4);
    s.runs = room((size_t)(B + 1) * 4);
    s.pml = room(pieces * sizeof(float2));
    s.po = room(pieces * HD * sizeof(float));
    if (acc) {
        s.ml = room((size_t)T * Hq * sizeof(float2));
        s.scores = room(std::min(kFewScores, few_scores(T, Hq, max_blocks)));  // (calls with more keep none)
    }
    s.bytes = at;
    return s;
}

static const void* few_fn(int HD, int NT, bool acc) {
#define FEW_NT(hd, ac) \
    (NT == 1 ? (const void*)few_rows_kernel<hd, 1, ac> \
             : NT == 2 ? (const void*)few_rows_kernel<hd, 2, ac> \
                       : NT == 3 ? (const void*)few_rows_kernel<hd, 3, ac> : (const void*)few_rows_kernel<hd, 4, ac>)
    if (HD == 128) return acc ? FEW_NT(128, true) : FEW_NT(128, false);
    return acc ? FEW_NT(64, true) : FEW_NT(64, false);
#undef FEW_NT
}
template <int HD, bool ACC, int WARPS>
static const void* chunk_nt(int NT) {
    return NT == 1 ? (const void*)chunk_rows_kernel<HD, 1, ACC, WARPS>
           : NT == 2 ? (const void*)chunk_rows_kernel<HD, 2, ACC, WARPS>
           : NT == 3 ? (const void*)chunk_rows_kernel<HD, 3, ACC, WARPS> : (const void*)chunk_rows_kernel<HD, 4, ACC, WARPS>;
}
static const void* chunk_fn(int HD, int NT, bool acc, int warps) {
    if (HD == 128) return warps == 8 ? (acc ? chunk_nt<128, true, 8>(NT) : chunk_nt<128, false, 8>(NT))
                                     : (acc ? chunk_nt<128, true, 4>(NT) : chunk_nt<128, false, 4>(NT));
    return warps == 8 ? (acc ? chunk_nt<64, true, 8>(NT) : chunk_nt<64, false, 8>(NT))
                      : (acc ? chunk_nt<64, true, 4>(NT) : chunk_nt<64, false, 4>(NT));
}
static size_t chunk_smem(int HD, int NT, int warps) {
    return HD == 128 ? (warps == 8 ? ChunkCfg<128, 8>::smem(NT) : ChunkCfg<128, 4>::smem(NT))
                     : (warps == 8 ? ChunkCfg<64, 8>::smem(NT) : ChunkCfg<64, 4>::smem(NT));
}
static int few_sms(int* out) {  // SMs of the current device; sets the kernels' shared memory on it once
    static std::atomic<int> facts[64];
    int dev = 0;
    SD_CUDA(cudaGetDevice(&dev));
    SD_CHECK(dev >= 0 && dev < 64, SPECDEC_ENOTSUP, "attention: device index above 63");
    int n = facts[dev].load();
    if (!n) {
        for (int i = 0; i < 32; ++i) {
            const int hd = i & 1 ? 128 : 64, warps = i & 2 ? 8 : 4, acc = i >> 2 & 1, nt = (i >> 3) + 1;
            SD_CUDA(cudaFuncSetAttribute(chunk_fn(hd, nt, acc, warps), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)chunk_smem(hd, nt, warps)));
        }
        for (int nt = 1; nt <= 4; ++nt)
            for (int acc = 0; acc < 2; ++acc) {
                SD_CUDA(cudaFuncSetAttribute(few_fn(128, nt, acc), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)FewCfg<128, 2>::smem(kBoundMaxSeqs)));
                SD_CUDA(cudaFuncSetAttribute(few_fn(64, nt, acc), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)FewCfg<64, 2>::smem(kBoundMaxSeqs)));
            }
        SD_CUDA(cudaFuncSetAttribute(weigh_rows_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)WeighCfg<128>::smem));
        SD_CUDA(cudaFuncSetAttribute(weigh_rows_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)WeighCfg<64>::smem));
        SD_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        facts[dev].store(n);
    }
    *out = n;
    return SPECDEC_OK;
}

// Rows past kFewMaxRows a sequence with weights: the attention on the tensor cores, which leaves (m, 1 / l), then the weights.
static int launch_many(FewArgs a, int HD, void* ws, cudaStream_t s) {
    int sms = 0;
    int rc = few_sms(&sms);
    if (rc) return rc;
    a.ml = static_cast<float2*>(ws);
    a.status = device_status_ptr();
    a.slots_max = a.max_blocks * 16;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)HD));
    rc = rows_packed_launch(a.q, a.ldq, a.kv, a.num_blocks, a.Hkv, HD, a.tables, a.max_blocks, a.ctx_len, a.row_off, a.B,
                            a.T, a.Hq, a.window, 0, a.least, a.ml, a.out, a.ldo,
                            static_cast<char*>(ws) + up256((size_t)a.T * a.Hq * sizeof(float2)), s);
    if (rc) return rc;
    CUtensorMap qmap, kmap;
    if ((rc = make_q_tmap(&qmap, a.q, a.ldq, a.T, a.Hq, HD, a.G, 128 / a.G))) return rc;
    if ((rc = make_kv_tmap(&kmap, a.kv, a.num_blocks, a.Hkv, HD, 1, 1))) return rc;
    cudaLaunchConfig_t cfg = {};
    // a CTA for each run of slots (two for each SM, in tables that are full), or for several where tables are far wider
    // than most sequences
    const int tiles = (a.max_blocks + 7) / 8;
    a.chunk = (int)std::min<long long>(kWeighTiles, std::max<long long>(1, (long long)a.B * a.Hkv * tiles / (2 * kFewMaxSms)));
    const int runs = (tiles + a.chunk - 1) / a.chunk;
    cfg.gridDim = dim3((unsigned)a.Hkv, (unsigned)a.B, (unsigned)std::min(runs, std::max(1, kChunkCtas / (a.B * a.Hkv))));
    cfg.blockDim = dim3(kWeighThreads);
    cfg.dynamicSmemBytes = HD == 128 ? WeighCfg<128>::smem : WeighCfg<64>::smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    SD_CUDA(cudaLaunchKernelEx(&cfg, HD == 128 ? weigh_rows_kernel<128> : weigh_rows_kernel<64>, qmap, kmap, a));
    return SPECDEC_OK;
}

using FewJoin = void (*)(const FewArgs, int, unsigned, unsigned);
static FewJoin join_fn(int HD, int G) {
    const int v = G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
    if (HD == 128) return v == 4 ? few_join_kernel<128, 4> : v == 2 ? few_join_kernel<128, 2> : few_join_kernel<128, 1>;
    return v == 4 ? few_join_kernel<64, 4> : v == 2 ? few_join_kernel<64, 2> : few_join_kernel<64, 1>;
}

static int launch_few(FewArgs a, int HD, bool acc, void* ws, cudaStream_t s) {
    int sms = 0;
    int rc = few_sms(&sms);
    if (rc) return rc;
    const FewSpace sp = few_space(a.B, a.T, a.Hq, a.Hkv, HD, a.max_blocks, acc);
    char* w = static_cast<char*>(ws);
    a.pre = reinterpret_cast<long long*>(w + sp.pre);
    a.np = reinterpret_cast<int32_t*>(w + sp.np);
    a.runs = reinterpret_cast<int32_t*>(w + sp.runs);
    a.pml = reinterpret_cast<float2*>(w + sp.pml);
    a.po = reinterpret_cast<float*>(w + sp.po);
    a.ml = acc ? reinterpret_cast<float2*>(w + sp.ml) : nullptr;
    a.scores = acc ? reinterpret_cast<float*>(w + sp.scores) : nullptr;
    a.status = device_status_ptr();
    a.slots_max = a.max_blocks * 16;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)HD));
    // rows of a tile: what a sequence has on average
    const long long want = std::min<long long>(kFewMaxRows, (((long long)a.T + a.B - 1) / a.B) * a.G);
    const int NT = (int)((want + 7) / 8);
    a.tpt = 8 * NT / a.G;
    a.ctas = few_ctas(sms, NT, a.T, a.Hkv, a.max_blocks);
    a.waves = few_waves(NT);
    // With few pages for each warp the wave's pieces cost more than it gains, the sooner the more rows they have.  In us,
    // with one wave and with two, of 64 sequences under tables of 2048 pages, 8 heads of 128, L tokens (L * 32 / 1776
    // pages a warp at 3 CTAs of an SM): one row a piece on 1536 / 4096 / 12,288 73.6, 73.6 / 171, 168 / 487, 474; four
    // 89.7, 91.0 / 185, 180 / 493, 485; five 82.3, 97.5 / 180, 187 / 489, 489; eight 82.8, 96.9 / 181, 188 / 493, 494,
    // on 16,384 667, 663; sixteen on 2048 / 8192 / 16,384 125, 139 / 375, 381 / 718, 709.
    a.wave_pages = want <= 4 ? 24 : 200;
    CUtensorMap map;
    if ((rc = make_kv_tmap(&map, a.kv, a.num_blocks, a.Hkv, HD, HD / 64, 2))) return rc;
    const size_t few_smem = HD == 128 ? (NT == 1 ? FewCfg<128, 1>::smem(a.B) : FewCfg<128, 2>::smem(a.B))
                                  : (NT == 1 ? FewCfg<64, 1>::smem(a.B) : FewCfg<64, 2>::smem(a.B));
    const FewChunks ch = few_chunks(a.B, a.Hkv, a.max_blocks);
    a.chunk = ch.pages;
    a.chunks = ch.count;
    void* args[] = {&map, &a};
    if (a.chunk) {
        // (eight warps on a run where CTAs are few)
        const int warps = (long long)a.B * a.Hkv * a.chunks <= sms ? 8 : 4;
        SD_CUDA(cudaLaunchKernel(chunk_fn(HD, NT, acc, warps), dim3((unsigned)a.Hkv, (unsigned)a.B, (unsigned)a.chunks),
                                 dim3(32 * warps), args, chunk_smem(HD, NT, warps), s));
        if (a.chunks == 1) return SPECDEC_OK;
    } else {
        SD_CUDA(cudaLaunchKernel(few_fn(HD, NT, acc), dim3((unsigned)(a.ctas * a.waves)), dim3(32 * kFewWarps), args, few_smem, s));
    }
    cudaLaunchConfig_t cfg = {};
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const long long rows = (long long)a.T * a.Hq;
    const int kind = rows <= 256 ? 0 : rows <= 2048 ? 1 : 2;
    if (acc && a.chunk && rows <= kFewJoin) {
        const unsigned merges = (unsigned)rows, runs = (unsigned)((a.max_blocks + 31) / 32);
        cfg.gridDim = dim3(merges + runs * (unsigned)(a.B * a.Hkv));
        cfg.blockDim = dim3(128);
        SD_CUDA(cudaLaunchKernelEx(&cfg, join_fn(HD, a.G), a, 8 * NT, merges, runs));
        return SPECDEC_OK;
    }
    cfg.gridDim = dim3((unsigned)(kind < 2 ? rows : (rows + 3) / 4));
    cfg.blockDim = dim3(kind == 0 ? 512 : 128);
    const auto merge =
        HD == 128 ? (kind == 0 ? few_merge_kernel<128, 1, 16> : kind == 1 ? few_merge_kernel<128, 1, 4> : few_merge_kernel<128, 4, 4>)
                  : (kind == 0 ? few_merge_kernel<64, 1, 16> : kind == 1 ? few_merge_kernel<64, 1, 4> : few_merge_kernel<64, 4, 4>);
    SD_CUDA(cudaLaunchKernelEx(&cfg, merge, a, 8 * NT));
    if (acc) {
        const long long runs = (long long)a.B * a.Hkv * ((a.max_blocks + 7) / 8);
        cfg.gridDim = a.chunk ? dim3((unsigned)((a.max_blocks + 63) / 64), (unsigned)a.Hkv, (unsigned)a.B)
                              : dim3((unsigned)std::min<long long>((runs + 7) / 8, 8LL * sms));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = a.chunk ? 0 : (size_t)(a.B + 1) * 4;
        const auto weigh = a.G % 4 == 0 ? few_weights_kernel<4> : (a.G % 2 == 0 ? few_weights_kernel<2> : few_weights_kernel<1>);
        SD_CUDA(cudaLaunchKernelEx(&cfg, weigh, a));
    }
    return SPECDEC_OK;
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
    const struct {
        const void* p;
        const char* what;
    } given[] = {{q, "q"}, {kv, "the KV pool"}, {out, "out"}, {tables, "tables"}, {ctx_len, "ctx_len"},
                 {row_off, "row_off"}, {ws, "the workspace"}};
    for (const auto& g : given) {
        const int rc = check_on_device(g.p, g.what);
        if (rc) {
            set_error(std::string(who) + ": " + specdec_last_error());
            return rc;
        }
    }
    return SPECDEC_OK;
}

}  // namespace specdec

using namespace specdec;

static size_t accumulate_space(int B, int T, int Hq, int Hkv, int HD, int max_blocks) {
    const int most = (int)std::min<long long>(T, (long long)B * (kFewMaxRows / std::max(1, std::min(kFewMaxRows, Hq / Hkv))));
    return few_space(B, most, Hq, Hkv, HD, max_blocks, true).bytes + up256((size_t)T * Hq * sizeof(float2)) +
           rows_packed_workspace(B, T, Hq, HD, max_blocks);
}
static bool few_rows(int B, int T, int G) { return G <= kFewMaxRows && T <= (long long)B * (kFewMaxRows / G); }
// Rows that a sequence of a few-row call may have at most, else it is left to the packed rows' kernels; 0: there is no
// such bound.  A call's average says nothing of its longest sequence, whose tiles would go one after the other through
// the CTAs of its heads, each reading K and V again.  In us, 32/8 heads of 128, undivided / divided (with weights), and
// all by the packed rows' kernels without a window:
//   63 single tokens on 4096 beside 190 rows on 8000   1613 / 249 (2032 / 402), 212
//   31 beside 90                                        773 / 138 (982 / 211), 157
//   50, 10 rows on 8000, 10 empty sequences             253 / 174 (295 / 211), 165
// Where no sequence is long the other launches find nothing to do, for 8 to 18:
//   32 x 5 rows on 4096                                 105 / 114 (144 / 160), 123
//   32 x 5 on 512                                      22.4 / 30.4 (29.1 / 41.2), 39.6
//   64 x 2 on 2048                                      100 / 109 (120 / 138), 118
// So calls of up to one row a sequence, which are single tokens unless others are empty, are not divided.  If others are,
// a long one takes its time: 64 rows on 8000 among 63 empty sequences 787 (922), alone 36 (52).
static int few_most(int B, int T, int G) {
    const int most = kFewMaxRows / G;
    return T > B && T > most ? most : 0;
}
static FewArgs few_args(const uint16_t* q, int ldq, const uint16_t* kv_layer, int num_blocks, int n_kv_heads,
                        const int32_t* tables, int max_blocks, const int32_t* ctx_len, const int32_t* row_off, int B,
                        int T, int n_q_heads, uint16_t* out, int ldo) {
    FewArgs a = {};
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
    a.window = kBoundSlots;
    a.most = INT_MAX;
    a.out = reinterpret_cast<__half*>(out);
    a.ldo = ldo;
    return a;
}

extern "C" size_t specdec_attention_window_workspace_bytes(int B, int T, int n_q_heads, int n_kv_heads, int head_dim,
                                                           int max_blocks) {
    if (B <= 0 || T <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || max_blocks <= 0) return 0;
    return few_space(B, T, n_q_heads, n_kv_heads, head_dim, max_blocks, false).bytes +
           rows_packed_workspace(B, T, n_q_heads, head_dim, max_blocks);
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
    // past the last slot that a row could have both change nothing (and sums with them stay in 32 bits)
    window = std::min(window, kBoundSlots);
    sinks = std::min(sinks, 16 * max_blocks);
    char* rest = static_cast<char*>(workspace);
    int least = 0;
    if (few_rows(B, T, n_q_heads / n_kv_heads)) {
        FewArgs f = few_args(q, ldq, kv_layer, num_blocks, n_kv_heads, tables, max_blocks, ctx_len, row_off, B, T,
                             n_q_heads, out, ldo);
        f.window = window;
        f.sinks = sinks;
        least = few_most(B, T, f.G);
        if (least) f.most = least;
        if ((rc = launch_few(f, head_dim, false, workspace, as_stream(stream))) || !least) return rc;
        rest += few_space(B, T, n_q_heads, n_kv_heads, head_dim, max_blocks, false).bytes;
    }
    return rows_packed_launch(reinterpret_cast<const __half*>(q), ldq, reinterpret_cast<const __half*>(kv_layer),
                              num_blocks, n_kv_heads, head_dim, tables, max_blocks, ctx_len, row_off, B, T, n_q_heads,
                              window, sinks, least, nullptr, reinterpret_cast<__half*>(out), ldo, rest, as_stream(stream));
}

extern "C" size_t specdec_attention_accumulate_workspace_bytes(int B, int T, int n_q_heads, int n_kv_heads,
                                                               int head_dim, int max_blocks) {
    if (B <= 0 || T <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || max_blocks <= 0) return 0;
    return accumulate_space(B, T, n_q_heads, n_kv_heads, head_dim, max_blocks);
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
    // (the weights of many rows read the queries again when the outputs are written)
    SD_CHECK(q != out, SPECDEC_EINVAL, "attention_accumulate: out must not be q");
    SD_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 31) == 0 &&
                 workspace_bytes >=
                     specdec_attention_accumulate_workspace_bytes(B, T, n_q_heads, n_kv_heads, head_dim, max_blocks),
             SPECDEC_EINVAL, "attention_accumulate: workspace too small or not 32-byte aligned");
    if ((rc = check_bound_memory(who, q, kv_layer, out, tables, ctx_len, row_off, workspace))) return rc;
    if ((rc = check_on_device(weights, "attention_accumulate: weights"))) return rc;
    FewArgs f = few_args(q, ldq, kv_layer, num_blocks, n_kv_heads, tables, max_blocks, ctx_len, row_off, B, T, n_q_heads,
                         out, ldo);
    f.weights = weights;
    f.ldw = ldw;
    const bool few = few_rows(B, T, n_q_heads / n_kv_heads) && few_scores(T, n_q_heads, max_blocks) <= kFewScores;
    char* rest = static_cast<char*>(workspace);
    if (few) {
        const int most = few_most(B, T, f.G);
        if (most) f.most = most;
        if ((rc = launch_few(f, head_dim, true, workspace, as_stream(stream))) || !most) return rc;
        rest += few_space(B, T, n_q_heads, n_kv_heads, head_dim, max_blocks, true).bytes;
        f.least = most;
        f.most = INT_MAX;
    }
    return launch_many(f, head_dim, rest, as_stream(stream));
}
