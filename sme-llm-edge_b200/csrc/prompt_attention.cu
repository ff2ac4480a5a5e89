// prompt_attention.cu -- attention of packed prompt rows, and of verify rows
// whose sequences share a prefix, over paged fp16 KV (sm_100a).
//
// Both are the same work: a tile of query rows of one KV head (all G = Hq/Hkv
// query heads together, row = token * G + g, as many whole tokens as fit into
// 128 rows) against a range of one block table's slots.  A segment is
//   a sequence's packed rows, causal             (specdec_attention_prompt)
//   the same within a window and behind the first
//   tokens                                       (specdec_attention_window)
//   a group's rows against its shared pages      (specdec_attention_shared_prefix)
//   a sequence's rows against its own pages,
//   with the mask of its new rows                (specdec_attention_shared_prefix)
// An item is a KV head, one of the S pieces into which the segment's key range
// is cut, and
//   a pair   two adjacent tiles of the segment against the same keys (the
//            second may be empty),
//   a dual   one tile, its even and odd 128-key tiles apart: two chains of
//            Q.K^T, softmax and P.V at a time (short segments).
//
// Mathematics, with x = score * log2(e) / sqrt(hd): in blocks of 128 keys
//   m' = max(m, rowmax x),  P = 2^(x - m' + 7),  l = l 2^(m - m') + rowsum P,
//   O = O 2^(m - m') + P V;  out = O / l.
// m only moves when a row's maximum has grown by more than 8, so O is rarely
// rescaled.  P is rounded to fp16, as the tensor core multiplies fp16 by fp16:
// at most 2^-11 of a weight, or 2^-32 of the row's largest where that is more.
// The 7 is what takes P, up to 2^15 with the 8, near the end of fp16's range:
// without it weights below 2^-14 of the largest lost bits and those below 2^-25
// were gone, which a long context of small weights shows (131,072 of 2^-25.2
// beside one of 1: 3.4e-3 of V).  m, l, O are fp32.
//
// One persistent CTA per SM, 12 warps:
//   warps 0-3, 4-7  softmax of tile slot 0 / 1, one thread per query row
//   warp 8          MMA issuer
//   warp 9          TMA loads: the tiles' queries, 128-key tiles of K and V
//   warp 10         makes V safe: zeroes the slots behind the range's end in its
//                   last page, and replaces infinities and NaN in slots that
//                   not every row sees (0 * NaN would reach rows that do not
//                   see them)
//   warp 11         scheduler: takes items, decodes them, passes them on
// An operation is S = Q K^T, softmax, O += P V for one tile and 128 keys.  The
// operations of a CTA use tile slots 0 and 1 in turn, through all its items (a
// pair's tile t is in the slot of its operation 2j + t), and one thread issues
// their MMAs as P.V of an operation, then Q.K^T of the next on that slot: the
// tensor cores work for one slot while the softmax of the other runs.  (With an
// issuer for each slot the two interleave MMA by MMA, both softmaxes run at the
// same time and then neither: 6,900 clocks a pair of operations.)
// P overlays S in tensor memory (columns: S0 0, S1 128, O0 256, O1 256 + hd).
//
// With a window (WIN) an item's slots are numbered without the pages between the
// first tokens and the item's first row's window: what lies there is not read, and
// the rest of the kernel sees one range.  A row sees slot j of it iff
// j <= its own and (j < sinks or j > its own - window).
//
// Splits of the key range write unnormalised fp32 O with (m, l) into the
// workspace; rows_merge_kernel joins them in their order.
//
// An infinity or a NaN of V reaches every row that sees its slot, whatever the
// weight: no weight is 0 by the definition, though in fp16 (or beside a larger
// piece) it may be, and 0 times infinity would be NaN.  Rows that hold one at the
// end, or whose item warp 10 found one in, look their slots through again
// (rows_nonfinite); a piece with one carries its l negative.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace specdec {

constexpr int kRowsMaxSeqs = 1024;   // sequences of a call: the plan's tables live in shared memory
constexpr int kRowsMaxSplits = 32;   // pieces of one key range
// Up to so many segments are kept in shared memory (it holds no more beside the tiles, and their places are bytes) and
// taken longest first.  Sorted and as they come, in us: 128 x 5 rows under 8192 tokens (129 segments) 143.6 and 148.5;
// 256 single rows on 64 to 16,384 tokens 152 and 158, on 4096 tokens each 199 and 196.5.  Of 257, as they come and read
// from global memory for every item, the same calls take 158 and 200.
constexpr int kRowsSorted = 256;
constexpr int kRowsThreads = 384;
constexpr int kRowsMmaWarp = 8, kRowsLoadWarp = 9, kRowsFixWarp = 10, kRowsSchedWarp = 11;
constexpr int kRowsItems = 3;        // items known ahead in a CTA
constexpr int kBlockHalf = 2048;     // 16 tokens x 64 columns fp16, 128-byte rows, 128B swizzle
constexpr int kRowsTmemCols = 512;
constexpr float kHalfMax = 65504.0f, kHalfOver = 65520.0f;  // fp16's largest; from here on it rounds to infinity
constexpr float kRowsLag = 8.0f;     // what a row's maximum may grow by before m follows
constexpr float kRowsLift = 7.0f;    // P is 2^7 times the weight: at most 2^(8 + 7) < 65504
constexpr float kRowsUnlift = 128.0f;
// From this maximum on (in units of x) score * scale - m is not one fused
// operation: that leaves the rounding of m = score * scale in x, 32 at 2^29, and
// P would be 2^(x + 7).  Product and difference apart, the largest gives 0.  Below
// it x is off by 2^-13 at most (where 7 - m takes a bit more than m).
constexpr float kRowsHuge = 4096.0f;

enum { kModeCausal = 0, kModeAll = 1, kModeMask = 2, kModeWindow = 3 };
enum { kPair = 0, kDual = 1 };

// Where the partial results of a sequence's rows lie (rows of the partial buffers).
struct RowsMeta {
    int n_pre, base_pre, stride_pre;  // pieces of the shared prefix
    int n_own, base_own, stride_own;  // pieces of the own range; both 0: written by the main kernel
};

// x / d for 0 <= x < 2^31 by a multiplication: mul = ceil(2^(31 + s) / d), 2^s >= d.
struct RowsDiv {
    uint32_t mul, shift;
};
static RowsDiv rows_div(uint32_t d) {
    uint32_t s = 0;
    while ((1u << s) < d) ++s;
    return {(uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d), 31 + s};
}
__device__ __forceinline__ int rows_quot(int x, RowsDiv d) { return (int)(((uint64_t)(uint32_t)x * d.mul) >> d.shift); }

struct RowsArgs {
    const __half* kv;
    int num_blocks, Hkv, Hq, G, tpt;  // tpt = tokens of a 128-row tile
    const int32_t* tables;
    int max_blocks;
    const int32_t* ctx_len;
    const int32_t* row_off;  // prompt: [B + 1]; null: R rows for every sequence
    const uint64_t* mask;
    const int32_t* group_off;
    const int32_t* shared_blocks;
    int n_groups, B, T, R;
    int tq_small;  // tokens of the small query box
    int window, sinks;  // kModeWindow
    int least;          // kModeWindow: sequences of up to so many rows are left out
    float2* ml;         // kModeWindow, may be null: [T][Hq] each row's m and 2^7 / l (l is that of the lifted weights)
    RowsDiv by_item, by_hkv;  // 2 * tpt tokens of an item; KV heads
    int slots_max;  // max_blocks * 16
    __half* out;
    int ldo;
    float scale_log2;
    // workspace
    uint32_t* counter;  // null: items go round the CTAs
    int* any_parts;     // set by the plan: some rows have pieces to join
    RowsMeta* meta;
    float2* pml;
    float* po;
    int prows;  // rows of the partial buffers
    DeviceStatus* status;
};

struct RowsSeg {
    int lo, n;      // token rows
    int ctx;        // slot of the first row's token (causal, mask)
    int base, end;  // slots [base, end) are what the segment reads at most
    int tiles, kt;  // items along the rows; 128-key tiles of the longest
    int trow, mode;
};

struct RowsItem {
    int n_kt;          // 128-key tiles; -1: no more items
    int slot0, end;    // first slot (a multiple of 16); slots from `end` on are not read
    int trow, kvh;
    int tok0, i0;      // first token row; its index within the segment
    int ntok0, ntok1;  // tokens of the two tiles
    int ctx, mode, kind;
    int scan;          // slots >= scan are not seen by every row
    int prow;          // row of the partial buffers for tok0, -1: the result is final
    int pnext;         // a dual's odd tiles: so many rows behind (0: it has one tile only)
    int bad;           // warp 10 found an infinity or NaN past `scan`
};
struct RowsGap {
    int sinkp, gap;  // pages of the first tokens; of the table between them and the window
};
struct RowsWinItem : RowsItem, RowsGap {};
template <bool WIN>
using RowsItemOf = std::conditional_t<WIN, RowsWinItem, RowsItem>;

// ------------------------------------------------------------------ the plan
__device__ __forceinline__ int rows_clamp(int v, int lo, int hi) { return max(lo, min(hi, v)); }

// Segment i; off: the bounds of the sequences' rows (prompt) or of the groups.
template <bool WIN>
__device__ __forceinline__ RowsSeg rows_seg(const RowsArgs& a, int i, const int* off, const int* ctx_len,
                                            const int* group_pages, const int16_t* seq_group) {
    RowsSeg s;
    if (a.row_off) {
        s.lo = rows_clamp(off[i], 0, a.T);
        s.n = rows_clamp(off[i + 1], s.lo, a.T) - s.lo;
        if (WIN && s.n <= a.least) s.n = 0;
        s.ctx = rows_clamp(ctx_len[i], 0, 1 << 30);
        s.base = 0;
        s.end = min(s.ctx + s.n, a.slots_max);
        s.trow = i;
        s.mode = WIN ? kModeWindow : kModeCausal;
    } else if (i < a.n_groups) {
        const int b0 = rows_clamp(off[i], 0, a.B), b1 = rows_clamp(off[i + 1], b0, a.B);
        s.lo = b0 * a.R;
        s.n = (b1 - b0) * a.R;
        s.ctx = 0;
        s.base = 0;
        s.end = group_pages[i] * 16;
        s.trow = min(b0, a.B - 1);
        s.mode = kModeAll;
        if (s.end == 0) s.n = 0;
    } else {
        const int b = i - a.n_groups;
        s.lo = b * a.R;
        s.n = a.R;
        s.ctx = rows_clamp(ctx_len[b], 0, 1 << 30);
        s.base = seq_group[b] >= 0 ? group_pages[seq_group[b]] * 16 : 0;
        s.end = max(s.base, min(s.ctx + a.R, a.slots_max));
        s.trow = b;
        s.mode = kModeMask;
    }
    s.tiles = rows_quot(s.n + 2 * a.tpt - 1, a.by_item);
    s.kt = (s.end - s.base + 127) / 128;
    // of any item: the first tokens' pages, its tokens' windows and the rest of a page at each end
    if constexpr (WIN) s.kt = min(s.kt, (int)(((uint32_t)((a.sinks + 15) & ~15) + a.window + 2 * a.tpt + 30 + 127) / 128));
    return s;
}
// What of a sequence's table the item p along the rows leaves out.
__device__ __forceinline__ RowsGap rows_gap(const RowsArgs& a, const RowsSeg& s, int p) {
    const int first = s.ctx + p * 2 * a.tpt, end = min(s.end, s.ctx + min(s.n, (p + 1) * 2 * a.tpt));
    RowsGap g;
    g.sinkp = (min(a.sinks, end) + 15) >> 4;
    g.gap = max(0, (max(0, first - a.window + 1) >> 4) - g.sinkp);
    return g;
}
// 128-key tiles of the segment's item p along the rows
template <bool WIN>
__device__ __forceinline__ int rows_item_end(const RowsArgs& a, const RowsSeg& s, int p) {
    if constexpr (WIN) {
        const int end = min(s.end, s.ctx + min(s.n, (p + 1) * 2 * a.tpt));
        const RowsGap g = rows_gap(a, s, p);
        return g.gap ? max(min(end, 16 * g.sinkp), end - 16 * g.gap) : end;
    }
    return s.mode == kModeCausal ? min(s.end, s.ctx + min(s.n, (p + 1) * 2 * a.tpt)) : s.end;
}
template <bool WIN>
__device__ __forceinline__ int rows_item_kt(const RowsArgs& a, const RowsSeg& s, int p) {
    return (rows_item_end<WIN>(a, s, p) - s.base + 127) / 128;
}
// How long the pieces of a key range are, in key tiles: about `fine` where there
// are few rows (memory-bound: partial results are small), about `coarse`
// elsewhere.  A segment of many rows is cut only where one range is more than a
// CTA's share of the work (`whole`): its pieces' results cost as much as two key
// tiles each.
struct RowsCut {
    float per_fine, per_coarse;  // reciprocals
    int whole;
    int dual;  // key tiles from which a segment of one tile is worked on as duals
    int few;   // tokens of a segment of few rows
};
__device__ __forceinline__ bool rows_dual(const RowsArgs& a, const RowsSeg& s, const RowsCut& cut) {
    return s.n <= a.tpt && s.kt >= cut.dual;
}
__device__ __forceinline__ int rows_splits(const RowsArgs& a, const RowsSeg& s, const RowsCut& cut) {
    const int S = s.n <= cut.few ? (int)ceilf((float)s.kt * cut.per_fine)
                                  : (s.kt <= cut.whole ? 1 : (int)rintf((float)s.kt * cut.per_coarse));
    const int most = rows_dual(a, s, cut) ? min(kRowsMaxSplits, s.kt) / 2 : min(kRowsMaxSplits, s.kt);
    return rows_clamp(S, 1, max(1, most));
}
// Results of the segment's rows to join: 0 where the item's own is final.
__device__ __forceinline__ int rows_parts(const RowsArgs& a, const RowsSeg& s, const RowsCut& cut, int S) {
    return rows_dual(a, s, cut) ? 2 * S : (s.mode == kModeAll || S > 1 || s.base > 0 ? S : 0);
}

// False only for group bounds that overlap: what would not fit is left out.
__device__ __forceinline__ bool rows_fit(const RowsArgs& a, const RowsSeg& s, int parts, int prow) {
    return (long long)prow + (long long)s.n * parts <= a.prows;
}

struct RowsPlan {
    int pre[2 * kRowsMaxSeqs + 1];  // items before position i (without the KV heads)
    int prow[2 * kRowsMaxSeqs];     // partial rows before position i
    int group_pages[kRowsMaxSeqs];
    int16_t seq_group[kRowsMaxSeqs];  // -1: of no group
    RowsSeg segs[kRowsSorted];
    uint8_t order[kRowsSorted];   // segment at position i
    uint8_t splits[kRowsSorted];  // its pieces
    int wsum[2][32];
    float wwork[32];
    int nseg, items;
    RowsCut cut;
};

// Sums over the CTA; every thread gets them.  before_*: the sums of the threads in front.
__device__ __forceinline__ void rows_scan2(RowsPlan& p, int va, int vb, int* before_a, int* before_b, int* tot_a,
                                           int* tot_b) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    auto scan = [&](int& x, int& y) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) {
                x += u;
                y += v;
            }
        }
    };
    int xa = va, xb = vb;
    scan(xa, xb);
    __syncthreads();
    if (lane == 31) {
        p.wsum[0][w] = xa;
        p.wsum[1][w] = xb;
    }
    __syncthreads();
    int ta = lane < kRowsThreads / 32 ? p.wsum[0][lane] : 0, tb = lane < kRowsThreads / 32 ? p.wsum[1][lane] : 0;
    scan(ta, tb);
    const int ba = __shfl_sync(0xffffffffu, ta, max(0, w - 1)), bb = __shfl_sync(0xffffffffu, tb, max(0, w - 1));
    *tot_a = __shfl_sync(0xffffffffu, ta, 31);
    *tot_b = __shfl_sync(0xffffffffu, tb, 31);
    *before_a = (w ? ba : 0) + xa - va;
    *before_b = (w ? bb : 0) + xb - vb;
}

// Every CTA makes the same plan from the lengths in device memory (so a
// captured call serves other lengths); CTA 0 writes where the partials lie.  It
// is on every call's path: lengths and bounds are loaded once, together, and up
// to kRowsSorted segments stay in shared memory.  What it takes is the fetching of
// code that runs once: its loops are not unrolled.
template <bool WIN>
__device__ void rows_plan(const RowsArgs& a, RowsPlan& p) {
    const int tid = threadIdx.x;
    const int nseg = a.row_off ? a.B : a.n_groups + a.B;
    const bool small = nseg <= kRowsSorted;
    if (blockIdx.x == 0 && a.meta)  // before a barrier; a group's thread sets it behind
#pragma unroll 1
        for (int b = tid; b < a.B; b += kRowsThreads) a.meta[b].n_pre = 0;
    const int32_t* off = a.row_off ? a.row_off : a.group_off;
    const int32_t* ctx = a.ctx_len;
    if (small) {  // copies, where pre and prow will be
        const int n_off = a.row_off ? a.B + 1 : (a.n_groups ? a.n_groups + 1 : 0);
        if (tid < n_off) p.pre[tid] = off[tid];
        if (tid < a.B) p.prow[tid] = ctx[tid];
        off = p.pre;
        ctx = p.prow;
    }
    if (!a.row_off) {
        // shared pages of a group: announced, and within every member's context
#pragma unroll 1
        for (int g = tid; g < a.n_groups; g += kRowsThreads)
            p.group_pages[g] = rows_clamp(a.shared_blocks[g], 0, a.max_blocks);
        __syncthreads();
#pragma unroll 1
        for (int b = tid; b < a.B; b += kRowsThreads) {
            int lo = 0, hi = a.n_groups;  // first group whose end is past b
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (off[mid + 1] > b) hi = mid;
                else lo = mid + 1;
            }
            const int g = lo < a.n_groups && off[lo] <= b ? lo : -1;
            p.seq_group[b] = (int16_t)g;
            if (g >= 0) {
                // a group of one shares nothing worth a second pass
                const bool one = off[g + 1] - off[g] < 2;
                atomicMin(&p.group_pages[g], one ? 0 : rows_clamp(ctx[b], 0, 1 << 30) / 16);
            }
        }
    }
    __syncthreads();
    const int per = small ? 1 : (nseg + kRowsThreads - 1) / kRowsThreads;
    const int s0 = min(nseg, tid * per), s1 = min(nseg, s0 + per);
    auto seg_of = [&](int i) { return rows_seg<WIN>(a, i, off, ctx, p.group_pages, p.seq_group); };
    // total work in key tiles (in fp32: an estimate, the same in every CTA)
    float work = 0.f;
#pragma unroll 1
    for (int i = s0; i < s1; ++i) {
        const RowsSeg s = seg_of(i);
        if (s.tiles > 0) work += (float)s.tiles * 0.5f * (float)(rows_item_kt<WIN>(a, s, 0) + s.kt) * (float)a.Hkv;
        if (small) p.segs[i] = s;
    }
    work = warp_sum(work);
    if ((tid & 31) == 0) p.wwork[tid >> 5] = work;
    __syncthreads();
    work = warp_sum((tid & 31) < kRowsThreads / 32 ? p.wwork[tid & 31] : 0.f);
    if (small) {  // the longest first
        if (tid < nseg) {
            const int len = p.segs[tid].kt;
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < nseg; ++j) rank += p.segs[j].kt > len || (p.segs[j].kt == len && j < tid);
            p.order[rank] = (uint8_t)tid;
        }
        __syncthreads();
    }
    // pieces of about a quarter of a CTA's share; of half of it where they have many rows (128 x 5 rows under 8192
    // tokens: 144 us, with a third 158, with three quarters 171)
    const float mean = work / (float)gridDim.x;
    const float none = 1e-9f;  // of 2^23 key tiles at most: one piece
    RowsCut cut = {a.prows ? 1.f / fmaxf(4.f, 0.25f * mean) : none, a.prows ? 1.f / fmaxf(8.f, 0.5f * mean) : none,
                   (int)fminf(1.1f * mean, (float)(1 << 26)), a.prows ? 2 : 1 << 30, (WIN ? 16 : 64) / a.G};
    int item0 = 0, prow0 = 0, tot_items = 0, tot_prows = 0;
#pragma unroll 1
    for (int round = 0;; ++round) {
        int items = 0, prows = 0;
#pragma unroll 1
        for (int i = s0; i < s1; ++i) {
            const RowsSeg s = small ? p.segs[p.order[i]] : seg_of(i);
            const int S = rows_splits(a, s, cut);
            items += s.tiles * S;
            prows += s.n * rows_parts(a, s, cut, S);
        }
        rows_scan2(p, items, prows, &item0, &prow0, &tot_items, &tot_prows);
        if (tot_prows <= a.prows || round >= 11) break;
        // Less until the results fit.  First the duals of short ranges, whose two halves take room and need no
        // piece (all duals after three rounds), then pieces; at last one a segment, which always does.  (With duals
        // of any length kept, 250 sequences of 5 rows beside one token on 100,000 slots used the room up, and
        // that token's range was not cut at all.)
        if (round < 3) {
            cut.dual = round < 2 ? 4 * cut.dual : 1 << 30;
        } else {
            cut.per_fine = round == 10 ? none : 0.5f * cut.per_fine;
            cut.per_coarse = round == 10 ? none : 0.5f * cut.per_coarse;
        }
    }
#pragma unroll 1
    for (int i = s0; i < s1; ++i) {
        const RowsSeg s = small ? p.segs[p.order[i]] : seg_of(i);
        const int S = rows_splits(a, s, cut);
        const int parts = rows_parts(a, s, cut, S);
        p.pre[i] = item0;
        p.prow[i] = prow0;
        if (small) p.splits[i] = (uint8_t)S;
        if (blockIdx.x == 0 && a.meta) {
            if (s.mode == kModeAll) {
#pragma unroll 1
                for (int b = s.lo / a.R; b < (s.lo + s.n) / a.R; ++b) {
                    a.meta[b].n_pre = rows_fit(a, s, parts, prow0) ? parts : 0;
                    a.meta[b].base_pre = prow0 + (b * a.R - s.lo);
                    a.meta[b].stride_pre = s.n;
                }
            } else {
                RowsMeta& m = a.meta[s.trow];
                // (a sequence that is left out has rows, which are not this kernel's)
                m.n_own = (!WIN || s.n > 0) && rows_fit(a, s, parts, prow0) ? parts : 0;
                m.base_own = prow0;
                m.stride_own = s.n;
            }
        }
        item0 += s.tiles * S;
        prow0 += s.n * parts;
    }
    if (tid == 0) {
        p.pre[nseg] = tot_items;
        p.nseg = nseg;
        p.items = tot_items * a.Hkv;
        p.cut = cut;
        if (blockIdx.x == 0 && a.meta) *a.any_parts = tot_prows > 0;
    }
    __syncthreads();
}

template <bool WIN>
__device__ __forceinline__ RowsItemOf<WIN> rows_item(const RowsArgs& a, const RowsPlan& p, int idx) {
    RowsItemOf<WIN> it;
    it.n_kt = -1;
    it.bad = 0;
    if (idx < 0 || idx >= p.items) return it;
    const int r = rows_quot(idx, a.by_hkv);
    it.kvh = idx - r * a.Hkv;
    int lo = 0, hi = p.nseg;  // last position with pre <= r
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.pre[mid] <= r) lo = mid;
        else hi = mid;
    }
    const RowsSeg s = p.nseg <= kRowsSorted
                          ? p.segs[p.order[lo]]
                          : rows_seg<WIN>(a, lo, a.row_off ? a.row_off : a.group_off, a.ctx_len, p.group_pages, p.seq_group);
    const int S = p.nseg <= kRowsSorted ? p.splits[lo] : rows_splits(a, s, p.cut);
    const int local = r - p.pre[lo];
    const int along = S == 1 ? local : local / S;
    const int tile = s.tiles - 1 - along, piece = local - along * S;  // the longest first
    const int parts = rows_parts(a, s, p.cut, S);
    if (local < 0 || tile < 0 || (parts && !rows_fit(a, s, parts, p.prow[lo]))) {  // bounds that overlap: an empty item
        it.n_kt = it.ntok0 = it.ntok1 = 0;
        it.kind = kDual;
        it.pnext = 0;
        it.prow = -1;
        return it;
    }
    const int kt = rows_item_kt<WIN>(a, s, tile);
    const int k0 = S == 1 ? 0 : piece * kt / S, k1 = S == 1 ? kt : (piece + 1) * kt / S;  // S <= 32, kt < 2^24
    it.n_kt = k1 - k0;
    it.slot0 = s.base + 128 * k0;
    it.end = min(rows_item_end<WIN>(a, s, tile), s.base + 128 * k1);
    it.trow = s.trow;
    it.i0 = tile * 2 * a.tpt;
    it.tok0 = s.lo + it.i0;
    it.ntok0 = min(a.tpt, s.n - it.i0);
    it.ntok1 = rows_clamp(s.n - it.i0 - a.tpt, 0, a.tpt);
    it.ctx = s.ctx;
    it.mode = s.mode;
    it.scan = s.mode == kModeCausal ? s.ctx + it.i0 + 1 : (s.mode == kModeMask ? s.ctx : it.end);
    if constexpr (WIN) {
        const RowsGap g = rows_gap(a, s, tile);
        it.sinkp = g.sinkp;
        it.gap = g.gap;
        it.ctx -= 16 * g.gap;
        it.scan = it.ctx + it.i0 + 1;
    }
    it.kind = rows_dual(a, s, p.cut) || (it.ntok1 == 0 && it.n_kt <= 1) ? kDual : kPair;
    it.pnext = rows_dual(a, s, p.cut) ? s.n : 0;
    it.prow = parts ? p.prow[lo] + piece * (parts > S ? 2 : 1) * s.n + it.i0 : -1;
    return it;
}

// ------------------------------------------------------------------ the kernel
template <int HD>
struct RowsCfg {
    static constexpr int NH = HD / 64;                  // 64-column halves
    static constexpr int TILE = NH * 16384;             // 128 rows x HD fp16
    static constexpr int RING = HD == 128 ? 2 : 4;      // K tiles and V tiles in flight
    static constexpr int NBAR = 5 * 2 + 5 * RING + 2 * kRowsItems + 1;
    static constexpr size_t smem = 1024 + (size_t)TILE * (2 + 2 * RING) + sizeof(RowsPlan) +
                                   kRowsItems * sizeof(RowsWinItem) + NBAR * 8 + 16;
    static_assert(smem <= 232448, "shared memory of a CTA");
};

// The rows of an item without keys.
template <int HD>
__device__ void rows_zero(const RowsArgs& a, const RowsItem& it, int lane) {
    const int rows = (it.ntok0 + it.ntok1) * a.G;
    for (int r = lane; r < rows; r += 32) {
        const int t = r / a.G, head = it.kvh * a.G + r % a.G;
        if (it.prow < 0) {
            uint4* dst = reinterpret_cast<uint4*>(a.out + (size_t)(it.tok0 + t) * a.ldo + (size_t)head * HD);
            for (int e = 0; e < HD / 8; ++e) dst[e] = make_uint4(0, 0, 0, 0);
        } else {  // a piece of no weight: the merge reads no O of it
            a.pml[(size_t)(it.prow + t) * a.Hq + head] = make_float2(-INFINITY, 0.f);
            if (it.pnext) a.pml[(size_t)(it.prow + it.pnext + t) * a.Hq + head] = make_float2(-INFINITY, 0.f);
        }
    }
}

// Sets the columns of a row in which it sees an infinity or a NaN of V; `at` is
// the row's token (final) or its place in the partial buffers.  The whole warp
// goes through the slots (all: from the item's first, else those warp 10 looked
// at), a lane's columns being lane * (HD / 32) + j; only rows that are `mine` are
// written.  True where a column was.  Before it, a final row's infinities become
// kHalfMax: its finite means that the weights' rounding (2^-11) took past 65520.
template <int HD, bool WIN>
__device__ __noinline__ bool rows_nonfinite(const RowsArgs& a, const RowsItemOf<WIN>& it, bool mine, bool all, int i,
                                            uint64_t bits, int head, size_t at) {
    constexpr int W = HD / 32;  // columns of a lane
    const int lane = threadIdx.x & 31;
    const int mode = it.mode, ctx = it.ctx, end = min(it.end, it.slot0 + 128 * it.n_kt);
    const int32_t* tab = a.tables + (size_t)it.trow * a.max_blocks;
    uint32_t up[W], down[W];  // bit l of [j]: an infinity (NaN: both) in column l * W + j
#pragma unroll
    for (int j = 0; j < W; ++j) up[j] = down[j] = 0;
    const int start = all || WIN ? it.slot0 : max(it.scan, it.slot0);
#pragma unroll 1
    for (int s0 = start & ~15; s0 < end; s0 += 16) {  // a page
        int x;
        if constexpr (WIN) x = tab[(s0 >> 4) + (s0 >> 4 < it.sinkp ? 0 : it.gap)];
        else x = tab[s0 >> 4];
        const int page = x < 0 || x >= a.num_blocks ? 0 : x;
        const __half* src = a.kv + (((size_t)page * 2 + 1) * a.Hkv + it.kvh) * 16 * HD + lane * W;
        alignas(8) uint16_t v[16][W];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const __half* at_u = src + rows_clamp(u, max(0, start - s0), min(15, end - 1 - s0)) * HD;
            if constexpr (W == 4) *reinterpret_cast<uint2*>(v[u]) = *reinterpret_cast<const uint2*>(at_u);
            else *reinterpret_cast<uint32_t*>(v[u]) = *reinterpret_cast<const uint32_t*>(at_u);
        }
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < W; ++j) any |= (v[u][j] & 0x7C00) == 0x7C00;
            if (!__any_sync(0xffffffffu, any)) continue;
            const int d = s0 + rows_clamp(u, max(0, start - s0), min(15, end - 1 - s0)) - ctx;
            const bool seen = WIN ? d <= i && (d + ctx < a.sinks || d > i - a.window)
                                  : mode == kModeAll ||
                                        (mode == kModeCausal ? d <= i : d < 0 || (d < 64 && ((bits >> d) & 1ull)));
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const uint32_t y = v[u][j];  // 0x7C00 infinity, 0xFC00 its opposite, above either NaN
                const uint32_t plus = __ballot_sync(0xffffffffu, (y & 0x7FFF) > 0x7C00 || y == 0x7C00);
                const uint32_t minus = __ballot_sync(0xffffffffu, (y & 0x7FFF) > 0x7C00 || y == 0xFC00);
                if (seen) {
                    up[j] |= plus;
                    down[j] |= minus;
                }
            }
        }
    }
    bool found = false;
    if (mine && it.prow < 0) {
#pragma unroll 1
        for (int e = 0; e < HD; ++e) {
            __half* o = a.out + at * a.ldo + (size_t)head * HD + e;
            const float y = __half2float(*o);
            if (fabsf(y) == INFINITY) *o = __float2half_rn(copysignf(kHalfMax, y));
        }
    }
    if (mine) {
#pragma unroll
        for (int j = 0; j < W; ++j) {
            for (uint32_t left = up[j] | down[j]; left; left &= left - 1) {
                const int l = __ffs(left) - 1, e = l * W + j;
                const bool p = (up[j] >> l) & 1u, n = (down[j] >> l) & 1u;
                const float y = p && n ? __int_as_float(0x7FC00000) : (p ? INFINITY : -INFINITY);
                if (it.prow < 0) a.out[at * a.ldo + (size_t)head * HD + e] = __float2half_rn(y);
                else a.po[at * HD + e] = y;
                found = true;
            }
        }
    }
    __syncwarp();
    return found;
}

// Bit c = slot key0 + c of a row is seen.
template <bool WIN>
__device__ __forceinline__ void rows_seen(const RowsArgs& a, const RowsItem& it, int key0, int i, uint64_t bits,
                                          uint64_t& lo, uint64_t& hi) {
    auto below = [](int k) -> uint64_t { return k <= 0 ? 0ull : (k >= 64 ? ~0ull : (1ull << k) - 1ull); };
    const int n = it.end - key0;
    if constexpr (WIN) {
        const int p = it.ctx + i + 1 - key0, k = min(n, p), w = p - a.window, f = a.sinks - key0;
        lo = below(k) & (~below(w) | below(f));
        hi = below(k - 64) & (~below(w - 64) | below(f - 64));
    } else if (it.mode == kModeMask) {
        const int d = it.ctx - key0;  // column of the first new row
        lo = below(d);
        hi = below(d - 64);
        if (d > -64 && d < 64) lo |= d >= 0 ? bits << d : bits >> -d;
        const int e = d - 64;
        if (e > -64 && e < 64) hi |= e >= 0 ? bits << e : bits >> -e;
        lo &= below(n);
        hi &= below(n - 64);
    } else {
        const int k = it.mode == kModeCausal ? min(n, it.ctx + i + 1 - key0) : n;
        lo = below(k);
        hi = below(k - 64);
    }
}

// Two fp32 values in a register pair: one instruction works on both.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t d, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(d));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// The largest of three; NaN if one is.
__device__ __forceinline__ float rows_max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 2^x on the special-function unit (2 ulp); the result is rounded to fp16 next.
// A quarter of them by a polynomial on the FMA units instead made an 8192-token
// prompt 5% slower: that unit is 44% busy there, and the code grows.
__device__ __forceinline__ uint64_t exp2_unit2(uint64_t x) {
    float x0, x1, y0, y1;
    unpack2(x, x0, x1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"(x0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y1) : "f"(x1));
    return pack2(y0, y1);
}

// A row's O times f.
template <int HD>
__device__ __forceinline__ void rows_rescale(uint32_t t_o, float f) {
#pragma unroll 1
    for (int c0 = 0; c0 < HD; c0 += 16) {
        uint32_t ov[16];
        tc_ld_x16(t_o + c0, ov);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * f);
        tc_st_x16(t_o + c0, ov);
    }
}

// A row's scores v become (v scale - m) / scale, product and difference rounded apart.
__device__ __noinline__ void rows_subtract(uint32_t t_s, float scale, float m) {
    const float back = 1.0f / scale;
#pragma unroll 1
    for (int q = 0; q < 8; ++q) {
        uint32_t v[16];
        tc_ld_x16(t_s + 16 * q, v);
        tc_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e)
            v[e] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(v[e]), scale), m) * back);
        tc_st_x16(t_s + 16 * q, v);
    }
    tc_wait_st();
}

// The CTA's barriers, in shared memory.
template <int RING>
struct RowsBars {
    uint64_t *q_full, *q_empty;  // [2] queries of a slot landed; their last Q.K^T is done
    uint64_t* s_full;            // [2] scores landed
    uint64_t* p_full;            // [2] P written, O rescaled, V safe, O of the item before read (4 warps)
    uint64_t* o_full;            // [2] the item's last P.V is done
    uint64_t *k_full, *k_empty;  // [RING]
    uint64_t *v_raw, *v_full, *v_empty;  // [RING] V landed; is safe to multiply
    uint64_t *i_full, *i_empty;  // [kRowsItems] empty: 8 softmax warps, the MMA issuer, loads, fix
    uint64_t* i_want;            // the loads of an item are nearly out: the next is wanted
    __device__ explicit RowsBars(uint64_t* b)
        : q_full(b),
          q_empty(b + 2),
          s_full(b + 4),
          p_full(b + 6),
          o_full(b + 8),
          k_full(b + 10),
          k_empty(k_full + RING),
          v_raw(k_empty + RING),
          v_full(v_raw + RING),
          v_empty(v_full + RING),
          i_full(v_empty + RING),
          i_empty(i_full + kRowsItems),
          i_want(i_empty + kRowsItems) {}
};

// The MMA issuer.  P.V of operation i and Q.K^T of operation i + 2 on the same
// slot go out together (MMAs execute in the order of issue, so the second may
// overwrite the P that the first reads), and one commit tells of all MMAs
// before it: scores that have landed mean that the slot's P.V before them has,
// too.  The whole warp walks the operations, so that the operands are
// warp-uniform, and one lane issues.  The softmax warps answer for V and O; the
// issuer waits for P alone.  Keys behind the range's end cost Q.K^T columns that
// the softmax masks; P.V takes the pages that exist.
template <int HD, bool WIN>
__device__ __forceinline__ void rows_mma(const RowsArgs& a, RowsItemOf<WIN>* items, uint32_t tmem, uint32_t sq, uint32_t sk,
                                         uint32_t sv, uint64_t* bars, volatile int* abort_flag) {
    using C = RowsCfg<HD>;
    constexpr int NH = C::NH, RING = C::RING;
    const RowsBars<RING> bar(bars);
    const uint64_t qd0 = sw128_desc(sq), kd0 = sw128_desc(sk), vd0 = sw128_mn_desc(sv, kBlockHalf, 1024);
    const bool on = (threadIdx.x & 31) == 0;
    bool ok = true, more = true;  // no wait ran out; items may be left
    auto same = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    auto ready = [&](uint64_t* b, int parity) { return mbar_test_warp(s_addr(b), (uint32_t)parity & 1u); };
    auto wait = [&](uint64_t* b, int parity) {
        ok = ok && mbar_spin_warp(s_addr(b), (uint32_t)parity & 1u);
        return ok;
    };
    // the next Q.K^T: operation x of the n of item k, on the CTA's key tile `tile`
    int k = -1, x = 0, n = 0, tile = 0, pair = 0, np_last = 0;
    // what P.V of an operation needs to know: ring place | pages | first, last of the item on its slot | last use of V
    int rec = -1, rec_next = -1;    // of the operation in turn and of the one after; -1: none
    int begun[2] = {0, 0}, ended[2] = {0, 0};  // items whose Q.K^T began on a slot, whose P.V ended on it
    // Is the operation of the next Q.K^T known, and has its data landed?
    // block: waits for it.  False without block: not yet, or none is left.
    auto next_ready = [&](auto slot, bool block) -> bool {
        constexpr int s = decltype(slot)::value;
        while (x == n) {  // to the next item
            const int d = (k + 1) % kRowsItems, turn = (k + 1) / kRowsItems;
            if (block ? !wait(&bar.i_full[d], turn) : !ready(&bar.i_full[d], turn)) return false;
            const volatile RowsItem& it = static_cast<const RowsItem&>(items[d]);
            const int n_kt = same(it.n_kt);
            if (n_kt < 0) {
                more = false;
                return false;
            }
            pair = same(it.kind) == kPair;
            np_last = same(((it.end + 15) >> 4) - (it.slot0 >> 4)) - 8 * (n_kt - 1);
            ++k;
            x = 0;
            n = pair ? 2 * n_kt : n_kt;
            __syncwarp();
            if (on) mbar_arrive(s_addr(&bar.i_empty[d]));
        }
        if (block) return wait(&bar.k_full[tile % RING], tile / RING) && (x >= 2 || wait(&bar.q_full[s], begun[s]));
        return ready(&bar.k_full[tile % RING], tile / RING) && (x >= 2 || ready(&bar.q_full[s], begun[s]));
    };
    auto issue_qk = [&](auto slot) -> int {
        constexpr int s = decltype(slot)::value;
        const int at = tile % RING;
        const uint64_t qd = qd0 + (uint64_t)(s * (C::TILE >> 4)), kd = kd0 + (uint64_t)(at * (C::TILE >> 4));
        const bool first = x < 2, last = x + 2 >= n, last_use = !pair || (x & 1);
        const int np = x + (pair ? 2 : 1) >= n ? np_last : 8;
        const uint32_t d = tmem + s * 128, sb = s_addr(&bar.s_full[s]), qb = s_addr(&bar.q_empty[s]),
                       kb = s_addr(&bar.k_empty[at]);
        if (on) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
                tc_mma_f16_ss(d, qd + (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4),
                              kd + (uint64_t)(((kk >> 2) * 16384 + (kk & 3) * 32) >> 4), idesc_f16(128, 128),
                              kk > 0 ? 1u : 0u);
            tc_commit(sb);
            if (last) tc_commit(qb);
            if (last_use) tc_commit(kb);
        }
        __syncwarp();
        begun[s] += first;
        tile += last_use;
        ++x;
        return at | np << 4 | (int)first << 8 | (int)last << 9 | (int)last_use << 10;
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    if (next_ready(S0(), true)) {
        tc_fence_after();
        rec = issue_qk(S0());
        if (next_ready(S1(), true)) {
            tc_fence_after();
            rec_next = issue_qk(S1());
        }
    }
    int asked = (rec >= 0) + (rec_next >= 0);
    // P.V of the operation in turn and Q.K^T of the slot's next
    auto turn = [&](auto slot, int phase) {
        constexpr int s = decltype(slot)::value;
        const bool next = more && next_ready(slot, false);
        if (!wait(&bar.p_full[s], phase)) return;
        tc_fence_after();
        const int at = rec & 15, np = (rec >> 4) & 15;
        const bool first = (rec >> 8) & 1, last = (rec >> 9) & 1, last_use = (rec >> 10) & 1;
        const uint64_t vd = vd0 + (uint64_t)(at * (C::TILE >> 4));
        const uint32_t o = tmem + 256 + s * HD, pa = tmem + s * 128, ob = s_addr(&bar.o_full[s]),
                       vb = s_addr(&bar.v_empty[at]);
        auto step = [&](int i, uint32_t add) {  // the 16 keys of page i
            tc_mma_f16_ts(o, pa + i * 8, vd + (uint64_t)((i * NH * kBlockHalf) >> 4), idesc_f16_bmn(128, HD), add);
        };
        if (on) {
            if (first) step(0, 0u);
            else step(0, 1u);
            if (np == 8) {
#pragma unroll
                for (int i = 1; i < 8; ++i) step(i, 1u);
            } else {
#pragma unroll 1
                for (int i = 1; i < np; ++i) step(i, 1u);
            }
            if (last) tc_commit(ob);
        }
        __syncwarp();
        ended[s] += last;
        int made = -1;
        if (next) made = issue_qk(slot);
        if (last_use && on) tc_commit(vb);
        __syncwarp();
        if (!next && more && next_ready(slot, true)) {
            tc_fence_after();
            made = issue_qk(slot);
        }
        asked += made >= 0;
        rec = rec_next;
        rec_next = made;
    };
#pragma unroll 1
    for (int phase = 0; rec >= 0; ++phase) {
        turn(S0(), phase);
        if (!ok || rec < 0) break;
        turn(S1(), phase);
        if (!ok) break;
    }
    if (!ok && on) {
        *abort_flag = 1;
        record_timeout(a.status, 24);
    }
    // every MMA has finished with shared and tensor memory before the CTA leaves
    if (asked > 0) (void)mbar_spin_warp(s_addr(&bar.s_full[0]), (uint32_t)((asked + 1) / 2 - 1) & 1u);
    if (asked > 1) (void)mbar_spin_warp(s_addr(&bar.s_full[1]), (uint32_t)(asked / 2 - 1) & 1u);
    if (ended[0]) (void)mbar_spin_warp(s_addr(&bar.o_full[0]), (uint32_t)(ended[0] - 1) & 1u);
    if (ended[1]) (void)mbar_spin_warp(s_addr(&bar.o_full[1]), (uint32_t)(ended[1] - 1) & 1u);
    __syncwarp();
}

template <int HD, bool WIN>
__global__ void __launch_bounds__(kRowsThreads, 1)
    rows_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap qmap_small,
                          const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                          const __grid_constant__ RowsArgs a) {
    using C = RowsCfg<HD>;
    constexpr int NH = C::NH, RING = C::RING;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sQ = base;                       // [2 slots][NH][128 rows][128 B]
    unsigned char* sK = sQ + 2 * C::TILE;           // [RING][NH][128 keys][128 B]
    unsigned char* sV = sK + RING * C::TILE;        // [RING][8 pages][NH][16][128 B]
    RowsPlan& plan = *reinterpret_cast<RowsPlan*>(sV + RING * C::TILE);
    using Item = RowsItemOf<WIN>;
    Item* items = reinterpret_cast<Item*>(&plan + 1);
    uint64_t* bars = reinterpret_cast<uint64_t*>(
        (reinterpret_cast<uintptr_t>(items + kRowsItems) + 7) & ~uintptr_t(7));
    const RowsBars<C::RING> bar(bars);
    uint64_t *q_full = bar.q_full, *q_empty = bar.q_empty, *s_full = bar.s_full, *p_full = bar.p_full,
             *o_full = bar.o_full, *k_full = bar.k_full,
             *k_empty = bar.k_empty, *v_raw = bar.v_raw, *v_full = bar.v_full, *v_empty = bar.v_empty,
             *i_full = bar.i_full, *i_empty = bar.i_empty;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar.i_want + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    if constexpr (WIN) {
        if (a.least > 0) {  // nothing but sequences that are left out
            bool some = false;
            for (int b = threadIdx.x; b < a.B; b += kRowsThreads) {
                const int lo = rows_clamp(a.row_off[b], 0, a.T);
                some |= rows_clamp(a.row_off[b + 1], lo, a.T) - lo > a.least;
            }
            if (!__syncthreads_or(some)) {
                if (blockIdx.x == 0 && threadIdx.x == 0) *a.any_parts = 0;
                return;
            }
        }
    }
    pdl_trigger();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_addr(&q_full[i]), 1);
            mbar_init(s_addr(&q_empty[i]), 1);
            mbar_init(s_addr(&s_full[i]), 1);
            mbar_init(s_addr(&p_full[i]), 4);
            mbar_init(s_addr(&o_full[i]), 1);
        }
        for (int i = 0; i < RING; ++i) {
            mbar_init(s_addr(&k_full[i]), 1);
            mbar_init(s_addr(&k_empty[i]), 1);
            mbar_init(s_addr(&v_raw[i]), 1);
            mbar_init(s_addr(&v_full[i]), 1);
            mbar_init(s_addr(&v_empty[i]), 1);
        }
        for (int i = 0; i < kRowsItems; ++i) {
            mbar_init(s_addr(&i_full[i]), 1);
            mbar_init(s_addr(&i_empty[i]), 11);
        }
        mbar_init(s_addr(bar.i_want), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kRowsMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_slot)),
                     "r"(kRowsTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        tc_fence_before();
    }
    rows_plan<WIN>(a, plan);  // ends with a CTA-wide barrier
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    auto give_up = [&](int site) {  // a bounded wait ran out: every role leaves at its next wait
        if (lane == 0) {
            *abort_flag = 1;
            record_timeout(a.status, site);
        }
    };
    auto stopped = [&]() { return __any_sync(0xffffffffu, *abort_flag != 0) != 0; };
    auto wait = [&](uint64_t* bar, int parity) -> bool {
        return mbar_test_warp(s_addr(bar), (uint32_t)parity & 1u) ||
               __all_sync(0xffffffffu, mbar_wait(s_addr(bar), (uint32_t)parity & 1u)) != 0;
    };
    // the k-th item of this CTA; false: none is left, or a wait ran out
    auto next_item = [&](int k, Item& it) -> bool {
        const int d = k % kRowsItems;
        if (!wait(&i_full[d], k / kRowsItems)) {
            give_up(20);
            return false;
        }
        if (stopped()) return false;
        it = items[d];
        return it.n_kt >= 0;
    };
    auto done_item = [&](int k) {
        __syncwarp();
        if (lane == 0) mbar_arrive(s_addr(&i_empty[k % kRowsItems]));
    };

    if (warp < kRowsMmaWarp) {
        // ------------------------------------------------------------ softmax, one thread per query row
        const int ws = warp >> 2;                      // tile slot
        const int quarter = warp & 3;                  // TMEM lanes of this warp
        const int row = quarter * 32 + lane;
        const int ti = row / a.G, g = row % a.G;       // token of the tile, head of the group
        const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t t_s = t_lane + ws * 128, t_o = t_lane + 256 + ws * HD;
        // rows begin at 32-byte sectors: each is written by one store
        const bool sectors = WIN && ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)a.ldo * 2) & 31) == 0;
        int c = 0, ended = 0;   // operations and items done on this slot
        int op = 0, tile = 0;   // operations (on both slots) and key tiles of the items before
        bool ok = true;
        Item it;
        for (int k = 0; ok && next_item(k, it); ++k) {
            // this slot's part: a pair's tile, a dual's even (0) or odd (1) key tiles
            const int role = (op ^ ws) & 1, tile0 = tile;
            op += it.n_kt * (it.kind == kPair ? 2 : 1);
            tile += it.n_kt;
            if (it.kind == kDual && role && !it.pnext) {
                done_item(k);
                continue;
            }
            const int t = it.kind == kPair ? role : 0;
            const int j0 = it.kind == kPair ? 0 : role, jstep = it.kind == kPair ? 1 : 2;
            const bool ops = it.n_kt > j0;
            const int ntok = t ? it.ntok1 : it.ntok0;
            const int i = it.i0 + t * a.tpt + ti;      // row of the segment
            const bool real = ti < ntok;
            const bool here = quarter * 32 < ntok * a.G;  // the warp holds a real row
            const uint64_t bits = it.mode == kModeMask && real ? a.mask[i] : 0ull;
            // slots below `every` are seen by all rows of the tile
            const int every = WIN || it.mode == kModeCausal ? min(it.end, it.ctx + it.i0 + t * a.tpt + 1)
                                                            : (it.mode == kModeMask ? min(it.end, it.ctx) : it.end);
            // the last slot behind the first tokens that not every row of the tile sees
            const int far = WIN ? it.ctx + it.i0 + t * a.tpt + max(ntok, 1) - 1 - a.window : 0;
            float m = real ? -INFINITY : 0.f, l = 0.f;
            for (int j = j0; j < it.n_kt; j += jstep, ++c) {
                if (!(ok = wait(&s_full[ws], c))) break;
                tc_fence_after();
                if (here) {
                    // Two passes over the scores, 32 columns at a time with the next 32 on
                    // their way.  What counts is code that the instruction cache holds: all
                    // 128 columns unrolled, in one pass with the maximum of the tiles before,
                    // took a quarter longer for an 8192-token prompt, and masking within the
                    // first pass 3%.
                    const int key0 = it.slot0 + 128 * j;
                    const bool masked = key0 + 128 > every || (WIN && key0 <= far && key0 + 128 > a.sinks);
                    uint64_t seen_lo = ~0ull, seen_hi = ~0ull;
                    if (masked) rows_seen<WIN>(a, it, key0, i, bits, seen_lo, seen_hi);
                    float mx[2] = {-INFINITY, -INFINITY};
                    uint32_t va[32], vb[32];
                    auto largest = [&](uint32_t(&v)[32], int q) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            mx[0] = rows_max3(mx[0], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                            mx[1] = rows_max3(mx[1], __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
                        }
                    };
                    // What the row does not see: -infinity.  With a window a fifth of the tiles
                    // or more are masked: there it is done on the way through the maximum.
                    auto hide = [&](uint32_t(&v)[32], int q) {
                        const uint32_t w = (uint32_t)((q & 2 ? seen_hi : seen_lo) >> (32 * (q & 1)));
                        if (__all_sync(0xffffffffu, w == 0xFFFFFFFFu)) return;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!((w >> e) & 1u)) v[e] = 0xFF800000u;
                        tc_st_x32(t_s + 32 * q, v);
                    };
                    if (WIN && masked) {
                        tc_ld_x32(t_s, va);
                        tc_wait_ld();
#pragma unroll 1
                        for (int q = 0; q < 4; q += 2) {
                            tc_ld_x32(t_s + 32 * (q + 1), vb);
                            hide(va, q);
                            largest(va, q);
                            tc_wait_ld();
                            if (q == 0) tc_ld_x32(t_s + 64, va);
                            hide(vb, q + 1);
                            largest(vb, q + 1);
                            tc_wait_ld();
                        }
                        tc_wait_st();
                    } else if (masked) {
#pragma unroll 1
                        for (int q = 0; q < 8; ++q) {
                            const uint32_t w = (uint32_t)((q & 4 ? seen_hi : seen_lo) >> (16 * (q & 3)));
                            if (__all_sync(0xffffffffu, (w & 0xFFFFu) == 0xFFFFu)) continue;
                            uint32_t v[16];
                            tc_ld_x16(t_s + 16 * q, v);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e)
                                if (!((w >> e) & 1u)) v[e] = 0xFF800000u;
                            tc_st_x16(t_s + 16 * q, v);
                        }
                        tc_wait_st();
                    }
                    if (!(WIN && masked)) {
                        tc_ld_x32(t_s, va);
                        tc_wait_ld();
#pragma unroll 1
                        for (int q = 0; q < 4; q += 2) {
                            tc_ld_x32(t_s + 32 * (q + 1), vb);
                            largest(va, q);
                            tc_wait_ld();
                            if (q == 0) tc_ld_x32(t_s + 64, va);
                            largest(vb, q + 1);
                            tc_wait_ld();
                        }
                    }
                    tc_ld_x32(t_s, va);
                    const float top = rows_max3(mx[0], mx[1], mx[1]) * a.scale_log2;
                    const bool grow = real && !(top <= m + kRowsLag);  // also where the row had seen nothing yet, and for NaN
                    float alpha = 1.f;
                    bool huge = false;
                    if (__any_sync(0xffffffffu, grow || fabsf(m) >= kRowsHuge)) {
                        // O holds the tiles before this one (their P.V came before these scores)
                        if (grow) {
                            alpha = m == -INFINITY ? 0.f : exp2f(m - top);
                            m = top;
                        }
                        if (j != j0 && __any_sync(0xffffffffu, grow)) rows_rescale<HD>(t_o, alpha);
                        huge = __any_sync(0xffffffffu, fabsf(m) >= kRowsHuge && fabsf(m) < INFINITY);
                    }
                    // a NaN or infinite maximum makes every weight, and so the row, NaN
                    float sub = m == -INFINITY ? 0.f : (m < INFINITY ? m : __int_as_float(0x7FC00000));
                    if (huge) {
                        tc_wait_ld();
                        rows_subtract(t_s, a.scale_log2, sub);
                        tc_ld_x32(t_s, va);
                        sub = 0.f;
                    }
                    const uint64_t scale2 = pack2(a.scale_log2, a.scale_log2),
                                   lift2 = pack2(kRowsLift - sub, kRowsLift - sub);
                    uint64_t sum2[2] = {0ull, 0ull};
                    auto weights = [&](uint32_t(&v)[32], int q) {
                        uint32_t pw[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const uint64_t x =
                                fma2(pack2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), scale2, lift2);
                            const uint64_t y = exp2_unit2(x);
                            sum2[e & 1] = add2(sum2[e & 1], y);
                            float y0, y1;
                            unpack2(y, y0, y1);
                            const __half2 h = __floats2half2_rn(y0, y1);
                            pw[e] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        tc_st_x16(t_s + 16 * q, pw);  // over scores that were read
                    };
                    tc_wait_ld();
#pragma unroll 1
                    for (int q = 0; q < 4; q += 2) {
                        tc_ld_x32(t_s + 32 * (q + 1), vb);
                        weights(va, q);
                        tc_wait_ld();
                        if (q == 0) tc_ld_x32(t_s + 64, va);
                        weights(vb, q + 1);
                        tc_wait_ld();
                    }
                    float s0, s1;
                    unpack2(add2(sum2[0], sum2[1]), s0, s1);
                    l = l * alpha + (s0 + s1);
                    tc_wait_st();
                }
                if (quarter == 0) {  // V of these keys is there and safe
                    const int at = tile0 + j;
                    if (!(ok = wait(&v_full[at % RING], at / RING))) break;
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_addr(&p_full[ws]));
            }
            if (!ok) give_up(25);
            if (!ok) break;
            if (ops) {
                if (!(ok = wait(&o_full[ws], ended++))) {
                    give_up(26);
                    break;
                }
                tc_fence_after();
            }
            // ---- the item's rows: O / l, or O with (m, l) for the merge
            if (here) {
                const bool bad = ops && *reinterpret_cast<volatile int*>(&items[k % kRowsItems].bad) != 0;
                const int head = it.kvh * a.G + g, tok = it.tok0 + t * a.tpt + ti;
                const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
                const size_t prow = (size_t)(it.prow + (it.kind == kDual ? role * it.pnext : 0) + t * a.tpt + ti) * a.Hq + head;
                float far = 0.f;  // the row's largest |O|; NaN if one is
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t ov[32];
                    __syncwarp();  // rows that are not real skip the stores below
                    if (ops) {
                        tc_ld_x32(t_o + c0, ov);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = 0u;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        far = rows_max3(far, fabsf(__uint_as_float(ov[e])), fabsf(__uint_as_float(ov[e + 1])));
                    if (real && it.prow < 0) {
                        __half* dst = a.out + (size_t)tok * a.ldo + (size_t)head * HD + c0;
                        if (WIN && sectors) {
#pragma unroll
                            for (int e = 0; e < 32; e += 16) {
                                uint32_t w[8];
#pragma unroll
                                for (int q = 0; q < 8; ++q) {
                                    const __half2 h = __floats2half2_rn(__uint_as_float(ov[e + 2 * q]) * inv,
                                                                        __uint_as_float(ov[e + 2 * q + 1]) * inv);
                                    w[q] = *reinterpret_cast<const uint32_t*>(&h);
                                }
                                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + e),
                                             "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                             : "memory");
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; e += 8) {
                                uint4 w;
                                uint32_t* wp = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    const __half2 h = __floats2half2_rn(__uint_as_float(ov[e + 2 * q]) * inv,
                                                                        __uint_as_float(ov[e + 2 * q + 1]) * inv);
                                    wp[q] = *reinterpret_cast<const uint32_t*>(&h);
                                }
                                *reinterpret_cast<uint4*>(dst + e) = w;
                            }
                        }
                    } else if (real) {
                        // whole 32-byte sectors: a lane's row is far from the next lane's
                        float* dst = a.po + prow * HD + c0;
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + e),
                                         "r"(ov[e]), "r"(ov[e + 1]), "r"(ov[e + 2]), "r"(ov[e + 3]), "r"(ov[e + 4]),
                                         "r"(ov[e + 5]), "r"(ov[e + 6]), "r"(ov[e + 7])
                                         : "memory");
                    }
                }
                // (a row whose l is NaN is NaN in every column already)
                const bool spoilt = !(far < INFINITY);
                const bool mine = real && l == l && (bad || !(far * inv < kHalfOver));
                if (__any_sync(0xffffffffu, mine)) {
                    const bool all = __any_sync(0xffffffffu, mine && spoilt);
                    if (rows_nonfinite<HD, WIN>(a, items[k % kRowsItems], mine, all, i, bits, head,
                                           it.prow < 0 ? (size_t)tok : prow))
                        l = -l;
                }
                if (it.prow >= 0 && real) a.pml[prow] = make_float2(m, l);
                if constexpr (WIN)
                    if (a.ml && it.prow < 0 && real) a.ml[(size_t)tok * a.Hq + head] = make_float2(m, inv * kRowsUnlift);
            }
            tc_fence_before();  // O was read before the slot's next P is announced
            done_item(k);
        }
    } else if (warp == kRowsSchedWarp) {
        // ------------------------------------------------------------ scheduler
        // The items that it passes on have at least one operation: the MMA
        // issuer may wait for an item while operations of the one before are
        // open, which an empty one between would keep from ending.
        int next = blockIdx.x;
        for (int k = 0;; ++k) {
            const int d = k % kRowsItems;
            // An item is taken when the loads of the one before are nearly out: taken
            // earlier it would wait here while other CTAs have none left.
            if ((k && !wait(bar.i_want, k - 1)) || (k >= kRowsItems && !wait(&i_empty[d], k / kRowsItems - 1))) {
                give_up(21);
                break;
            }
            if (stopped()) break;
            int more = 0;
            for (;;) {
                int idx = next;
                if (a.counter) idx = __shfl_sync(0xffffffffu, lane == 0 ? (int)atomicAdd(a.counter, 1u) : 0, 0);
                else next += gridDim.x;
                const Item it = rows_item<WIN>(a, plan, idx);
                if (it.n_kt == 0) {  // no keys: the rows' results are zero
                    rows_zero<HD>(a, it, lane);
                    continue;
                }
                more = it.n_kt > 0;
                if (lane == 0) {
                    items[d] = it;
                    mbar_arrive(s_addr(&i_full[d]));
                }
                break;
            }
            __syncwarp();
            if (!more) break;
        }
    } else if (warp == kRowsLoadWarp) {
        // ------------------------------------------------------------ loads
        int kc = 0, vc = 0, qn[2] = {0, 0};  // K and V tiles loaded; query loads of a slot
        int op = 0;                          // operations of the items before
        bool ok = true;
        Item it;
        for (int k = 0; ok && next_item(k, it); ++k) {
            const int page0 = it.slot0 >> 4, pages = ((it.end + 15) >> 4) - page0;
            const int32_t* tab = a.tables + (size_t)it.trow * a.max_blocks + page0;
            auto page_at = [&](int i) {
                int x = 0;
                if (i < pages) {
                    if constexpr (WIN) x = tab[page0 + i < it.sinkp ? i : i + it.gap];
                    else x = tab[i];
                }
                return x < 0 || x >= a.num_blocks ? 0 : x;  // a malformed table reads block 0, never out of range
            };
            int pg = page_at(lane), pg_next = 0;  // pages of four tiles, one a lane
            int page_v = 0;                       // of V of the tile before
            // V goes one tile behind K: the place of K is free again when the scores
            // are there, that of V when P.V is, and a load that waits holds up the next
            // (64 single rows on 8k tokens: 137 us, V of a tile right behind its K 145).
            for (int j = 0; j <= it.n_kt && ok; ++j) {
                if (j < it.n_kt) {
                    if ((j & 3) == 0) {
                        if (j) pg = pg_next;
                        pg_next = page_at(8 * j + 32 + lane);
                    }
                    const int np = min(8, pages - 8 * j), slot = kc % RING, turn = kc / RING;
                    const int page = __shfl_sync(0xffffffffu, pg, 8 * (j & 3) + (lane / NH) % 8);
                    if (j == max(0, it.n_kt - 2) && lane == 0) mbar_arrive(s_addr(bar.i_want));
                    if (turn && !(ok = wait(&k_empty[slot], turn - 1))) break;
                    if (lane == 0) mbar_expect_tx(s_addr(&k_full[slot]), (uint32_t)(np * NH * kBlockHalf));
                    __syncwarp();
                    if (lane < np * NH)
                        tma_load_5d(s_addr(sK + slot * C::TILE + (lane % NH) * 16384 + (lane / NH) * kBlockHalf), &kmap, 0,
                                    it.kvh * 16, lane % NH, 0, page, s_addr(&k_full[slot]));
                    ++kc;
                }
                if (j == 0) {  // the queries, behind the first keys
                    const int loads = it.kind == kPair || it.n_kt > 1 ? 2 : 1;
                    for (int u = 0; u < loads && ok; ++u) {
                        const int qs = (op + u) & 1, t = it.kind == kPair && it.ntok1 > 0 ? u : 0;
                        if (qn[qs] && !(ok = wait(&q_empty[qs], qn[qs] - 1))) break;
                        ++qn[qs];
                        const int ntok = t ? it.ntok1 : it.ntok0;
                        const bool small = ntok <= a.tq_small;
                        const uint32_t bytes = (uint32_t)((small ? a.tq_small : a.tpt) * a.G * 128);
                        if (lane == 0) {
                            mbar_expect_tx(s_addr(&q_full[qs]), bytes * NH);
                            for (int h = 0; h < NH; ++h)
                                tma_load_4d(s_addr(sQ + qs * C::TILE + h * 16384), small ? &qmap_small : &qmap, 0, h,
                                            it.kvh * a.G, it.tok0 + t * a.tpt, s_addr(&q_full[qs]));
                        }
                        __syncwarp();
                    }
                } else {
                    const int np = min(8, pages - 8 * (j - 1)), slot = vc % RING, turn = vc / RING;
                    if (turn && !(ok = wait(&v_empty[slot], turn - 1))) break;
                    if (lane == 0) mbar_expect_tx(s_addr(&v_raw[slot]), (uint32_t)(np * NH * kBlockHalf));
                    __syncwarp();
                    if (lane < np)
                        tma_load_5d(s_addr(sV + slot * C::TILE + lane * NH * kBlockHalf), &vmap, 0, it.kvh * 16, 0, 1,
                                    page_v, s_addr(&v_raw[slot]));
                    ++vc;
                }
                page_v = __shfl_sync(0xffffffffu, pg, 8 * (j & 3) + lane % 8);
            }
            op += it.n_kt * (it.kind == kPair ? 2 : 1);
            if (!ok) give_up(22);
            if (!ok) break;
            done_item(k);
        }
        // the copies in flight land before the CTA leaves, also where another role's wait runs out after this
        for (int s = 0; s < 2; ++s)
            if (qn[s]) (void)wait(&q_full[s], qn[s] - 1);
        for (int c = max(0, kc - RING); c < kc; ++c) (void)wait(&k_full[c % RING], c / RING);
        for (int c = max(0, vc - RING); c < vc; ++c) (void)wait(&v_raw[c % RING], c / RING);
    } else if (warp == kRowsFixWarp) {
        // ------------------------------------------------------------ V made safe
        int vc = 0;
        bool ok = true;
        Item it;
        for (int k = 0; ok && next_item(k, it); ++k) {
            for (int j = 0; j < it.n_kt; ++j, ++vc) {
                const int slot = vc % RING, key0 = it.slot0 + 128 * j;
                if (!(ok = wait(&v_raw[slot], vc / RING))) break;
                unsigned char* v = sV + slot * C::TILE;
                const int n = min(128, it.end - key0);           // slots that exist
                const int np = (n + 15) >> 4;
                const int lo = rows_clamp(it.scan - key0, 0, n);  // from here not every row sees them
                bool touched = false;
                if (n < 16 * np) {
                    for (int i = n * NH * 8 + lane; i < 16 * np * NH * 8; i += 32) {
                        const int row = i / (NH * 8), h = i / 8 % NH;
                        *reinterpret_cast<uint4*>(v + ((row >> 4) * NH + h) * kBlockHalf + (row & 15) * 128 +
                                                  (i & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    touched = true;
                }
                bool found = false;
                auto place = [&](int i) {  // the i-th 16 bytes
                    const int row = i / (NH * 8), h = i / 8 % NH;
                    return reinterpret_cast<uint4*>(v + ((row >> 4) * NH + h) * kBlockHalf + (row & 15) * 128 + (i & 7) * 16);
                };
                // the top bit of a half: its exponent is all ones
                auto wild = [](uint32_t w) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; };
                auto clean = [&](uint32_t w) {
                    const uint32_t t = wild(w);
                    return w & ~((t & 0x8000u ? 0xFFFFu : 0u) | (t & 0x80000000u ? 0xFFFF0000u : 0u));
                };
                // U pieces of a lane at a time.  With a window P.V of two tiles of each item and slot waits for this warp
                // (one piece at a time took 1.5 us of a tile); without one, one at a time is the smaller code.
                constexpr int U = WIN ? 4 : 1;
                auto look = [&](int from, int to) {
                    const int i1 = to * NH * 8;
                    for (int i0 = from * NH * 8 + lane; i0 < i1; i0 += 32 * U) {
                        uint4 x[U];
#pragma unroll
                        for (int u = 0; u < U; ++u) x[u] = i0 + 32 * u < i1 ? *place(i0 + 32 * u) : make_uint4(0, 0, 0, 0);
                        uint32_t any = 0;
#pragma unroll
                        for (int u = 0; u < U; ++u) any |= wild(x[u].x) | wild(x[u].y) | wild(x[u].z) | wild(x[u].w);
                        if (any == 0) continue;
                        found = true;
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            if (i0 + 32 * u < i1)
                                *place(i0 + 32 * u) = make_uint4(clean(x[u].x), clean(x[u].y), clean(x[u].z), clean(x[u].w));
                    }
                };
                look(lo, n);
                // and between the first tokens and the last row's window
                if constexpr (WIN)
                    look(rows_clamp(a.sinks - key0, 0, lo),
                         rows_clamp(it.ctx + it.i0 + it.ntok0 + it.ntok1 - key0 - a.window, 0, lo));
                found = __any_sync(0xffffffffu, found);
                if (found && lane == 0) items[k % kRowsItems].bad = 1;
                if (touched || found) fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_addr(&v_full[slot]));
            }
            if (!ok) give_up(23);
            if (!ok) break;
            done_item(k);
        }
    } else if (warp == kRowsMmaWarp) {
        rows_mma<HD, WIN>(a, items, tmem, s_addr(sQ), s_addr(sK), s_addr(sV), bars, abort_flag);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kRowsMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kRowsTmemCols));
    }
}

// A row's merge (below) where a piece holds an infinity or a NaN (its l is
// negative or NaN): they stay, whatever the piece's weight.
template <int HD>
__device__ __noinline__ void rows_merge_nonfinite(const RowsArgs& a, const RowsMeta mt, int i, int tok, int head) {
    const int n = mt.n_pre + mt.n_own;
    auto place = [&](int p) {
        const int r = p < mt.n_pre ? mt.base_pre + p * mt.stride_pre : mt.base_own + (p - mt.n_pre) * mt.stride_own;
        return (size_t)min(r + i, a.prows - 1) * a.Hq + head;
    };
    float top = -INFINITY, l = 0.f;
    for (int p = 0; p < n; ++p) top = fmaxf(top, a.pml[place(p)].x);
    const float sub = top == -INFINITY ? 0.f : top;
    for (int p = 0; p < n; ++p) {
        const float2 ml = a.pml[place(p)];
        l += exp2f(ml.x - sub) * fabsf(ml.y);
    }
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    if (a.ml && (threadIdx.x & 7) == 0) a.ml[(size_t)tok * a.Hq + head] = make_float2(top, inv * kRowsUnlift);
    for (int e = threadIdx.x & 7; e < HD; e += 8) {
        float sum = 0.f, bad = 0.f;
        for (int p = 0; p < n; ++p) {
            const float2 ml = a.pml[place(p)];
            if (ml.x == -INFINITY) continue;  // no key of the piece is seen
            const float y = a.po[place(p) * HD + e];
            if (isfinite(y)) sum += exp2f(ml.x - sub) * y;
            else bad += y;
        }
        float y = sum * inv;
        if (fabsf(y) > kHalfMax) y = copysignf(kHalfMax, y);
        a.out[(size_t)tok * a.ldo + (size_t)head * HD + e] = __float2half_rn(l == l && bad != 0.f ? bad : y);
    }
}

// out = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p over a row's pieces, in
// their order, M being the largest so far.  Bound by L2 and by latency (where the
// pieces lie, then their results: two loads that wait for one another).  Eight
// lanes per token row and head; (m, l) and O of four pieces are in flight
// together, O too before its weight is known.  Against a warp for each row, that
// first shares out all weights: 128 x 5 rows under 8192 tokens 171 -> 162 us a
// call, 16 x 21 under 2048 61 -> 57; two or eight pieces at a time, or 16 lanes a
// row, gain in one case what they lose in another.  The CTAs go round the rows:
// one for every few rows cost 12 us where no row has pieces.
template <int HD>
__device__ __forceinline__ void rows_merge_row(const RowsArgs& a, int tok, int head) {
    constexpr int K = HD / 32, P = 4;  // 16-byte pieces of a lane's columns; pieces at a time
    const int lane = threadIdx.x & 7;
    int b, i;
    if (a.row_off) {
        int lo = 0, hi = a.B;  // first sequence whose end is past tok
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.row_off[mid + 1] > tok) hi = mid;
            else lo = mid + 1;
        }
        b = lo;
        if (b >= a.B) return;
        i = tok - max(0, a.row_off[b]);
        if (i < 0) return;
    } else {
        b = tok / a.R;
        i = tok - b * a.R;
    }
    const RowsMeta mt = a.meta[b];
    const int n = mt.n_pre + mt.n_own;
    if (n == 0) return;
    float M = -INFINITY, l = 0.f;
    bool bad = false;
    float o[K][4];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][e] = 0.f;
#pragma unroll 1
    for (int p0 = 0; p0 < n; p0 += P) {
        float2 ml[P];
        float4 v[P][K];
#pragma unroll
        for (int u = 0; u < P; ++u) {
            const int p = min(p0 + u, n - 1);
            const int r = p < mt.n_pre ? mt.base_pre + p * mt.stride_pre : mt.base_own + (p - mt.n_pre) * mt.stride_own;
            const size_t at = (size_t)min(r + i, a.prows - 1) * a.Hq + head;  // bounds that overlap: never out of range
            ml[u] = a.pml[at];
            if (p0 + u >= n) ml[u] = make_float2(-INFINITY, 0.f);
            bad |= !(ml[u].y >= 0.f);
            const float4* src = reinterpret_cast<const float4*>(a.po + at * HD) + lane;
#pragma unroll
            for (int k = 0; k < K; ++k) v[u][k] = src[8 * k];
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < P; ++u) top = fmaxf(top, ml[u].x);
        const float sub = top == -INFINITY ? 0.f : top;
        const float f = exp2f(M - sub);
        M = top;
        l *= f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[k][e] *= f;
#pragma unroll
        for (int u = 0; u < P; ++u) {
            const float w = exp2f(ml[u].x - sub);
            if (w == 0.f) continue;  // a piece without keys may hold anything
            l += w * ml[u].y;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                o[k][0] += w * v[u][k].x;
                o[k][1] += w * v[u][k].y;
                o[k][2] += w * v[u][k].z;
                o[k][3] += w * v[u][k].w;
            }
        }
    }
    if (bad) {
        rows_merge_nonfinite<HD>(a, mt, i, tok, head);
        return;
    }
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    if (a.ml && lane == 0) a.ml[(size_t)tok * a.Hq + head] = make_float2(M, inv * kRowsUnlift);
    __half* dst = a.out + (size_t)tok * a.ldo + (size_t)head * HD + 4 * lane;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        alignas(8) __half h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = __float2half_rn(fminf(fmaxf(o[k][e] * inv, -kHalfMax), kHalfMax));
        *reinterpret_cast<uint2*>(dst + 32 * k) = *reinterpret_cast<const uint2*>(h);
    }
}

template <int HD>
__global__ void __launch_bounds__(256) rows_merge_kernel(const __grid_constant__ RowsArgs a) {
    if (a.ml) pdl_trigger();  // what weighs the slots may load its first keys
    pdl_wait();
    if (*a.any_parts == 0) return;
    const int rows = a.T * a.Hq;
    for (int r = blockIdx.x * 32 + (threadIdx.x >> 3); r < rows; r += gridDim.x * 32) {
        const int tok = r / a.Hq;
        rows_merge_row<HD>(a, tok, r - tok * a.Hq);
    }
}

// ------------------------------------------------------------------ host side
// The queries as [T][Hq][HD / 64][64]: one box is `tokens` tokens of one group
// and column half, rows token * G + g of 128 bytes.
int make_q_tmap(CUtensorMap* map, const __half* q, int ldq, int T, int Hq, int HD, int G, int tokens) {
    auto enc = attn_encode();
    SD_CHECK(enc, SPECDEC_ENOTSUP, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[4] = {64, (cuuint64_t)(HD / 64), (cuuint64_t)Hq, (cuuint64_t)T};
    cuuint64_t strides[3] = {128, (cuuint64_t)HD * 2, (cuuint64_t)ldq * 2};
    cuuint32_t box[4] = {64, 1, (cuuint32_t)G, (cuuint32_t)tokens};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<__half*>(q), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    SD_CHECK(r == CUDA_SUCCESS, SPECDEC_EINVAL, "attention: cuTensorMapEncodeTiled failed for the queries");
    return SPECDEC_OK;
}

constexpr int kRowsPartialRows = 8192;   // room for pieces, in token rows
constexpr int kRowsMoreRows = 4096;      // shared prefix: room for duals, and for pieces

// Rows of the partial buffers.
// Tables of up to 256 slots have two key tiles: no pieces, and no merge behind
// them (a single row on 40 slots: 14.9 us a call with its launch, 12.2 without).
// More rows never have less room: a workspace for a server's largest call does
// for the smaller ones (and 2800 rows of prompts beside 250 sequences of 5 rows
// and a token on 100,000 slots take 304 us, 2900 rows 314; with a quarter of the
// room from 4096 rows in all on, 343).
static size_t prompt_partial_rows(int T, int max_blocks) {
    return max_blocks <= 16 ? 0 : std::min<size_t>((size_t)kRowsMaxSplits * T, kRowsPartialRows);
}
// Under a shared prefix every row has two results to join, its own range's and
// the prefix's; what lies beyond is for duals and pieces, and limited, as it only
// makes the call faster (128 sequences of 64 rows, 32 heads of 128: 24,576 rows,
// 409 MB).  Without groups, short tables have none.
static size_t shared_partial_rows(int T, int n_groups, int max_blocks) {
    if (n_groups == 0 && max_blocks <= 16) return 0;
    const size_t t = (size_t)T, duals = std::min<size_t>(2 * t, kRowsMoreRows);
    const size_t pieces = max_blocks <= 16 ? 0 : std::min<size_t>(2 * (kRowsMaxSplits - 2) * t, kRowsMoreRows);
    return (n_groups ? 2 * t : 0) + duals + pieces;
}
static size_t align256(size_t n) { return (n + 255) & ~size_t(255); }
static size_t rows_workspace(size_t prows, int B, int Hq, int HD) {
    return 256 + align256(sizeof(RowsMeta) * (size_t)B) + align256(prows * Hq * sizeof(float2)) +
           prows * Hq * HD * sizeof(float);
}

struct DeviceFacts {
    std::atomic<int> sms{0};
};
static int rows_sms(int* out) {  // SMs of the current device; sets the kernels' shared memory on it once
    static DeviceFacts facts[64];
    int dev = 0;
    SD_CUDA(cudaGetDevice(&dev));
    SD_CHECK(dev >= 0 && dev < 64, SPECDEC_ENOTSUP, "attention: device index above 63");
    int n = facts[dev].sms.load();
    if (!n) {
        const auto room = [](const void* fn, size_t bytes) {
            return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        };
        SD_CUDA(room((const void*)rows_attention_kernel<128, false>, RowsCfg<128>::smem));
        SD_CUDA(room((const void*)rows_attention_kernel<64, false>, RowsCfg<64>::smem));
        SD_CUDA(room((const void*)rows_attention_kernel<128, true>, RowsCfg<128>::smem));
        SD_CUDA(room((const void*)rows_attention_kernel<64, true>, RowsCfg<64>::smem));
        SD_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        facts[dev].sms.store(n);
    }
    *out = n;
    return SPECDEC_OK;
}

// Fills in what both calls share and launches.  tiles: an upper bound of the
// items before splits.
static int launch_rows(RowsArgs a, const __half* q, int ldq, const __half* kv, int HD, size_t prows, long long tiles,
                       void* ws, cudaStream_t s) {
    int sms = 0;
    int rc = rows_sms(&sms);
    if (!rc) rc = check_on_device(q, "attention: q");
    if (!rc) rc = check_on_device(kv, "attention: the KV pool");
    if (!rc) rc = check_on_device(a.out, "attention: out");
    if (!rc) rc = check_on_device(ws, "attention: the workspace");
    if (!rc) rc = check_on_device(a.tables, "attention: tables");
    if (!rc) rc = check_on_device(a.ctx_len, "attention: ctx_len");
    if (!rc && a.row_off) rc = check_on_device(a.row_off, "attention: row_off");
    if (!rc && a.mask) rc = check_on_device(a.mask, "attention: mask", sizeof(uint64_t));
    if (!rc && a.n_groups) rc = check_on_device(a.group_off, "attention: group_off");
    if (!rc && a.n_groups) rc = check_on_device(a.shared_blocks, "attention: shared_blocks");
    if (rc) return rc;
    a.G = a.Hq / a.Hkv;
    a.tpt = 128 / a.G;
    a.tq_small = std::min(a.tq_small, a.tpt);
    a.by_item = rows_div(2 * a.tpt);
    a.by_hkv = rows_div(a.Hkv);
    a.kv = kv;
    a.slots_max = a.max_blocks * 16;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)HD));
    a.status = device_status_ptr();
    a.prows = (int)prows;
    char* w = static_cast<char*>(ws);
    // more items than CTAs: they are taken from a counter, the longest first
    a.counter = tiles > sms ? reinterpret_cast<uint32_t*>(w) : nullptr;
    a.any_parts = reinterpret_cast<int*>(w + 128);
    a.meta = prows ? reinterpret_cast<RowsMeta*>(w + 256) : nullptr;
    w += 256 + align256(sizeof(RowsMeta) * (size_t)a.B);
    a.pml = reinterpret_cast<float2*>(w);
    a.po = reinterpret_cast<float*>(w + align256(prows * a.Hq * sizeof(float2)));
    CUtensorMap qmap, qsmall, kmap, vmap;
    rc = make_q_tmap(&qmap, q, ldq, a.T, a.Hq, HD, a.G, a.tpt);
    if (!rc) rc = make_q_tmap(&qsmall, q, ldq, a.T, a.Hq, HD, a.G, a.tq_small);
    if (!rc) rc = make_kv_tmap(&kmap, kv, a.num_blocks, a.Hkv, HD, 1, 1);
    if (!rc) rc = make_kv_tmap(&vmap, kv, a.num_blocks, a.Hkv, HD, HD / 64, 1);
    if (rc) return rc;
    if (a.counter) SD_CUDA(cudaMemsetAsync(a.counter, 0, sizeof(uint32_t), s));
    const unsigned grid = (unsigned)(prows ? sms : std::min<long long>(sms, tiles));
    const auto fn = HD == 128 ? (a.window ? rows_attention_kernel<128, true> : rows_attention_kernel<128, false>)
                              : (a.window ? rows_attention_kernel<64, true> : rows_attention_kernel<64, false>);
    fn<<<grid, kRowsThreads, HD == 128 ? RowsCfg<128>::smem : RowsCfg<64>::smem, s>>>(qmap, qsmall, kmap, vmap, a);
    SD_LAUNCH_CHECK("rows_attention_kernel");
    if (prows) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)std::min<long long>(((long long)a.T * a.Hq + 31) / 32, 8LL * sms));
        cfg.blockDim = dim3(256);
        cfg.stream = s;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        if (HD == 128) SD_CUDA(cudaLaunchKernelEx(&cfg, rows_merge_kernel<128>, a));
        else SD_CUDA(cudaLaunchKernelEx(&cfg, rows_merge_kernel<64>, a));
    }
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
    SD_CHECK(B >= 0 && B <= kRowsMaxSeqs, SPECDEC_EINVAL, w + ": 0 to 1024 sequences");
    SD_CHECK(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv) | reinterpret_cast<uintptr_t>(out)) &
              15) == 0,
             SPECDEC_EINVAL, w + ": q, KV pool and out must be 16-byte aligned");
    return SPECDEC_OK;
}
static int check_workspace(const char* who, const void* ws, size_t have, size_t need) {
    SD_CHECK(ws && have >= need && (reinterpret_cast<uintptr_t>(ws) & 31) == 0, SPECDEC_EINVAL,
             std::string(who) + ": workspace too small or not 32-byte aligned");
    return SPECDEC_OK;
}

// Packed rows within a window (window > 0) and behind the first tokens, or causal (0).
size_t rows_packed_workspace(int B, int T, int Hq, int HD, int max_blocks) {
    return rows_workspace(prompt_partial_rows(T, max_blocks), B, Hq, HD);
}
int rows_packed_launch(const __half* q, int ldq, const __half* kv, int num_blocks, int Hkv, int HD, const int32_t* tables,
                       int max_blocks, const int32_t* ctx_len, const int32_t* row_off, int B, int T, int Hq, int window,
                       int sinks, int least, float2* ml, __half* out, int ldo, void* ws, cudaStream_t s) {
    size_t prows = prompt_partial_rows(T, max_blocks);
    if ((long long)T * Hq >= 1 << 30) prows = 0;  // the merge counts rows and heads in 32 bits
    RowsArgs a = {};
    a.num_blocks = num_blocks;
    a.Hkv = Hkv;
    a.Hq = Hq;
    a.tables = tables;
    a.max_blocks = max_blocks;
    a.ctx_len = ctx_len;
    a.row_off = row_off;
    a.B = B;
    a.T = T;
    a.R = 1;
    a.tq_small = 1;
    a.window = window;
    a.sinks = sinks;
    a.least = least;
    a.ml = ml;
    a.out = out;
    a.ldo = ldo;
    const int tpt2 = 2 * (128 / (Hq / Hkv));
    return launch_rows(a, q, ldq, kv, HD, prows, (long long)Hkv * ((T + tpt2 - 1) / tpt2 + std::min(B, T)), ws, s);
}

}  // namespace specdec

using namespace specdec;

extern "C" size_t specdec_attention_prompt_workspace_bytes(int B, int T, int n_q_heads, int n_kv_heads, int head_dim,
                                                           int max_blocks) {
    (void)n_kv_heads;
    if (B <= 0 || T <= 0 || n_q_heads <= 0 || head_dim <= 0) return 0;
    return rows_packed_workspace(B, T, n_q_heads, head_dim, max_blocks);
}

extern "C" int specdec_attention_prompt(const uint16_t* q, int ldq, const uint16_t* kv_layer, int num_blocks,
                                        int n_kv_heads, int head_dim, const int32_t* tables, int max_blocks,
                                        const int32_t* ctx_len, const int32_t* row_off, int B, int T, int n_q_heads,
                                        uint16_t* out, int ldo, void* workspace, size_t workspace_bytes, void* stream) {
    // (an empty call's tensors may have no memory)
    SD_CHECK(B == 0 || T == 0 || (q && kv_layer && tables && ctx_len && row_off && out), SPECDEC_EINVAL,
             "attention_prompt: null argument");
    int rc = check_rows("attention_prompt", q, kv_layer, out, num_blocks, n_kv_heads, head_dim, max_blocks, B,
                        n_q_heads);
    if (rc) return rc;
    SD_CHECK(T >= 0 && T <= (1 << 24), SPECDEC_EINVAL, "attention_prompt: 0 to 2^24 rows");
    SD_CHECK(ldq >= n_q_heads * head_dim && ldq % 8 == 0 && ldo >= n_q_heads * head_dim && ldo % 8 == 0,
             SPECDEC_EINVAL, "attention_prompt: row strides hold all heads and are multiples of 8");
    if (B == 0 || T == 0) return SPECDEC_OK;
    if ((rc = check_workspace("attention_prompt", workspace, workspace_bytes,
                              rows_packed_workspace(B, T, n_q_heads, head_dim, max_blocks))))
        return rc;
    return rows_packed_launch(reinterpret_cast<const __half*>(q), ldq, reinterpret_cast<const __half*>(kv_layer),
                              num_blocks, n_kv_heads, head_dim, tables, max_blocks, ctx_len, row_off, B, T, n_q_heads, 0,
                              0, 0, nullptr, reinterpret_cast<__half*>(out), ldo, workspace, as_stream(stream));
}

extern "C" size_t specdec_attention_shared_prefix_workspace_bytes(int B, int R, int n_groups, int n_q_heads,
                                                                  int n_kv_heads, int head_dim, int max_blocks) {
    (void)n_kv_heads;
    if (B <= 0 || R <= 0 || B > kRowsMaxSeqs || R > 64 || n_q_heads <= 0 || head_dim <= 0) return 0;
    return rows_workspace(shared_partial_rows(B * R, n_groups, max_blocks), B, n_q_heads, head_dim);
}

extern "C" int specdec_attention_shared_prefix(const uint16_t* q, const uint16_t* kv_layer, int num_blocks,
                                               int n_kv_heads, int head_dim, const int32_t* tables, int max_blocks,
                                               const int32_t* ctx_len, const uint64_t* mask, const int32_t* group_off,
                                               const int32_t* shared_blocks, int n_groups, int B, int R, int n_q_heads,
                                               uint16_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    SD_CHECK(B == 0 || (q && kv_layer && tables && ctx_len && mask && out &&
                        (n_groups == 0 || (group_off && shared_blocks))),
             SPECDEC_EINVAL, "attention_shared_prefix: null argument");
    int rc = check_rows("attention_shared_prefix", q, kv_layer, out, num_blocks, n_kv_heads, head_dim, max_blocks, B,
                        n_q_heads);
    if (rc) return rc;
    SD_CHECK(R >= 1 && R <= 64, SPECDEC_EINVAL, "attention_shared_prefix: 1 to 64 rows");
    SD_CHECK(n_groups >= 0 && n_groups <= B, SPECDEC_EINVAL, "attention_shared_prefix: 0 to B groups");
    if (B == 0) return SPECDEC_OK;
    const size_t prows = shared_partial_rows(B * R, n_groups, max_blocks);
    if ((rc = check_workspace("attention_shared_prefix", workspace, workspace_bytes,
                              rows_workspace(prows, B, n_q_heads, head_dim))))
        return rc;
    RowsArgs a = {};
    a.num_blocks = num_blocks;
    a.Hkv = n_kv_heads;
    a.Hq = n_q_heads;
    a.tables = tables;
    a.max_blocks = max_blocks;
    a.ctx_len = ctx_len;
    a.mask = mask;
    a.group_off = group_off;
    a.shared_blocks = shared_blocks;
    a.n_groups = n_groups;
    a.B = B;
    a.T = B * R;
    a.R = R;
    a.tq_small = R;
    a.out = reinterpret_cast<__half*>(out);
    a.ldo = n_q_heads * head_dim;
    const int tpt2 = 2 * (128 / (n_q_heads / n_kv_heads));
    const long long tiles = (long long)n_kv_heads * ((a.T + tpt2 - 1) / tpt2 + n_groups + (long long)B * ((R + tpt2 - 1) / tpt2));
    return launch_rows(a, reinterpret_cast<const __half*>(q), a.ldo, reinterpret_cast<const __half*>(kv_layer),
                       head_dim, prows, tiles, workspace, as_stream(stream));
}
