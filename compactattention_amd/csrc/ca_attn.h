// What the attention kernels share: vector types, the parameters of a launch, a workgroup's work item
// and small device helpers.
#pragma once

#include "ca_common.h"
#include "ca_kernels.h"

namespace ca {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef float f32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4_t;

constexpr int kNW = 8;         // waves per workgroup (32 packed query rows each)
constexpr int kBM = 32 * kNW;  // packed query rows per workgroup
constexpr float kRescale = 8.0f;      // lazy-rescale slack (log2 units)

struct AttnParams {
    Shape s;
    SeqAddr q;
    KvAddr k, v;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* counts;
    PastBlocks pb;
    float scale_log2;  // softmax scale * log2(e)
    SeqAddr out;
    float* lse;
    int ntiles;       // packed-row tiles per KV row
    int sp0;          // kPlaceSplits: splits of every request
    int rows_total;   // Lq * G
    int total_items;  // B*Hkv*ntiles*splits
    int per_xcd;      // ceil(total_items / 8)
    float* ws_o;      // [max splits][B*Hkv][rows_total][128]
    float* ws_lse;    // [max splits][B*Hkv][rows_total]  (log2 domain)
    // Ragged prefill whose row tiles fill 3/4 of the CUs: the kernel runs unsplit when every
    // row's selected count is within 1.5x of their mean (workgroup 0 records the choice
    // here for the merge); null otherwise
    int32_t* ws_unsplit;
    int32_t qpos0[CA_MAX_BATCH];     // absolute position of each request's query row 0
    int32_t nkb[CA_MAX_BATCH];       // valid logical blocks of each request
    int32_t sp[CA_MAX_BATCH];        // splits of each request's block lists
    int32_t ioff[CA_MAX_BATCH + 1];  // first work item of each request (linear placement)
    int placement;                   // kPlace*: where a workgroup finds its unit
    int units;                       // kPlaceSplits: units in all
    int unit_splits;                 // kPlaceRows, kPlaceTable: the splits of every unit, 0 when they differ
    int32_t xoff[9];                 // kPlaceTable
    uint32_t unit[kPlanRows];
    int window, sinks;               // the window kernels: tokens (WindowList)
};

// The blocks that a tile of queries at positions first .. last sees under a window: a query at p sees key j <= p
// where p - j < window or j < sinks.  Entries [0, full) are the blocks that every query of the tile sees whole (sinks,
// then the window's), [full, total) those where the mask cuts (the block in which the sinks end, the window's first
// blocks, the queries' own), so that the loops run their unmasked part first and masked blocks after it: the order of
// blocks is free in an online softmax.  All from six values, without a list in memory.
struct WindowList {
    int s1, c1;          // sinks: blocks [0, s1) whole, [s1, c1) in part
    int d0, b0, b1, e1;  // the window: [d0, b0) in part, [b0, b1) whole, [b1, e1) in part
    int full, total;

    __host__ __device__ __forceinline__ WindowList(int first, int last, int window, int sinks) {
        const int lo = first - window + 1;  // the first key that the window shows to the tile
        const int out = last - window;      // the last key that it hides from some query
        const int whole = (first + 1) >> 6;  // blocks [0, whole) hold no key past the first query
        d0 = lo > 0 ? lo >> 6 : 0;
        e1 = (last >> 6) + 1;
        c1 = (sinks >> 6) + ((sinks & 63) != 0);
        c1 = c1 < d0 ? c1 : d0;  // (d0 <= whole)
        s1 = (sinks >> 6) < c1 ? sinks >> 6 : c1;
        b0 = out < 0 ? 0 : (out >> 6) + 1;  // >= d0, <= e1
        b1 = whole > b0 ? whole : b0;
        full = s1 + b1 - b0;
        total = full + (c1 - s1) + (b0 - d0) + (e1 - b1);
    }
    __host__ __device__ __forceinline__ int block(int e) const {
        int at = 0, off = 0;
        auto part = [&](int from, int to) {  // entries from `at` on stand for blocks from `from` on
            off = e >= at ? from - at : off;
            at += to - from;
        };
        part(0, s1);
        part(b0, b1);
        part(s1, c1);
        part(d0, b0);
        part(b1, e1);
        return e + off;
    }
    // whether the mask cuts in block kb of the list
    __device__ __forceinline__ bool cut(int kb) const { return kb >= s1 && (kb < b0 || kb >= b1); }
};

// The work item of a workgroup: KV row, request, split of the row's list (of p.sp[b]) and, for
// kernels with row tiles, the tile.
struct Item {
    int row, b, split, tile;
};
// Workgroup L runs on XCD L % 8 and is that XCD's (L / 8)-th; false when the XCD has no such
// item.  Where all units hold the same number of splits the unit's place is computed: equal
// requests need no table (kPlaceRows, kPlaceSplits), a ragged launch reads one entry.  The units
// of a ragged launch differ where its requests have split counts of their own (decodes, and pages
// of 4 bits) and all splits are more than kPlanRows, so that units are whole rows; those are read
// 64 at a time, one per lane, and found by a prefix sum over their items.
// Every workgroup starts with this, so its latency shows in short launches (decode, from graph
// replays: a scalar scan over the units, the prefix sum in all ragged launches, this): 5 requests
// of 254-23110 tokens, 8 / 8 heads 33.6, 34.6, 33.9 us; 4 of 460-42073, 16 / 2 heads 26.1, 26.5,
// 25.8; 7 of 136-8722, 16 / 2 heads 15.8, 14.7, 14.1.
__device__ __forceinline__ bool find_item(const AttnParams& p, int ntiles, Item* it) {
    const int x = blockIdx.x & 7;
    int k = blockIdx.x >> 3;
    const int Hkv = p.s.Hkv;
    int lo = 0, cnt = p.unit_splits;
    auto unit = [&](uint32_t word) {
        it->row = word & (kPlanRows - 1);
        it->b = (word >> kUnitReq) & (CA_MAX_BATCH - 1);
        lo = (word >> kUnitLo) & 0xffu;
        cnt = word >> kUnitCnt;
    };
    if (cnt > 0) {
        const int per = ntiles * cnt;
        int u = k;
        if (per != 1) u = k / per;  // (an integer division is a chain of about 0.1 us)
        k -= u * per;
        if (p.placement == kPlaceRows) {
            it->row = x + 8 * u;
            if (it->row >= p.s.B * Hkv) return false;
            it->b = it->row / Hkv;
        } else {
            if (p.xoff[x] + u >= p.xoff[x + 1]) return false;
            unit(p.unit[p.xoff[x] + u]);
        }
    } else if (p.placement == kPlaceTable) {
        const int lane = threadIdx.x & 63;
        const int end = p.xoff[x + 1];
        for (int base = p.xoff[x];; base += 64) {
            if (base >= end) return false;
            const uint32_t w = base + lane < end ? p.unit[base + lane] : 0u;
            int sum = ntiles * static_cast<int>(w >> kUnitCnt);  // inclusive prefix of the units' items
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int y = __shfl_up(sum, o, 64);
                if (lane >= o) sum += y;
            }
            const int total = __builtin_amdgcn_readlane(sum, 63);
            if (k < total) {
                const int u = __popcll(__ballot(sum <= k));
                unit(__builtin_amdgcn_readlane(w, u));
                if (u > 0) k -= __builtin_amdgcn_readlane(sum, u - 1);
                break;
            }
            k -= total;
        }
    } else {
        if (p.placement == kPlaceSplits) {
            cnt = 1;
            const int u = x + 8 * (k / ntiles);
            if (u >= p.units) return false;
            it->row = u / p.sp0;
            lo = u - it->row * p.sp0;
            k %= ntiles;
        } else {
            const int W = x * p.per_xcd + k;
            if (W >= p.total_items) return false;
            int b = 0;
            while (b + 1 < p.s.B && p.ioff[b + 1] <= W) ++b;
            cnt = p.sp[b];
            const int local = W - p.ioff[b];
            const int u = local / (ntiles * cnt);
            it->row = b * Hkv + u;
            k = local - u * ntiles * cnt;
        }
        it->b = it->row / Hkv;
    }
    it->tile = k;
    if (cnt != 1) it->tile = k / cnt;
    it->split = lo + k - it->tile * cnt;
    return true;
}

__device__ __forceinline__ int swap23(int m) {
    return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1);
}

__device__ __forceinline__ lds_void_t* to_lds(const uint8_t* p) {
    return (lds_void_t*)(p);
}
__device__ __forceinline__ lds_i16x4_t* to_lds_v4(const uint8_t* p) {
    return (lds_i16x4_t*)(p);
}
// max(x, x of lane ^ 32): v_permlane32_swap hands each half the other half's values, so
// the max of its two outputs is the pair's max in every lane (no LDS round trip).
__device__ __forceinline__ float xor32_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// max(x, x of lane ^ 16), the same way with v_permlane16_swap
__device__ __forceinline__ float xor16_max(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// Wave-uniform reads of tables the kernel never writes (block ids, counts, page tables) go
// through the scalar data cache: s_load waits on lgkmcnt, so they do not queue behind the
// LDS-DMA loads in flight on vmcnt.
typedef const __attribute__((address_space(4))) int32_t const_i32_t;
__device__ __forceinline__ int32_t sload(const int32_t* p) {
    return *(const_i32_t*)p;
}

// The pages of the item's first block that another request reads too (requests that share a prefix
// share its leading blocks at the same places; entries past a request's last block are not read).
__device__ __forceinline__ bool shares_pages(const AttnParams& p, const Item& it, const int32_t* page_table, int64_t pts) {
    const int hk = it.row - it.b * p.s.Hkv;
    const int e0 = it.split * ((p.nkb[it.b] + p.sp[it.b] - 1) / p.sp[it.b]);
    if (e0 >= p.nkb[it.b]) return false;
    const int o = threadIdx.x & 63;  // another request (there are at most 64)
    const bool other = o < p.s.B && o != it.b && p.nkb[o] > e0;
    const int64_t at = (int64_t)((other ? o : it.b) * p.s.Hkv + hk) * pts + e0;
    const int id = page_table[at];
    return __ballot(other && id == sload(page_table + (int64_t)it.row * pts + e0)) != 0;
}

// Fills a launch's parameters and its plan.
void attn_fill(const AttnArgs& a, const AttnTiling& tiling, AttnParams* p, SplitPlan* plan);
// Merges the partial results of a launch whose plan has more than one split.  nan_lse: a row whose
// partial sums are NaN gets NaN as its lse (else -inf).
hipError_t launch_attn_merge(const AttnParams& p, bool nan_lse, hipStream_t stream);

}  // namespace ca
