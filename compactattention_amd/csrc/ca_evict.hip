// Eviction from a cache by accumulated attention weight: which tokens of every KV row stay, and the copy of their
// keys and values, in order, into other pages.

#include "ca_attn.h"
#include "ca_kv4.h"

namespace ca {
namespace {

constexpr int kPickThreads = 1024;
constexpr int kPickWaves = kPickThreads / 64;
constexpr int kBins = 2048;

struct PickParams {
    const float* mass;
    int64_t mass_stride;
    int32_t* keep;
    int64_t keep_stride;
    int Hkv, budget, sinks, recent;
    int slices;  // longer rows: workgroups of a row
    int* ws;     // and what they leave for the next launch
    int32_t len[CA_MAX_BATCH];
};

// Order-preserving bits of a weight; NaN counts least, -0 as 0.
__device__ __forceinline__ uint32_t rank_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x != x ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}

// The weight of the last token that stays is found digit by digit (11, 11 and 10 bits), by a histogram of the values that
// agree in the digits before.
constexpr int kLevels = 3;
__device__ __forceinline__ int level_shift(int level) { return level == 0 ? 21 : level == 1 ? 10 : 0; }
__device__ __forceinline__ int level_bins(int level) { return level == 2 ? 1024 : kBins; }
__device__ __forceinline__ uint32_t level_high(int level) { return level == 0 ? 0u : level == 1 ? 0xffe00000u : 0xfffffc00u; }

// What the digits so far say: the values above them stay, and `left` of those that agree in them.
struct Found {
    uint32_t prefix;
    int left;
};

// Weights of 0 are counted a wave at a time: keys of blocks that no table listed have none, and their lanes would wait for each
// other at one bin (16384 tokens, four fifths of them 0 by blocks: 25 us a value at a time, 16 so; without zeros 16 and 17).
constexpr uint32_t kZero = 0x80000000u;  // rank_bits(0)
template <int kN, typename Value, typename In>
__device__ __forceinline__ void count_values(int* hist, uint32_t prefix, int level, const Value& value, const In& in) {
    const uint32_t high = level_high(level);
    auto bin = [&](uint32_t u) { return (u >> level_shift(level)) & (level_bins(level) - 1); };
    if ((kZero & high) == prefix) {
        int zeros = 0;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const uint32_t u = value(i);
            zeros += __popcll(__ballot(in(i) && u == kZero));
            if (in(i) && u != kZero && (u & high) == prefix) atomicAdd(&hist[bin(u)], 1);
        }
        if ((threadIdx.x & 63) == 0 && zeros > 0) atomicAdd(&hist[bin(kZero)], zeros);
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const uint32_t u = value(i);
            if (in(i) && (u & high) == prefix) atomicAdd(&hist[bin(u)], 1);
        }
    }
}

// The bin that holds the left-th value from above, of the counts h0, h1 that thread i holds of bins - 1 - 2 i and the one
// below (0 past the lowest); every thread gets the result.  sums: kPickWaves ints, got: 2 ints.
__device__ __forceinline__ Found next_digit(Found f, int level, int h0, int h1, int* sums, int* got) {
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    int incl = h0 + h1;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(incl, o, 64);
        if (l >= o) incl += y;
    }
    if (l == 63) sums[w] = incl;
    __syncthreads();
    int before = incl - h0 - h1;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) before += i < w ? sums[i] : 0;
    if (before < f.left && before + h0 + h1 >= f.left) {
        const bool first = before + h0 >= f.left;
        got[0] = level_bins(level) - 1 - 2 * tid - (first ? 0 : 1);
        got[1] = f.left - (first ? before : before + h0);
    }
    __syncthreads();
    return Found{f.prefix | static_cast<uint32_t>(got[0]) << level_shift(level), got[1]};
}

// The range of a row's tokens between the sinks and the recent ones, and how many of them stay (0 where nothing is to be
// picked: the row keeps them all, or none).  The fixed tokens are written by the threads of the caller.
struct Middle {
    int from, to, need;
};
__device__ __forceinline__ Middle middle_of(const PickParams& p, int len, int32_t* keep, bool writes) {
    const int tid = threadIdx.x;
    if (len <= p.budget) {
        for (int i = tid; writes && i < p.budget; i += kPickThreads) keep[i] = i < len ? i : -1;
        return Middle{0, 0, 0};
    }
    const Middle m{p.sinks, len - p.recent, p.budget - p.sinks - p.recent};
    for (int i = tid; writes && i < p.sinks; i += kPickThreads) keep[i] = i;
    for (int i = tid; writes && i < p.recent; i += kPickThreads) keep[p.budget - p.recent + i] = m.to + i;
    return m;
}

// Rows of at most 1024 * kPer tokens: one workgroup a row, its values in registers.
template <int kPer>
__global__ __launch_bounds__(kPickThreads) void heavy_tokens_kernel(PickParams p) {
    __shared__ int hist[kBins];
    __shared__ int sums[kPickWaves], got[2];
    __shared__ int above_of[kPickWaves], equal_of[kPickWaves];
    const int row = blockIdx.x;
    int32_t* keep = p.keep + (int64_t)row * p.keep_stride;
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    const Middle m = middle_of(p, p.len[row / p.Hkv], keep, true);
    if (m.need == 0) return;
    // wave w: a sixteenth of the tokens between, in order, value i of a lane is token j0 + 64 i + l
    const float* mass = p.mass + (int64_t)row * p.mass_stride;
    const int per = ((m.to - m.from + kPickWaves - 1) / kPickWaves + 63) & ~63;
    const int j0 = min(m.to, m.from + w * per), j1 = min(m.to, j0 + per);
    uint32_t u[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) u[i] = j0 + 64 * i + l < j1 ? rank_bits(mass[j0 + 64 * i + l]) : 0u;
    Found f{0u, m.need};
#pragma unroll
    for (int level = 0; level < kLevels; ++level) {
        for (int i = tid; i < kBins; i += kPickThreads) hist[i] = 0;
        __syncthreads();
        count_values<kPer>(hist, f.prefix, level, [&](int i) { return u[i]; }, [&](int i) { return j0 + 64 * i + l < j1; });
        __syncthreads();
        const int b0 = level_bins(level) - 1 - 2 * tid;
        f = next_digit(f, level, b0 >= 1 ? hist[b0] : 0, b0 >= 1 ? hist[b0 - 1] : 0, sums, got);
    }
    int above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const bool in = j0 + 64 * i + l < j1;
        above += __popcll(__ballot(in && u[i] > f.prefix));
        equal += __popcll(__ballot(in && u[i] == f.prefix));
    }
    if (l == 0) {
        above_of[w] = above;
        equal_of[w] = equal;
    }
    __syncthreads();
    int at = p.sinks, eq = 0;  // the place of the wave's first kept token, the equal ones before it
    for (int i = 0; i < w; ++i) {
        at += above_of[i] + max(0, min(equal_of[i], f.left - eq));
        eq += equal_of[i];
    }
    const uint64_t below = (1ull << l) - 1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const bool in = j0 + 64 * i + l < j1;
        const uint64_t same = __ballot(in && u[i] == f.prefix);
        const bool stays = in && (u[i] > f.prefix || (u[i] == f.prefix && eq + __popcll(same & below) < f.left));
        const uint64_t kept = __ballot(stays);
        if (stays) keep[at + __popcll(kept & below)] = j0 + 64 * i + l;
        at += __popcll(kept);
        eq += __popcll(same);
    }
}

// Longer rows: p.slices workgroups a row, a launch a digit and one that writes.  Each workgroup counts its slice's values
// into a histogram of its own in p.ws (no sums whose order could change, nothing to clear); the next launch's workgroups
// add a row's histograms up and go on from the digit that they find.  131072 tokens of 8 rows: 4.5, 8.5, 8 and 10 us, most
// of it latency (one workgroup a row, reading the row five times, 160 us; slices of 16384 two launches' 3 us more).
struct SliceState {  // what a slice's workgroup of one launch leaves for the next one's
    uint32_t prefix;
    int left;
    int above;  // values above the last one that stays, as far as the digits tell, in the slices before
    int pad;
};
__device__ __forceinline__ int* slice_hist(const PickParams& p, int row, int level, int slice) {
    return p.ws + (((int64_t)row * kLevels + level) * p.slices + slice) * kBins;
}
__device__ __forceinline__ SliceState* slice_state(const PickParams& p, int row, int level, int slice) {
    const int64_t rows = gridDim.x / p.slices;
    return reinterpret_cast<SliceState*>(p.ws + rows * kLevels * p.slices * kBins) + (rows * (level & 1) + row) * p.slices + slice;
}
// What the first `level` digits say (level >= 1): those before the last one from the state that the last launch left, the
// last one from its histograms.  above, equal: the values above and of what was found in the slices before this one.
__device__ __forceinline__ Found found_at(const PickParams& p, int row, int slice, int level, int need, int* sums, int* got, int* above,
                                          int* equal) {
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    Found f{0u, need};
    int before = 0;
    if (level >= 2) {
        const SliceState st = *slice_state(p, row, level - 1, slice);
        f = Found{st.prefix, st.left};
        before = st.above;
    }
    const int b0 = level_bins(level - 1) - 1 - 2 * tid;
    int h0 = 0, h1 = 0, p0 = 0, p1 = 0;  // this thread's two bins over all slices, and over those before
    const int* hist = slice_hist(p, row, level - 1, 0) + max(b0 - 1, 0);
    constexpr int kAtOnce = 16;
    for (int k = 0; k < p.slices; k += kAtOnce) {
        int2 h[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) h[i] = b0 >= 1 && k + i < p.slices ? *reinterpret_cast<const int2*>(hist + (k + i) * kBins) : int2{0, 0};
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            h0 += h[i].y;
            h1 += h[i].x;
            p0 += k + i < slice ? h[i].y : 0;
            p1 += k + i < slice ? h[i].x : 0;
        }
    }
    f = next_digit(f, level - 1, h0, h1, sums, got);
    const int bin = got[0];
    int over = (b0 > bin ? p0 : 0) + (b0 - 1 > bin ? p1 : 0), same = (b0 == bin ? p0 : 0) + (b0 - 1 == bin ? p1 : 0);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        over += __shfl_xor(over, o, 64);
        same += __shfl_xor(same, o, 64);
    }
    __shared__ int overs[kPickWaves], sames[kPickWaves];
    if (l == 0) {
        overs[w] = over;
        sames[w] = same;
    }
    __syncthreads();
    *above = before;
    *equal = 0;
#pragma unroll
    for (int i = 0; i < kPickWaves; ++i) {
        *above += overs[i];
        *equal += sames[i];
    }
    return f;
}

constexpr int kSlice = 8192;                            // tokens of a slice, about
constexpr int kSliceAtOnce = kSlice / kPickThreads;  // values of a thread in flight

template <int kLevel>
__global__ __launch_bounds__(kPickThreads) void heavy_count_kernel(PickParams p) {
    __shared__ int hist[kBins];
    __shared__ int sums[kPickWaves], got[2];
    const int row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
    const int tid = threadIdx.x;
    const Middle m = middle_of(p, p.len[row / p.Hkv], nullptr, false);
    if (m.need == 0) return;
    const float* mass = p.mass + (int64_t)row * p.mass_stride;
    const int per = ((m.to - m.from + p.slices - 1) / p.slices + 63) & ~63;
    const int j0 = min(m.to, m.from + slice * per), j1 = min(m.to, j0 + per);
    float x[kSliceAtOnce];
    auto load = [&](int j) {
#pragma unroll
        for (int i = 0; i < kSliceAtOnce; ++i) x[i] = j + kPickThreads * i < j1 ? mass[j + kPickThreads * i] : 0.0f;
    };
    load(j0 + tid);  // (on their way while the histograms are added up)
    for (int i = tid; i < kBins; i += kPickThreads) hist[i] = 0;
    Found f{0u, m.need};
    if (kLevel > 0) {
        int above, equal;
        f = found_at(p, row, slice, kLevel, m.need, sums, got, &above, &equal);
        if (tid == 0) *slice_state(p, row, kLevel, slice) = SliceState{f.prefix, f.left, above, 0};
    }
    __syncthreads();
    for (int j = j0; j < j1;) {
        count_values<kSliceAtOnce>(hist, f.prefix, kLevel, [&](int i) { return rank_bits(x[i]); },
                                   [&](int i) { return j + tid + kPickThreads * i < j1; });
        j += kPickThreads * kSliceAtOnce;
        if (j < j1) load(j + tid);
    }
    __syncthreads();
    int* out = slice_hist(p, row, kLevel, slice);
    for (int i = tid; i < level_bins(kLevel); i += kPickThreads) out[i] = hist[i];
}

__global__ __launch_bounds__(kPickThreads) void heavy_write_kernel(PickParams p) {
    __shared__ int sums[kPickWaves], got[2];
    __shared__ int above_of[kPickWaves], equal_of[kPickWaves];
    const int row = blockIdx.x / p.slices, slice = blockIdx.x - row * p.slices;
    int32_t* keep = p.keep + (int64_t)row * p.keep_stride;
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    const Middle m = middle_of(p, p.len[row / p.Hkv], keep, slice == 0);
    if (m.need == 0) return;
    // wave w: a sixteenth of the slice, in order
    const float* mass = p.mass + (int64_t)row * p.mass_stride;
    const int per = ((m.to - m.from + p.slices - 1) / p.slices + 63) & ~63;
    const int s0 = min(m.to, m.from + slice * per), s1 = min(m.to, s0 + per);
    const int per_w = ((s1 - s0 + kPickWaves - 1) / kPickWaves + 63) & ~63;
    const int j0 = min(s1, s0 + w * per_w), j1 = min(s1, j0 + per_w);
    uint32_t u[kSliceAtOnce];
    auto load = [&](int j) {
#pragma unroll
        for (int i = 0; i < kSliceAtOnce; ++i) u[i] = j + 64 * i + l < j1 ? rank_bits(mass[j + 64 * i + l]) : 0u;
    };
    load(j0);
    int above_before, equal_before;
    const Found f = found_at(p, row, slice, kLevels, m.need, sums, got, &above_before, &equal_before);
    int above = 0, equal = 0;
    const bool once = per_w <= 64 * kSliceAtOnce;
    for (int j = j0; j < j1; j += 64 * kSliceAtOnce) {
        if (!once) load(j);
#pragma unroll
        for (int i = 0; i < kSliceAtOnce; ++i) {
            const bool in = j + 64 * i + l < j1;
            above += __popcll(__ballot(in && u[i] > f.prefix));
            equal += __popcll(__ballot(in && u[i] == f.prefix));
        }
    }
    if (l == 0) {
        above_of[w] = above;
        equal_of[w] = equal;
    }
    __syncthreads();
    // the place of the wave's first kept token, the equal ones before it
    int at = p.sinks + above_before + min(equal_before, f.left), eq = equal_before;
    for (int i = 0; i < w; ++i) {
        at += above_of[i] + max(0, min(equal_of[i], f.left - eq));
        eq += equal_of[i];
    }
    const uint64_t below = (1ull << l) - 1;
    for (int j = j0; j < j1; j += 64 * kSliceAtOnce) {
        if (!once) load(j);
#pragma unroll
        for (int i = 0; i < kSliceAtOnce; ++i) {
            const bool in = j + 64 * i + l < j1;
            const uint64_t same = __ballot(in && u[i] == f.prefix);
            const bool stays = in && (u[i] > f.prefix || (u[i] == f.prefix && eq + __popcll(same & below) < f.left));
            const uint64_t kept = __ballot(stays);
            if (stays) keep[at + __popcll(kept & below)] = j + 64 * i + l;
            at += __popcll(kept);
            eq += __popcll(same);
        }
    }
}

// ---------------------------------------------------------------------------------------
struct MoveParams {
    KvAddr k, v, k_dst, v_dst;
    Kv4Addr k4, v4, k4_dst, v4_dst;
    const int32_t* keep;
    int64_t keep_stride;
    const float* mass;
    int64_t mass_stride;
    float* mass_out;
    int64_t mass_out_stride;
    int Hkv, n, blocks;
    int32_t len[CA_MAX_BATCH];
};

// A workgroup copies one block of 64 tokens of a row.  Bound by memory: 128 rows of 4096 bf16 tokens (537 MB) 83 us,
// 6.5 TB/s; what is written goes past the caches (kept 110 us, as an ordinary copy; loads past them too 105).
template <bool kQ4>
__global__ __launch_bounds__(256) void move_tokens_kernel(MoveParams p) {
    __shared__ int from[64];     // position of every token's source
    __shared__ int kpage[64], vpage[64];
    const int row = blockIdx.x / p.blocks;
    const int kb = blockIdx.x - row * p.blocks;
    const int b = row / p.Hkv;
    const int hk = row - b * p.Hkv;
    const int len = p.len[b];
    const int n = min(p.n, len) - 64 * kb;  // tokens from this block on
    const int tid = threadIdx.x;
    if (tid < 64) {
        const int i = 64 * kb + tid;
        int j = 0, kp = 0, vp = 0;
        if (tid < n) {
            j = min(max(p.keep[(int64_t)row * p.keep_stride + i], 0), len - 1);
            if (kQ4) {
                kp = static_cast<int>(clamp_page(p.k4.page_table[(int64_t)row * p.k4.pts + (j >> 6)], p.k4.max_page));
                vp = static_cast<int>(clamp_page(p.v4.page_table[(int64_t)row * p.v4.pts + (j >> 6)], p.v4.max_page));
            } else {
                kp = p.k.page_table ? static_cast<int>(clamp_page(p.k.page_table[(int64_t)row * p.k.pts + (j >> 6)], p.k.max_page)) : j >> 6;
                vp = p.v.page_table ? static_cast<int>(clamp_page(p.v.page_table[(int64_t)row * p.v.pts + (j >> 6)], p.v.max_page)) : j >> 6;
            }
        }
        from[tid] = j;
        kpage[tid] = kp;
        vpage[tid] = vp;
        if (p.mass_out && i < p.n) p.mass_out[(int64_t)row * p.mass_out_stride + i] = tid < n ? p.mass[(int64_t)row * p.mass_stride + j] : 0.0f;
    }
    if (n <= 0) return;
    __syncthreads();
    if (!kQ4) {
        const int c = tid & 15;  // 16-byte chunk of a token
        // nothing is written through an id outside the pool
        auto place = [&](const KvAddr& t) {
            if (!t.page_table) return kb;
            const int id = sload(t.page_table + (int64_t)row * t.pts + kb);
            return id <= t.max_page ? id : -1;
        };
        const int kd = place(p.k_dst), vd = place(p.v_dst);
        uint16_t* ko = p.k_dst.data + b * p.k_dst.sb + hk * p.k_dst.sh + kd * p.k_dst.sblk + 8 * c;
        uint16_t* vo = p.v_dst.data + b * p.v_dst.sb + hk * p.v_dst.sh + vd * p.v_dst.sblk + 8 * c;
        const uint16_t* ki = p.k.data + b * p.k.sb + hk * p.k.sh + 8 * c;
        const uint16_t* vi = p.v.data + b * p.v.sb + hk * p.v.sh + 8 * c;
        u32x4_t x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = (tid >> 4) + 16 * i;
            if (t >= n) continue;
            const int j = from[t] & 63;
            x[i] = *reinterpret_cast<const u32x4_t*>(ki + (int64_t)kpage[t] * p.k.sblk + (int64_t)j * p.k.stok);
            y[i] = *reinterpret_cast<const u32x4_t*>(vi + (int64_t)vpage[t] * p.v.sblk + (int64_t)j * p.v.stok);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = (tid >> 4) + 16 * i;
            if (t >= n) continue;
            if (kd >= 0) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4_t*>(ko + (int64_t)t * p.k_dst.stok));
            if (vd >= 0) __builtin_nontemporal_store(y[i], reinterpret_cast<u32x4_t*>(vo + (int64_t)t * p.v_dst.stok));
        }
    } else {
        const int kd = sload(p.k4_dst.page_table + (int64_t)row * p.k4_dst.pts + kb);
        const int vd = sload(p.v4_dst.page_table + (int64_t)row * p.v4_dst.pts + kb);
        if (kd >= 0 && kd <= p.k4_dst.max_page) {
            uint8_t* to = p.k4_dst.data + kd * p.k4_dst.stride;
            // codes: a quarter of a token a thread; scale bytes: one of a token
            const int t = tid >> 2, c = tid & 3;
            if (t < n) {
                const uint8_t* page = p.k4.data + kpage[t] * p.k4.stride;
                const int j = from[t] & 63;
                *reinterpret_cast<u32x4_t*>(to + 64 * t + 16 * c) = *reinterpret_cast<const u32x4_t*>(page + 64 * j + 16 * c);
                to[k4_scale(t, c)] = page[k4_scale(j, c)];
            }
        }
        if (vd >= 0 && vd <= p.v4_dst.max_page) {
            uint8_t* to = p.v4_dst.data + vd * p.v4_dst.stride;
            const int m = tid & 15;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // 8 dims of token 4 (tid / 16) + i
                const int t = 4 * (tid >> 4) + i;
                if (t < n) {
                    const int j = from[t] & 63;
                    *reinterpret_cast<uint32_t*>(to + v4_code(t, 8 * m)) =
                        *reinterpret_cast<const uint32_t*>(p.v4.data + vpage[t] * p.v4.stride + v4_code(j, 8 * m));
                }
            }
            const int t = tid >> 2, c = tid & 3;
            if (t < n) to[v4_scale(t, c)] = p.v4.data[vpage[t] * p.v4.stride + v4_scale(from[t] & 63, c)];
        }
    }
}

}  // namespace

// Rows of up to 16384 tokens are held in one workgroup's registers, longer ones are cut into slices of about 8192, at most 32 of
// them: past 262144 tokens slices are longer, and their workgroups go through them in several loads.
static int heavy_slices(int longest) { return longest <= 16 * kPickThreads ? 1 : min((longest + kSlice - 1) / kSlice, 32); }

int64_t heavy_tokens_workspace_bytes(int rows, int longest, int budget) {
    const int slices = heavy_slices(longest);
    if (slices == 1 || longest <= budget) return 0;
    return (int64_t)rows * slices * (kLevels * kBins * (int64_t)sizeof(int) + 2 * (int64_t)sizeof(SliceState));
}

hipError_t launch_heavy_tokens(const float* mass, int64_t mass_stride, int B, int Hkv, const int32_t* len, int budget, int sinks,
                               int recent, int32_t* keep, int64_t keep_stride, void* workspace, hipStream_t stream) {
    PickParams p{mass, mass_stride, keep, keep_stride, Hkv, budget, sinks, recent, 1, static_cast<int*>(workspace), {}};
    int longest = 0;
    for (int b = 0; b < B; ++b) {
        p.len[b] = len[b];
        longest = max(longest, len[b]);
    }
    const int rows = B * Hkv;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(rows * p.slices), dim3(kPickThreads), 0, stream, p); };
    if (longest <= budget || longest <= 4 * kPickThreads) {
        launch(heavy_tokens_kernel<4>);
        return hipGetLastError();
    }
    if (longest <= 8 * kPickThreads) {
        launch(heavy_tokens_kernel<8>);
        return hipGetLastError();
    }
    p.slices = heavy_slices(longest);
    if (p.slices == 1) {
        launch(heavy_tokens_kernel<16>);
        return hipGetLastError();
    }
    launch(heavy_count_kernel<0>);
    launch(heavy_count_kernel<1>);
    launch(heavy_count_kernel<2>);
    launch(heavy_write_kernel);
    return hipGetLastError();
}

hipError_t launch_move_tokens(const MoveArgs& a, hipStream_t stream) {
    MoveParams p{};
    const bool q4 = a.k4 != nullptr;
    if (q4) {
        p.k4 = *a.k4;
        p.v4 = *a.v4;
        p.k4_dst = *a.k4_dst;
        p.v4_dst = *a.v4_dst;
    } else {
        p.k = *a.k;
        p.v = *a.v;
        p.k_dst = *a.k_dst;
        p.v_dst = *a.v_dst;
    }
    p.keep = a.keep;
    p.keep_stride = a.keep_stride;
    p.mass = a.mass;
    p.mass_stride = a.mass_stride;
    p.mass_out = a.mass_out;
    p.mass_out_stride = a.mass_out_stride;
    p.Hkv = a.Hkv;
    p.n = a.n;
    p.blocks = (a.n + 63) / 64;
    for (int b = 0; b < a.B; ++b) p.len[b] = a.len[b];
    const dim3 grid(static_cast<unsigned>((int64_t)a.B * a.Hkv * p.blocks));
    if (q4)
        hipLaunchKernelGGL(move_tokens_kernel<true>, grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(move_tokens_kernel<false>, grid, dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace ca
