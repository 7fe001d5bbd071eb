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
    int32_t len[CA_MAX_BATCH];
};

// Order-preserving bits of a weight; NaN counts least, -0 as 0.
__device__ __forceinline__ uint32_t rank_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x != x ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}

// One workgroup a row.  The weight of the last token that stays is found digit by digit (11, 11 and 10 bits), by a
// histogram of the values that agree in the digits so far; then every wave writes what it keeps of its part of the row.
__global__ __launch_bounds__(kPickThreads) void heavy_tokens_kernel(PickParams p) {
    __shared__ int hist[kBins];
    __shared__ int wave_sum[kPickWaves];
    __shared__ int found[2];
    __shared__ int above_of[kPickWaves], equal_of[kPickWaves];
    const int row = blockIdx.x;
    const int len = p.len[row / p.Hkv];
    int32_t* keep = p.keep + (int64_t)row * p.keep_stride;
    const int tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    if (len <= p.budget) {
        for (int i = tid; i < p.budget; i += kPickThreads) keep[i] = i < len ? i : -1;
        return;
    }
    const float* mass = p.mass + (int64_t)row * p.mass_stride;
    const int from = p.sinks, to = len - p.recent;
    const int need = p.budget - p.sinks - p.recent;  // of the tokens between
    for (int i = tid; i < p.sinks; i += kPickThreads) keep[i] = i;
    for (int i = tid; i < p.recent; i += kPickThreads) keep[p.budget - p.recent + i] = to + i;
    if (need == 0) return;
    uint32_t prefix = 0;  // the digits found, in place
    int left = need;      // how many of the values that agree in them stay
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bins = pass == 2 ? 1024 : 2048;
        const uint32_t high = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
        for (int i = tid; i < kBins; i += kPickThreads) hist[i] = 0;
        __syncthreads();
        for (int j = from + tid; j < to; j += kPickThreads) {
            const uint32_t u = rank_bits(mass[j]);
            if ((u & high) == prefix) atomicAdd(&hist[(u >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        // the bin that holds the left-th value from above: thread i has bins 2 i, 2 i + 1 counted from the top
        const int b0 = bins - 1 - 2 * tid;
        const int h0 = b0 >= 1 ? hist[b0] : 0, h1 = b0 >= 1 ? hist[b0 - 1] : 0;
        int incl = h0 + h1;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(incl, o, 64);
            if (l >= o) incl += y;
        }
        if (l == 63) wave_sum[w] = incl;
        __syncthreads();
        int before = incl - h0 - h1;
        for (int i = 0; i < w; ++i) before += wave_sum[i];
        if (before < left && before + h0 + h1 >= left) {
            const bool first = before + h0 >= left;
            found[0] = first ? b0 : b0 - 1;
            found[1] = left - (first ? before : before + h0);
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(found[0]) << shift;
        left = found[1];
        __syncthreads();
    }
    // wave w's part: a sixteenth of the tokens between, in order
    const int per = ((to - from + kPickWaves - 1) / kPickWaves + 63) & ~63;
    const int j0 = min(to, from + w * per), j1 = min(to, j0 + per);
    int above = 0, equal = 0;
    for (int j = j0; j < j1; j += 64) {
        const uint32_t u = j + l < j1 ? rank_bits(mass[j + l]) : 0u;
        above += __popcll(__ballot(j + l < j1 && u > prefix));
        equal += __popcll(__ballot(j + l < j1 && u == prefix));
    }
    if (l == 0) {
        above_of[w] = above;
        equal_of[w] = equal;
    }
    __syncthreads();
    int at = p.sinks, eq = 0;  // the place of the wave's first kept token, the equal ones before it
    for (int i = 0; i < w; ++i) {
        at += above_of[i] + max(0, min(equal_of[i], left - eq));
        eq += equal_of[i];
    }
    const uint64_t below = (1ull << l) - 1;
    for (int j = j0; j < j1; j += 64) {
        const bool in = j + l < j1;
        const uint32_t u = in ? rank_bits(mass[j + l]) : 0u;
        const uint64_t same = __ballot(in && u == prefix);
        const bool stays = in && (u > prefix || (u == prefix && eq + __popcll(same & below) < left));
        const uint64_t kept = __ballot(stays);
        if (stays) keep[at + __popcll(kept & below)] = j + l;
        at += __popcll(kept);
        eq += __popcll(same);
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

// A workgroup copies one block of 64 tokens of a row.
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
            if (kd >= 0) *reinterpret_cast<u32x4_t*>(ko + (int64_t)t * p.k_dst.stok) = x[i];
            if (vd >= 0) *reinterpret_cast<u32x4_t*>(vo + (int64_t)t * p.v_dst.stok) = y[i];
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

hipError_t launch_heavy_tokens(const float* mass, int64_t mass_stride, int B, int Hkv, const int32_t* len, int budget, int sinks,
                               int recent, int32_t* keep, int64_t keep_stride, hipStream_t stream) {
    PickParams p{mass, mass_stride, keep, keep_stride, Hkv, budget, sinks, recent, {}};
    for (int b = 0; b < B; ++b) p.len[b] = len[b];
    hipLaunchKernelGGL(heavy_tokens_kernel, dim3(B * Hkv), dim3(kPickThreads), 0, stream, p);
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
