// The attention weight that every cached key received: out[row][j] = mass[row][j] + the sum over the queries and the
// query heads of the row's group that see key j of exp(q . k_j * scale - lse).
//
// The scores are S^T = K Q^T (32x32x16 bf16 MFMAs, fp32), so a lane holds 16 keys of one query row, and the sum over
// query rows stays in the lane until the end: one fma, exp2 and add a score, and no atomics.  A wave keeps the 64 keys of
// one block in registers and goes through the packed query rows r = t * G + g, 32 at a time; K is read once.
// kParts waves of a workgroup share a block, each with every kParts-th tile of rows, and join in LDS in a fixed order, so
// results do not depend on what runs when.

#include <type_traits>

#include "ca_attn.h"
#include "ca_kv4.h"

namespace ca {
namespace {

constexpr int kMassWaves = 8;

struct MassParams {
    Shape s;
    SeqAddr q;
    KvAddr k;
    Kv4Addr k4;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* counts;
    const float* lse;
    int64_t lse_sb, lse_sh;
    const float* mass;
    int64_t mass_stride;
    float* out;
    int64_t out_stride;
    float scale_log2;
    int window, sinks;
    int items;  // workgroups of a row
    int32_t start[CA_MAX_BATCH];
};

// kQ4: keys held in 4 bits.  kTab: the blocks of per-row lists, else all of them.
template <bool kQ4, bool kTab, int kParts>
__global__ __launch_bounds__(kMassWaves * 64) __attribute__((amdgpu_waves_per_eu(2))) void key_mass_kernel(MassParams p) {
    constexpr int kBlocks = kMassWaves / kParts;  // of a workgroup
    __shared__ float part[kMassWaves][64];
    const Shape& s = p.s;
    const int rows = s.B * s.Hkv;
    // a row's workgroups on one XCD, whose L2 then holds its queries once
    int row, item;
    if (rows % 8 == 0) {
        const int k = blockIdx.x >> 3;
        const int u = k / p.items;
        row = (blockIdx.x & 7) + 8 * u;
        item = k - u * p.items;
    } else {
        row = blockIdx.x / p.items;
        item = blockIdx.x - row * p.items;
    }
    const int b = row / s.Hkv;
    const int hk = row - b * s.Hkv;
    const int G = s.G;
    const int R = s.Lq * G;
    const int start = p.start[b];
    const int tokens = start + s.Lq;
    const int nkb = (tokens + 63) >> 6;
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l = tid & 63;
    const int n = l & 31;
    const int h = l >> 5;
    const int32_t* tab = kTab ? p.table + (int64_t)row * p.table_stride : nullptr;
    const int count = kTab ? min(max(sload(p.counts + row), 0), min(s.cap, nkb)) : nkb;
    const float* mass = p.mass + (int64_t)row * p.mass_stride;
    float* out = p.out + (int64_t)row * p.out_stride;
    const int e = item * kBlocks + w / kParts;
    const int sub = w % kParts;
    const bool here = e < count;
    const int kb = !here ? 0 : kTab ? min(max(sload(tab + e), 0), nkb - 1) : e;

    // blocks that the list leaves out keep their weights: those before an entry (after the one before it) go with the
    // entry, those after the last one with the place after it
    if (kTab && p.out != p.mass && sub == 0 && e <= count) {
        const int from = e == 0 ? 0 : min(max(sload(tab + e - 1), 0), nkb - 1) + 1;
        const int to = here ? kb : nkb;
        for (int j = 64 * from + l; j < min(64 * to, tokens); j += 64) out[j] = mass[j];
    }

    float acc[2][16];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[kt][j] = 0.0f;

    if (here) {
        // ---- keys: lane (n, h) holds key 32 kt + n, of the 16 dims of step ds the eight from dim(ds) on ----
        auto dim = [&](int ds) { return kQ4 ? 32 * (2 * (ds >> 2) + h) + 8 * (ds & 3) : 16 * ds + 8 * h; };
        bf16x8_t kf[2][8];
        const int rows_here = min(64, tokens - 64 * kb);
        if (kQ4) {
            const uint8_t* page = p.k4.data + clamp_page(sload(p.k4.page_table + (int64_t)row * p.k4.pts + kb), p.k4.max_page) * p.k4.stride;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int t = 32 * kt + n, g = 2 * c + h;
                    const u32x4_t code = *reinterpret_cast<const u32x4_t*>(page + 64 * t + 16 * g);
                    const float sc = scale_of(page[k4_scale(t, g)], 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const u32x4_t x = {decode2<0>(code[i], sc), decode2<1>(code[i], sc), decode2<2>(code[i], sc), decode2<3>(code[i], sc)};
                        kf[kt][4 * c + i] = __builtin_bit_cast(bf16x8_t, x);
                    }
                }
        } else {
            const int64_t phys = p.k.page_table ? clamp_page(sload(p.k.page_table + (int64_t)row * p.k.pts + kb), p.k.max_page) : kb;
            const uint16_t* base = p.k.data + b * p.k.sb + hk * p.k.sh + phys * p.k.sblk;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                // (past the cache's end: its last token, whose place is written by nobody here)
                const uint16_t* kp = base + (int64_t)min(32 * kt + n, rows_here - 1) * p.k.stok;
#pragma unroll
                for (int ds = 0; ds < 8; ++ds) kf[kt][ds] = *reinterpret_cast<const bf16x8_t*>(kp + dim(ds));
            }
        }
        // ---- query tiles that see the block ----
        // first: t >= 64 kb - start; last (windows): t <= 64 kb + 63 + window - 1 - start, unless sinks lie in it
        const int tiles = (R + 31) >> 5;
        const int t_from = max(64 * kb - start, 0);
        const int t_to = p.window > 0 && 64 * kb >= p.sinks ? min(64 * kb - start + 62 + p.window, s.Lq - 1) : s.Lq - 1;
        const int u0 = (int)(((int64_t)t_from * G) >> 5);
        const int u1 = t_to < t_from ? 0 : min(tiles, (int)(((int64_t)(t_to + 1) * G + 31) >> 5));
        struct Tile {
            bf16x8_t q[8];
            float neg;  // -lse in log2 units
            int pos;    // the query's position, -1 where there is none or it sees no key
        };
        auto load = [&](int u) {
            Tile x;
            const int r = 32 * u + n;
            const bool valid = r < R;
            const int t = valid ? r / G : 0;
            const int hq = hk * G + (valid ? r - t * G : 0);
            const uint16_t* qp = p.q.data + b * p.q.sb + (int64_t)t * p.q.st + (int64_t)hq * p.q.sh;
#pragma unroll
            for (int ds = 0; ds < 8; ++ds) x.q[ds] = *reinterpret_cast<const bf16x8_t*>(qp + dim(ds));
            const float lse = p.lse[b * p.lse_sb + (int64_t)hq * p.lse_sh + t];
            x.neg = -lse * 1.4426950408889634f;
            x.pos = valid && lse != -__builtin_inff() ? start + t : -1;
            return x;
        };
        auto compute = [&](const Tile& x, int u) {
            f32x16_t sc[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int j = 0; j < 16; ++j) sc[kt][j] = 0.0f;
#pragma unroll
            for (int ds = 0; ds < 8; ++ds)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) sc[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kt][ds], x.q[ds], sc[kt], 0, 0, 0);
            // whole: every row of the tile sees the whole block
            // (a row without a key, at -1, sees none)
            const bool whole = x.pos >= 64 * kb + 63 && (p.window == 0 || x.pos - 64 * kb < p.window || 64 * kb + 63 < p.sinks);
            if (__ballot(!whole) == 0) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int j = 0; j < 16; ++j) acc[kt][j] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kt][j], p.scale_log2, x.neg));
            } else {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const int key = 64 * kb + 32 * kt + 8 * (j >> 2) + 4 * h + (j & 3);
                        const bool seen = key <= x.pos && (p.window == 0 || x.pos - key < p.window || key < p.sinks);
                        const float wt = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kt][j], p.scale_log2, x.neg));
                        acc[kt][j] += seen ? wt : 0.0f;
                    }
            }
            (void)u;
        };
        int u = u0 + sub;
        if (u < u1) {
            Tile a = load(u);
            for (; u < u1; u += kParts) {
                Tile next = a;
                if (u + kParts < u1) next = load(u + kParts);
                compute(a, u);
                a = next;
            }
        }
    }

    // ---- the sum over the 32 query rows of the lanes: of 32 values a lane gives half away at every step ----
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = acc[i >> 4][i & 15];
#pragma unroll
    for (int step = 0; step < 5; ++step) {
        const int half = 16 >> step;  // lanes n and n ^ half; the one whose bit is set keeps the upper values
        const bool up = (n & half) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = up ? v[i] : v[i + half];
            const float keep = up ? v[i + half] : v[i];
            v[i] = keep + __shfl_xor(give, half, 64);
        }
    }
    // lane (n, h) now holds the sum of value n: kt = n / 16, j = n % 16
    const int key = 32 * (n >> 4) + 8 * ((n & 15) >> 2) + 4 * h + (n & 3);
    float sum = v[0];
    if (kParts > 1) {
        part[w][l] = sum;
        __syncthreads();
        if (sub != 0) return;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kParts; ++i) sum += part[w + i][l];
    }
    const int j = 64 * kb + key;
    if (here && j < tokens) out[j] = mass[j] + sum;
}

}  // namespace

hipError_t launch_key_mass(const MassArgs& a, hipStream_t stream) {
    MassParams p{};
    p.s = a.s;
    p.q = a.q;
    if (a.k) p.k = *a.k;
    if (a.k4) p.k4 = *a.k4;
    p.table = a.table;
    p.table_stride = a.table_stride;
    p.counts = a.counts;
    p.lse = a.lse;
    p.lse_sb = a.lse_sb;
    p.lse_sh = a.lse_sh;
    p.mass = a.mass;
    p.mass_stride = a.mass_stride;
    p.out = a.out;
    p.out_stride = a.out_stride;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.window = a.window;
    p.sinks = a.sinks;
    int nkb = 1;
    int64_t blocks = 0;
    for (int b = 0; b < a.s.B; ++b) {
        p.start[b] = a.start[b];
        const int n = (a.start[b] + a.s.Lq + 63) / 64;
        nkb = max(nkb, n);
        blocks += (int64_t)a.s.Hkv * n;
    }
    if (a.table) blocks = (blocks + 3) / 4;
    const int tiles = (a.s.Lq * a.s.G + 31) / 32;
    int parts = 1;
    while (parts < 8 && tiles >= 2 * parts && blocks * parts < 8 * 512) parts *= 2;
    const int per = kMassWaves / parts;
    p.items = (nkb + (a.table ? 1 : 0) + per - 1) / per;  // (a list's last place copies what follows it)
    const int64_t grid = (int64_t)p.items * a.s.B * a.s.Hkv;
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kMassWaves * 64), 0, stream, p);
    };
    auto pick = [&](auto n) {
        constexpr int kParts = decltype(n)::value;
        if (a.k4)
            a.table ? launch(key_mass_kernel<true, true, kParts>) : launch(key_mass_kernel<true, false, kParts>);
        else
            a.table ? launch(key_mass_kernel<false, true, kParts>) : launch(key_mass_kernel<false, false, kParts>);
    };
    if (parts == 1) pick(std::integral_constant<int, 1>{});
    else if (parts == 2) pick(std::integral_constant<int, 2>{});
    else if (parts == 4) pick(std::integral_constant<int, 4>{});
    else pick(std::integral_constant<int, 8>{});
    return hipGetLastError();
}

}  // namespace ca
