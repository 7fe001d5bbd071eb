// The attention weight that every cached key received: out[row][j] = mass[row][j] + the sum over the queries and the
// query heads of the row's group that see key j of exp(q . k_j * scale - lse).
//
// The scores are S^T = K Q^T (16x16x32 bf16 MFMAs, fp32), so a lane holds keys of one query row, and the sum over query
// rows stays in the lane until the end: one fma, exp2 and add a score, and no atomics.  A wave keeps the 64 keys of one
// block in registers and goes through the packed query rows r = t * G + g, 16 at a time; K is read once.
// Where waves share a block they join in a fixed order, so results do not depend on what runs when.

#include <type_traits>

#include "ca_attn.h"
#include "ca_kv4.h"

namespace ca {
namespace {

constexpr int kMassWaves = 4;

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
    int items;      // workgroups of a row (and part)
    int parts;      // of the query tiles, every parts-th each, with workgroups of their own
    float* ws;      // the parts' sums [parts][rows][ws_stride], null where there is one
    int64_t ws_stride;
    int32_t start[CA_MAX_BATCH];
};

// A workgroup's row, place in the row's list and part of the query tiles (p.parts is 1, 2, 4, 8 or 16).  Workgroup i runs on
// XCD i % 8.  The parts of an item lie on XCDs of their own and the items of a row on all, so the XCDs carry equal work
// whatever the lists' lengths, and the L2 of each holds its part of the queries (a chunk over 20 % of 32768 tokens 173 us
// with a row's workgroups on one XCD, 158 so).  All blocks in one part: whole rows by XCD where they divide (64 queries over
// 32768 tokens 40 us, 36 so; all four with tiles through registers).
__device__ __forceinline__ void find_rows(const MassParams& p, int* row, int* item, int* cut) {
    const int x = blockIdx.x & 7, k = blockIdx.x >> 3;
    if (p.parts == 1 && p.table == nullptr && (p.s.B * p.s.Hkv) % 8 == 0) {
        *cut = 0;
        *row = k / p.items;
        *item = k - *row * p.items;
        *row = x + 8 * *row;
        return;
    }
    int at;
    if (p.parts <= 8) {
        *cut = x & (p.parts - 1);
        at = k * (8 / p.parts) + x / p.parts;
    } else {
        *cut = x + 8 * (k & 1);
        at = k >> 1;
    }
    *row = at / p.items;
    *item = at - *row * p.items;
}

// Blocks that a list leaves out keep their weights: a wave copies those before its entry e (from the one before it on), the
// wave after the last entry those behind it.
template <bool kTab>
__device__ __forceinline__ void copy_rest(const MassParams& p, int row, int e, int count, int nkb, int tokens, int l) {
    if (!kTab || p.out == p.mass || e > count) return;
    const int32_t* tab = p.table + (int64_t)row * p.table_stride;
    const int from = e == 0 ? 0 : min(max(tab[e - 1], 0), nkb - 1) + 1;
    const int to = e < count ? min(max(tab[e], 0), nkb - 1) : nkb;
    const int end = min(64 * to, tokens);
    constexpr int kAtOnce = 8;
    for (int j0 = 64 * from + l; j0 < end; j0 += 64 * kAtOnce) {
        float x[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) x[i] = j0 + 64 * i < end ? p.mass[(int64_t)row * p.mass_stride + j0 + 64 * i] : 0.0f;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
            if (j0 + 64 * i < end) p.out[(int64_t)row * p.out_stride + j0 + 64 * i] = x[i];
    }
}

// The 64 keys of a block, bf16: lane (n = l % 16, g = l / 16) holds key 16 kt + n, of the 32 dims of step j the eight of
// chunk(j, g) (the order of a product's dims is free where both operands share it).
template <bool kQ4>
struct Keys {
    bf16x8_t f[4][4];
    static __device__ __forceinline__ int chunk(int j, int g) { return kQ4 ? 4 * g + j : 4 * j + g; }
    __device__ __forceinline__ void load(const MassParams& p, int row, int b, int hk, int kb, int tokens, int n, int g) {
        if (kQ4) {
            const uint8_t* page = p.k4.data + clamp_page(sload(p.k4.page_table + (int64_t)row * p.k4.pts + kb), p.k4.max_page) * p.k4.stride;
            const uint32_t scales = *reinterpret_cast<const uint32_t*>(page + k4_scale(n, g));  // of tokens n, 16 + n, 32 + n, 48 + n
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                const u32x4_t code = *reinterpret_cast<const u32x4_t*>(page + 64 * (16 * kt + n) + 16 * g);
                const float sc = scale_of(scales, kt);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x4_t x = {decode2<0>(code[j], sc), decode2<1>(code[j], sc), decode2<2>(code[j], sc), decode2<3>(code[j], sc)};
                    f[kt][j] = __builtin_bit_cast(bf16x8_t, x);
                }
            }
        } else {
            const int64_t phys = p.k.page_table ? clamp_page(sload(p.k.page_table + (int64_t)row * p.k.pts + kb), p.k.max_page) : kb;
            const uint16_t* base = p.k.data + b * p.k.sb + hk * p.k.sh + phys * p.k.sblk;
            const int last = min(64, tokens - 64 * kb) - 1;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                // (past the cache's end: its last token, for a sum that nobody writes)
                const uint16_t* kp = base + (int64_t)min(16 * kt + n, last) * p.k.stok;
#pragma unroll
                for (int j = 0; j < 4; ++j) f[kt][j] = *reinterpret_cast<const bf16x8_t*>(kp + 8 * chunk(j, g));
            }
        }
    }
};

// acc += the weights that 16 query rows give to the block: lane (n, g) has row n, value i of acc[kt] is key
// 16 kt + 4 g + i.  neg: -lse of the row in log2 units.  kMask: the row at position pos may not see the whole block (pos
// -1: it sees nothing).
template <bool kQ4, bool kMask>
__device__ __forceinline__ void add_weights(const MassParams& p, const Keys<kQ4>& keys, const bf16x8_t (&q)[4], float neg, int pos, int kb,
                                            int g, f32x4_t (&acc)[4]) {
    f32x4_t sc[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) sc[kt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) sc[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(keys.f[kt][j], q[j], sc[kt], 0, 0, 0);
    // a row sees keys [0, hi] of the block, under a window those from lo on or before sink
    const int hi = pos - 64 * kb - 4 * g;
    const int lo = p.window > 0 ? hi - p.window + 1 : -64, sink = p.sinks - 64 * kb - 4 * g;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = 16 * kt + i;  // + 4 g
            const float wt = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kt][i], p.scale_log2, neg));
            // (dropped by a select: a hidden key may hold anything)
            acc[kt][i] += !kMask || ((key <= hi) & ((key >= lo) | (key < sink))) ? wt : 0.0f;
        }
}

// -lse in log2 units; a query without a key (lse -inf) gives weights of 0
__device__ __forceinline__ float neg_lse(float lse) {
    return lse == -__builtin_inff() ? lse : lse * -1.4426950408889634f;
}

// The sum over the 16 query rows of the lanes: of 16 values a lane gives half away at every step, and lane (n, g) ends
// with that of key 16 (n / 4) + 4 g + n % 4.
template <int kHalf>
__device__ __forceinline__ void give_half(float (&v)[16], int n) {  // lanes n and n ^ kHalf; that with the bit keeps the upper values
    const bool up = (n & kHalf) != 0;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
        const float give = up ? v[i] : v[i + kHalf];
        const float keep = up ? v[i + kHalf] : v[i];
        v[i] = keep + __shfl_xor(give, kHalf, 64);
    }
}
__device__ __forceinline__ float sum_rows(const f32x4_t (&acc)[4], int n) {
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = acc[i >> 2][i & 3];
    give_half<8>(v, n);
    give_half<4>(v, n);
    give_half<2>(v, n);
    give_half<1>(v, n);
    return v[0];
}

// At most 16 query rows (single tokens): one tile, a wave a block.  Bound by memory, K's bytes read once: one token over
// 131072 tokens of 8 KV heads (277 MB with the weights) takes 45 us, 6.1 TB/s.  With 32x32 products, whose operand takes 32
// bytes of a key at a time where these take 64, it took 197 us.
template <bool kQ4, bool kTab>
__global__ __launch_bounds__(kMassWaves * 64) __attribute__((amdgpu_waves_per_eu(3))) void key_mass_token_kernel(MassParams p) {
    const Shape& s = p.s;
    const int row = blockIdx.x / p.items;
    const int b = row / s.Hkv;
    const int hk = row - b * s.Hkv;
    const int G = s.G;
    const int start = p.start[b];
    const int tokens = start + s.Lq;
    const int nkb = (tokens + 63) >> 6;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = threadIdx.x & 63;
    const int n = l & 15;
    const int g = l >> 4;
    const int count = kTab ? min(max(sload(p.counts + row), 0), min(s.cap, nkb)) : nkb;
    const int e = (blockIdx.x - row * p.items) * kMassWaves + w;
    copy_rest<kTab>(p, row, e, count, nkb, tokens, l);
    if (e >= count) return;
    const int kb = kTab ? min(max(sload(p.table + (int64_t)row * p.table_stride + e), 0), nkb - 1) : e;
    Keys<kQ4> keys;
    keys.load(p, row, b, hk, kb, tokens, n, g);
    const bool valid = n < s.Lq * G;
    const int t = valid ? n / G : 0;
    const int hq = hk * G + (valid ? n - t * G : 0);
    const uint16_t* qp = p.q.data + b * p.q.sb + (int64_t)t * p.q.st + (int64_t)hq * p.q.sh;
    bf16x8_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const bf16x8_t*>(qp + 8 * keys.chunk(j, g));
    const float neg = neg_lse(p.lse[b * p.lse_sb + (int64_t)hq * p.lse_sh + t]);
    // the key whose sum this lane ends with, and its weight so far
    const int key_at = 64 * kb + 16 * (n >> 2) + 4 * g + (n & 3);
    const float old = key_at < tokens ? p.mass[(int64_t)row * p.mass_stride + key_at] : 0.0f;
    f32x4_t acc[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) acc[kt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    add_weights<kQ4, true>(p, keys, q, neg, valid ? start + t : -1, kb, g, acc);
    const float sum = sum_rows(acc, n);
    if (key_at < tokens) p.out[(int64_t)row * p.out_stride + key_at] = old + sum;
}

// ---------------------------------------------------------------------------------------
// Many query rows.  Four waves, each with the 64 keys of a block in registers, go through the packed rows together, the rows of
// 32 / G tokens at a time from LDS (four places in turn: while one is read the next three tiles are on their way; through
// registers and two places a chunk over 20 % of 32768 tokens took 161 us where it takes 150).  A launch may deal the tiles to
// p.parts, each with workgroups of its own; their sums go to p.ws and are joined in order by key_mass_join_kernel.
// Bound by vector instructions (one fma, exp2 and add a score: 24 cycles of a wave, beside 16 of the matrix cores):
// 2048 queries over 32768 tokens (32 Q / 8 KV heads) 523 us, 1.02 PFLOP/s of the 1.21 that a large product reaches; 64 queries
// 34 us, where a third is K's way from memory.  32x32x16 products, at two waves a SIMD where these run three, took 12 %
// longer; products woven into the weights of the tile before, instruction by instruction, 10 %.
constexpr int kTileRows = 32;
constexpr int kPlaces = 4;                   // tiles in LDS
constexpr int kTileBytes = kTileRows * 256;

// Words of a raw buffer resource over `bytes` bytes at base (wave-uniform).
__device__ __forceinline__ u32x4_t range_of(const void* base, int bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4_t{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a))),
                   static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(a >> 32) & 0xffff)),
                   static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(bytes)), 0x00020000u};
}
// Loads that write LDS: lane L's 16 (4) bytes at byte off of the resource go to LDS byte dst + 16 L (4 L); out of its range
// they write zeros.  (Five wait states from a vector instruction that writes the resource to its use: s_mov and s_nop 3.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds16(u32x4_t rsrc, uint32_t off, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(off), "s"(rsrc), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(u32x4_t rsrc, uint32_t off, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dword %0, %1, 0 offen lds" : : "v"(off), "s"(rsrc), "s"(dst) : "memory", "m0");
}
#pragma clang diagnostic pop

template <bool kQ4, bool kTab>
__global__ __launch_bounds__(kMassWaves * 64) __attribute__((amdgpu_waves_per_eu(3))) void key_mass_rows_kernel(MassParams p) {
    __shared__ __attribute__((aligned(16))) uint8_t tile[kPlaces][kTileBytes];
    __shared__ float tile_lse[kPlaces][kMassWaves][64];
    const Shape& s = p.s;
    int row, item, cut;
    find_rows(p, &row, &item, &cut);
    if (row >= s.B * s.Hkv) return;
    const int b = row / s.Hkv;
    const int hk = row - b * s.Hkv;
    const int G = s.G;
    const int start = p.start[b];
    const int tokens = start + s.Lq;
    const int nkb = (tokens + 63) >> 6;
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l = tid & 63;
    const int n = l & 15;
    const int g = l >> 4;
    const int32_t* tab = kTab ? p.table + (int64_t)row * p.table_stride : nullptr;
    const int count = kTab ? min(max(sload(p.counts + row), 0), min(s.cap, nkb)) : nkb;
    const int e0 = item * kMassWaves;
    const int e = e0 + w;
    if (p.ws == nullptr) copy_rest<kTab>(p, row, e, count, nkb, tokens, l);
    if (e0 >= count) return;
    const bool here = e < count;
    const int kb = kTab ? min(max(sload(tab + min(e, count - 1)), 0), nkb - 1) : min(e, count - 1);
    const int first_kb = kTab ? min(max(sload(tab + e0), 0), nkb - 1) : e0;  // of the workgroup's blocks
    const int last_kb = kTab ? min(max(sload(tab + min(e0 + kMassWaves, count) - 1), 0), nkb - 1) : min(e0 + kMassWaves, count) - 1;

    Keys<kQ4> keys;
    keys.load(p, row, b, hk, kb, tokens, n, g);

    // ---- the tiles that see a key of the workgroup's blocks; those in [ua, ub) see all of them whole ----
    // a tile is T whole tokens' rows: its rows' heads and tokens are the same in every tile
    const int T = kTileRows / G;
    const int tiles = (s.Lq + T - 1) / T;
    auto first_tile = [&](int t) { return t >= s.Lq ? tiles : max(t, 0) / T; };                     // with token t
    auto tile_after = [&](int t) { return t >= s.Lq ? tiles : (max(t, 0) + T - 1) / T; };           // past the tokens before t
    const bool edge = p.window > 0 && 64 * first_kb >= p.sinks;  // (blocks with sinks are seen to the end)
    const int u1 = edge ? tile_after(64 * last_kb - start + 63 + p.window) : tiles;
    // of those the part's: every p.parts-th
    const int u0 = first_tile(64 * first_kb - start) + ((cut - first_tile(64 * first_kb - start)) & (p.parts - 1));
    const int ua = tile_after(64 * last_kb - start + 63);
    const bool always = p.window == 0 || 64 * last_kb + 64 <= p.sinks;
    const int ub = always ? s.Lq / T : min(first_tile(64 * first_kb - start + p.window), s.Lq / T);
    // Wave w moves rows 4 w + 16 i + l / 16 of a tile (i = 0, 1) and its own copy of the rows' lse; chunk c of row r stands at
    // chunk c ^ (r % 16), for reads without bank conflicts.  Rows past T tokens' (where the group does not divide 32) and
    // past the last token count nowhere.
    const int q_sh = static_cast<int>(p.q.sh) * 2, q_st = static_cast<int>(p.q.st) * 2;  // bytes (the host checks their range)
    const int lse_sh = static_cast<int>(p.lse_sh) * 4;
    const int q_bytes = (s.Lq - 1) * q_st + (G - 1) * q_sh + 256, lse_bytes = (s.Lq - 1) * 4 + (G - 1) * lse_sh + 4;
    const u32x4_t q_rsrc = range_of(p.q.data + b * p.q.sb + (int64_t)hk * G * p.q.sh, q_bytes);
    const u32x4_t lse_rsrc = range_of(p.lse + b * p.lse_sb + (int64_t)hk * G * p.lse_sh, lse_bytes);
    int at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = min(16 * i + (tid >> 4), T * G - 1);
        at[i] = r / G * q_st + r % G * q_sh + 16 * ((tid & 15) ^ (tid >> 4));
    }
    const int lse_r = min(l & 31, T * G - 1), lse_at = lse_r / G * 4 + lse_r % G * lse_sh;
    const uint32_t tile0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to_lds(tile[0]))) + w * 1024;
    const uint32_t lse0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to_lds(reinterpret_cast<const uint8_t*>(tile_lse[0][w]))));
    auto fetch = [&](int u, int to) {  // (a tile past the last one: out of the ranges, no access; the range check covers the
                                       // vector offset only)
        const uint32_t qo = u < u1 ? u * T * q_st : q_bytes, lo = u < u1 ? u * T * 4 : lse_bytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) to_lds16(q_rsrc, at[i] + qo, tile0 + to * kTileBytes + 4096 * i);
        to_lds4(lse_rsrc, lse_at + lo, lse0 + to * (kMassWaves * 256));
    };
    int row_t[2];  // the token of the lane's rows in a tile, none's past T tokens' rows
#pragma unroll
    for (int i = 0; i < 2; ++i) row_t[i] = 16 * i + n < T * G ? (16 * i + n) / G : -(1 << 30);
    f32x4_t acc[4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) acc[kt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    int u = u0, from = 0;
    auto run = [&](int end, auto masked) {
        constexpr bool kMask = decltype(masked)::value;
        for (; u < end; u += p.parts) {
            // the tile is there (the six loads of the two behind it may be on their way), and the last one's reads are over
            asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            fetch(u + 3 * p.parts, (from + 3) & 3);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                bf16x8_t q[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    q[j] = *reinterpret_cast<const bf16x8_t*>(tile[from] + 4096 * i + n * 256 + ((keys.chunk(j, g) ^ n) * 16));
                const int t = u * T + row_t[i];
                const float neg = row_t[i] >= 0 ? neg_lse(tile_lse[from][w][16 * i + n]) : -__builtin_inff();
                add_weights<kQ4, kMask>(p, keys, q, neg, kMask && t >= 0 && t < s.Lq ? start + t : -1, kb, g, acc);
            }
            from = (from + 1) & 3;
        }
    };
    if (u0 < u1) {
        for (int i = 0; i < 3; ++i) fetch(u0 + i * p.parts, i);
        run(min(ua, u1), std::true_type{});
        run(min(ub, u1), std::false_type{});
        run(u1, std::true_type{});
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (loads into LDS end before the workgroup)
    }
    const float sum = sum_rows(acc, n);
    if (!here) return;
    const int key = 16 * (n >> 2) + 4 * g + (n & 3);
    if (p.ws != nullptr) {
        p.ws[((int64_t)cut * s.B * s.Hkv + row) * p.ws_stride + 64 * e + key] = sum;
    } else if (64 * kb + key < tokens) {
        const int64_t j = 64 * kb + key;
        p.out[(int64_t)row * p.out_stride + j] = p.mass[(int64_t)row * p.mass_stride + j] + sum;
    }
}

// The parts' sums added to the weights, a wave a block.
template <bool kTab>
__global__ __launch_bounds__(kMassWaves * 64) void key_mass_join_kernel(MassParams p) {
    const Shape& s = p.s;
    const int rows = s.B * s.Hkv;
    const int row = blockIdx.x / p.items;
    const int e = (blockIdx.x - row * p.items) * kMassWaves + (threadIdx.x >> 6);
    const int l = threadIdx.x & 63;
    const int tokens = p.start[row / s.Hkv] + s.Lq;
    const int nkb = (tokens + 63) >> 6;
    const int count = kTab ? min(max(p.counts[row], 0), min(s.cap, nkb)) : nkb;
    copy_rest<kTab>(p, row, e, count, nkb, tokens, l);
    if (e >= count) return;
    const int kb = kTab ? min(max(p.table[(int64_t)row * p.table_stride + e], 0), nkb - 1) : e;
    if (64 * kb + l >= tokens) return;
    float sum = 0.0f;
    for (int i = 0; i < p.parts; ++i) sum += p.ws[((int64_t)i * rows + row) * p.ws_stride + 64 * e + l];
    const int64_t j = 64 * kb + l;
    p.out[(int64_t)row * p.out_stride + j] = p.mass[(int64_t)row * p.mass_stride + j] + sum;
}

struct MassPlan {
    bool rows;       // key_mass_rows_kernel, else a block a wave (key_mass_token_kernel)
    int parts;       // rows: of the query tiles, each with workgroups of its own
};

// The query tiles are dealt to parts where the blocks alone are too few to fill the CUs a few times over (a list is taken
// to name a quarter of the blocks), with 8 tiles or more to a part, or 3 where there are fewer workgroups than CUs (100 queries
// over 500 tokens, 32 Q / 8 KV heads, 20.2 -> 11.9 us; 235 over 10 % of 28955, 16 / 2, 34.7 -> 26.2; where they are more, 64
// over 32768, 34 -> 44).
MassPlan key_mass_plan(const Shape& s, const int32_t* start, bool lists) {
    int64_t blocks = 0;
    for (int b = 0; b < s.B; ++b) blocks += (int64_t)s.Hkv * ((start[b] + s.Lq + 63) / 64);
    if (lists) blocks = (blocks + 3) / 4;
    MassPlan plan{s.Lq * s.G > 16, 1};
    const int T = kTileRows / s.G, tiles = (s.Lq + T - 1) / T;
    const int64_t groups = (blocks + kMassWaves - 1) / kMassWaves;
    auto few = [&](int least, int places) { return tiles >= 2 * least * plan.parts && groups * plan.parts < places; };
    while (plan.rows && plan.parts < 16 && (few(8, 2048) || few(3, 256))) plan.parts *= 2;
    return plan;
}

}  // namespace

int64_t key_mass_workspace_bytes(const Shape& s, const int32_t* start, bool lists) {
    const MassPlan plan = key_mass_plan(s, start, lists);
    if (!plan.rows || plan.parts <= 1) return 0;
    int nkb = 1;
    for (int b = 0; b < s.B; ++b) nkb = max(nkb, (start[b] + s.Lq + 63) / 64);
    const int64_t items = (nkb + (lists ? 1 : 0) + kMassWaves - 1) / kMassWaves | (lists ? 1 : 0);
    return (int64_t)plan.parts * s.B * s.Hkv * items * kMassWaves * 64 * (int64_t)sizeof(float);
}

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
    for (int b = 0; b < a.s.B; ++b) {
        p.start[b] = a.start[b];
        nkb = max(nkb, (a.start[b] + a.s.Lq + 63) / 64);
    }
    const MassPlan plan = key_mass_plan(a.s, a.start, a.table != nullptr);
    const int rows = a.s.B * a.s.Hkv;
    const int entries = nkb + (a.table ? 1 : 0);  // (a list's last place copies what follows it)
    p.items = (entries + kMassWaves - 1) / kMassWaves;
    // (lists: the rows' first items are those with blocks, an odd count deals them to all XCDs; 142 queries of 14 requests
    // 41.7 -> 39.5 us)
    if (a.table) p.items |= 1;
    p.parts = plan.parts;
    p.ws = plan.parts > 1 ? static_cast<float*>(a.workspace) : nullptr;
    p.ws_stride = (int64_t)64 * kMassWaves * p.items;
    auto launch = [&](auto kernel, int64_t grid) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(grid)), dim3(kMassWaves * 64), 0, stream, p);
    };
    const int64_t grid = (int64_t)p.items * rows, grid_parts = (grid * p.parts + 15) / 16 * 16;
    if (!plan.rows) {
        if (a.k4)
            a.table ? launch(key_mass_token_kernel<true, true>, grid) : launch(key_mass_token_kernel<true, false>, grid);
        else
            a.table ? launch(key_mass_token_kernel<false, true>, grid) : launch(key_mass_token_kernel<false, false>, grid);
        return hipGetLastError();
    }
    if (a.k4)
        a.table ? launch(key_mass_rows_kernel<true, true>, grid_parts) : launch(key_mass_rows_kernel<true, false>, grid_parts);
    else
        a.table ? launch(key_mass_rows_kernel<false, true>, grid_parts) : launch(key_mass_rows_kernel<false, false>, grid_parts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    a.table ? launch(key_mass_join_kernel<true>, grid) : launch(key_mass_join_kernel<false>, grid);
    return hipGetLastError();
}

}  // namespace ca
