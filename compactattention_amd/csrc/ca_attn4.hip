// Attention over a KV cache held in 4 bits (pages and conversions: ca_kv4.h): single tokens and short
// drafts over the whole cache, and chunks over the selected blocks.  Queries, weights and outputs are as
// in the bf16 kernels: S = Q K^T * scale in fp32 from exact bf16 operands, an online softmax in fp32, the
// weights rounded to bf16 once for O = P V, their sum taken of the rounded weights, O in fp32.
//
// What a mask hides has no effect, whatever it holds: hidden scores are replaced by -inf, and in the
// blocks that hold a hidden key (those that reach past the first query's position) values that no query
// of the request may see are read as zero, while a NaN value that some may see is taken out of the
// product and given to the rows that see it.  In all other blocks every row sees every key, and NaN goes
// through the products.

#include "ca_attn.h"
#include "ca_kv4.h"

namespace ca {
namespace {

struct Attn4Params {
    AttnParams a;
    Kv4Addr k, v;
};
static_assert(sizeof(Attn4Params) <= 4096, "the arguments of a launch");

constexpr float kNegInf = -__builtin_inff();
constexpr int kNoKey = 0x7fffffff;

__device__ __forceinline__ u32x4_t load16(const uint8_t* p) { return *reinterpret_cast<const u32x4_t*>(p); }

// Whether a query sees one of the keys (a bit each) of a block under a window: at is its position and sinks the end of
// the sinks, counted from the block's start.
__device__ __forceinline__ bool sees(uint32_t lo, uint32_t hi, int at, int window, int sinks) {
    auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; };  // keys 0 .. n - 1
    const uint64_t seen = below(at + 1) & (~below(at + 1 - window) | below(sinks));
    return ((static_cast<uint64_t>(hi) << 32 | lo) & seen) != 0;
}

// 8 values of one word of codes under one scale: a row of 8 dims, bf16
__device__ __forceinline__ u32x4_t decode_row(uint32_t w, float s) {
    return u32x4_t{decode2<0>(w, s), decode2<1>(w, s), decode2<2>(w, s), decode2<3>(w, s)};
}

// ---------------------------------------------------------------------------------------
// Single tokens, drafts and small chunks: kN tiles of 16 packed query rows a workgroup (1 for at most 16
// rows, 2 for more, in several workgroups), over the whole cache or (kTab) the blocks of the per-row lists.
// 16x16x32 MFMAs, S^T = K Q^T and O^T += V^T P^T, with the packed rows as the N dimension.  Eight waves, each
// with pages of its own (e0 + w, e0 + w + 8, ...) and its own softmax; their results meet in LDS at the end.
// Every cached byte is read once for 16 rows (68 bytes a token of K and of V).  One token over 131072 (8 KV
// heads, 143 MB) takes 27 us, 5.3 TB/s; 6 us of every launch are its start, a first page's way from memory and
// the end in LDS, and what follows comes at 6.8 TB/s.  Short lists are bound by the conversions: a page is some
// 500 vector instructions, 0.8 us for the four SIMDs' pages of a turn.
//  - The contraction order of a product is free as long as both operands share it, so the page's layout
//    decides it and nothing crosses lanes: lane (n = l % 16, g = l / 16) has token 16 kt + n's group g
//    (16 bytes) as its share of K, and takes the dims 32 g + 8 s .. + 7 in step s; the scores then lie
//    with the lane as tokens 16 kt + 4 g + i, and its share of V is dims 8 n .. 8 n + 7 of those tokens.
//  - V's words are tokens, the MFMA wants tokens side by side: v_perm_b32 pairs them.  Output tile j
//    holds the dims 8 m + j, so a lane ends with 8 consecutive dims of its row.
constexpr int kWaves4 = 8;
constexpr int kOStride4 = 132;  // floats per row of a wave's partial O in LDS (padded)

struct Page4 {
    u32x4_t k[4], v[4], vs;  // by tile of 16 tokens: K, V; V's scale bytes (word: tile)
    uint32_t ks;             // K's scale bytes (byte: tile)
    int kb;                  // logical block
};

// One work item.  kStream: K and V are loaded with the non-temporal hint.  kWin: the blocks of a window (WindowList).
template <int kN, bool kTab, bool kStream, bool kWin = false>
__device__ __forceinline__ void decode4_item(const Attn4Params& p4, const Item& it, float* mo, float* ml) {
    constexpr int kCache = kStream ? 2 : 0;  // cache policy of the loads: nt
    const AttnParams& p = p4.a;
    const Shape& s = p.s;
    const int row = it.row;
    const int b = it.b;
    const int split = it.split;
    const int r0 = kN == 1 ? 0 : 16 * kN * it.tile;
    const int hk = row - b * s.Hkv;
    const int nsplit = p.sp[b];
    const int G = s.G;
    const int R = p.rows_total;
    const int qpos0 = p.qpos0[b];
    const int nkb = p.nkb[b];
    const int kv_tokens = qpos0 + s.Lq;
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l = tid & 63;
    const int n = l & 15;
    const int g = l >> 4;
    // blocks from here on hold keys past the tile's first query
    const int mask_from = (qpos0 + (kN == 1 ? 0 : r0 / G) + 1) >> 6;
    const int32_t* tab = kTab ? p.table + (int64_t)row * p.table_stride : nullptr;
    const WindowList win(qpos0 + (kN == 1 ? 0 : r0 / G), qpos0 + (kN == 1 ? s.Lq - 1 : min(r0 + 16 * kN - 1, R - 1) / G),
                         p.window, p.sinks);
    int n_vis = kWin ? win.total : nkb;
    if (kTab) {  // entries up to the last one that the tile can see
        const int lim = (qpos0 + min(r0 + 16 * kN - 1, R - 1) / G) >> 6;
        n_vis = 0;
        for (int end = min(max(sload(p.counts + row), 0), s.cap); end > 0; end -= 64) {
            const int e = end - 1 - l;
            const uint64_t seen = __ballot(e >= 0 && min(max(tab[max(e, 0)], 0), nkb - 1) <= lim);
            if (seen != 0) {
                n_vis = end - (__ffsll(static_cast<unsigned long long>(seen)) - 1);
                break;
            }
        }
    }
    const int chunk = (n_vis + nsplit - 1) / nsplit;
    const int e0 = min(n_vis, split * chunk);
    const int e1 = min(n_vis, e0 + chunk);

    const int32_t* kpt = p4.k.page_table + (int64_t)row * p4.k.pts;
    const int32_t* vpt = p4.v.page_table + (int64_t)row * p4.v.pts;
    const int k_off = 64 * n + 16 * g;
    const int v_off = 16 * l;
    const int ks_off = k4_scale(n, g);
    const int vs_off = v4_scale(4 * g, n >> 2);

    // this wave's pages, 64 at a time, one per lane
    const int nb_w = e0 + w < e1 ? (e1 - 1 - (e0 + w)) / kWaves4 + 1 : 0;
    int kbid = 0, kid = 0, vid = 0;
    auto load_ids = [&](int c) {
        const int e = max(min(e0 + w + kWaves4 * (64 * c + l), e1 - 1), 0);
        kbid = kTab ? min(max(tab[e], 0), nkb - 1) : kWin ? win.block(e) : e;
        const int kp = kpt[kbid], vp = vpt[kbid];
        kid = static_cast<int>(clamp_page(kp, p4.k.max_page));
        vid = static_cast<int>(clamp_page(vp, p4.v.max_page));
    };
    // Loads stand outside any branch: behind one, the page in use would wait for those ahead of it too (131072
    // tokens 30.6 us with the merge, 29.4 so; 32 requests of 1024 12.2, 10.8).  Past the last page their range is
    // empty and nothing is read.
    auto load_page = [&](int i) {
        if (i > 0 && (i & 63) == 0) load_ids(i >> 6);
        const int size = i < nb_w ? kPage4 : 0;
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(p4.k.data) + (int64_t)__builtin_amdgcn_readlane(kid, i & 63) * p4.k.stride, 0, size, 0x00020000);
        const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(p4.v.data) + (int64_t)__builtin_amdgcn_readlane(vid, i & 63) * p4.v.stride, 0, size, 0x00020000);
        Page4 x;
        x.kb = __builtin_amdgcn_readlane(kbid, i & 63);
        x.ks = __builtin_amdgcn_raw_buffer_load_b32(kr, ks_off, 0, kCache);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) x.k[kt] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off + 1024 * kt, 0, kCache);
        __builtin_amdgcn_sched_barrier(0);
        x.vs = __builtin_amdgcn_raw_buffer_load_b128(vr, vs_off, 0, kCache);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) x.v[kt] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_off + 1024 * kt, 0, kCache);
        return x;
    };
    load_ids(0);

    // the queries come before the pages: what is waited for first in the loop is then what was loaded first
    bf16x8_t qf[kN][4];
    int qpos[kN];
#pragma unroll
    for (int u = 0; u < kN; ++u) {
        const int r = r0 + 16 * u + n;
        const bool valid = r < R;
        const int qt = valid ? r / G : 0;
        const int qg = valid ? r - qt * G : 0;
        const uint16_t* qp = p.q.data + b * p.q.sb + (int64_t)qt * p.q.st + (int64_t)(hk * G + qg) * p.q.sh + 32 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u32x4_t z = {0u, 0u, 0u, 0u}, x = *reinterpret_cast<const u32x4_t*>(qp + 8 * j);
            qf[u][j] = __builtin_bit_cast(bf16x8_t, valid ? x : z);
        }
        qpos[u] = qpos0 + qt;
    }
    Page4 xa = load_page(0), xb;

    const float sl2 = p.scale_log2;
    f32x4_t oacc[kN][8];
    float m_run[kN], l_run[kN];
#pragma unroll
    for (int u = 0; u < kN; ++u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) oacc[u][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        m_run[u] = kNegInf;
        l_run[u] = 0.0f;
    }
    const bf16x2_t ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};

    auto compute = [&](Page4& x) {
        f32x4_t sc[kN][4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            const float ks = scale_of(x.ks, kt);
#pragma unroll
            for (int u = 0; u < kN; ++u) sc[u][kt] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf16x8_t kf = __builtin_bit_cast(bf16x8_t, decode_row(x.k[kt][j], ks));
#pragma unroll
                for (int u = 0; u < kN; ++u)
                    sc[u][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[u][j], sc[u][kt], 0, 0, 0);
            }
        }
        int nan_at = kNoKey;  // the first position with a NaN value in this lane's output dims
        uint32_t nan_lo = 0, nan_hi = 0;  // kWin: the block's keys with one, a bit each
        if (kWin ? win.cut(x.kb) : x.kb >= mask_from) {
            // value i of tile kt is key 64 kb + 16 kt + 4 g + i
            const int first = 64 * x.kb + 4 * g;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = first + 16 * kt + e;
#pragma unroll
                    for (int u = 0; u < kN; ++u)
                        if (key > qpos[u] || (kWin && key <= qpos[u] - p.window && key >= p.sinks)) sc[u][kt][e] = kNegInf;
                    const bool bad = ((x.vs[kt] >> (8 * e)) & 0xffu) == kScaleNan;
                    if (kWin) {
                        const uint32_t bit = bad && key < kv_tokens ? 1u << ((16 * kt + 4 * g + e) & 31) : 0u;
                        (kt < 2 ? nan_lo : nan_hi) |= bit;
                    } else if (bad && key < kv_tokens) {
                        nan_at = min(nan_at, key);
                    }
                    if (bad || key >= kv_tokens) {
                        x.v[kt][e] = 0;
                        x.vs[kt] &= ~(0xffu << (8 * e));
                    }
                }
            if (kWin && __ballot((nan_lo | nan_hi) != 0)) {
                // as below: over the lanes that hold this group of dims, then to those whose output dims these are
                auto gather = [&](uint32_t m) {
                    m |= __shfl_xor(m, 1, 64);
                    m |= __shfl_xor(m, 2, 64);
                    m |= __shfl_xor(m, 16, 64);
                    m |= __shfl_xor(m, 32, 64);
                    return static_cast<uint32_t>(__shfl(m, 4 * g, 64));
                };
                nan_lo = gather(nan_lo);
                nan_hi = gather(nan_hi);
            }
            if (!kWin && __ballot(nan_at != kNoKey)) {
                // over the four lanes and the four lane groups that hold this group of dims, then to the
                // lanes whose output dims these are: 8 (4 g + i) + j, group g
                nan_at = min(nan_at, __shfl_xor(nan_at, 1, 64));
                nan_at = min(nan_at, __shfl_xor(nan_at, 2, 64));
                nan_at = min(nan_at, __shfl_xor(nan_at, 16, 64));
                nan_at = min(nan_at, __shfl_xor(nan_at, 32, 64));
                nan_at = __shfl(nan_at, 4 * g, 64);
            }
        }
        bf16x8_t pf[kN][2];
#pragma unroll
        for (int u = 0; u < kN; ++u) {
            float mx = kNegInf;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, sc[u][kt][e]);
            mx = xor32_max(xor16_max(mx)) * sl2;
            float alpha = 1.0f;
            if (mx > m_run[u] + kRescale) {
                alpha = __builtin_amdgcn_exp2f(m_run[u] - mx);
                m_run[u] = mx;
                l_run[u] *= alpha;
            }
            if (__ballot(alpha != 1.0f)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) oacc[u][j] *= alpha;
            }
            const float m_use = m_run[u] == kNegInf ? 0.0f : m_run[u];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f32x8_t pv8;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    pv8[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][2 * half + (e >> 2)][e & 3], sl2, -m_use));
                const bf16x8_t pw = __builtin_convertvector(pv8, bf16x8_t);
                l_run[u] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pw, pw, 0, 1), ones, l_run[u], false);
                l_run[u] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pw, pw, 2, 3), ones, l_run[u], false);
                l_run[u] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pw, pw, 4, 5), ones, l_run[u], false);
                l_run[u] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_shufflevector(pw, pw, 6, 7), ones, l_run[u], false);
                pf[u][half] = pw;
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            u32x4_t t[8];  // the 8 tokens' rows of 8 dims
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int kt = 2 * half + (e >> 2);
                t[e] = decode_row(x.v[kt][e & 3], scale_of(x.vs[kt], e & 3));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
                const u32x4_t a = {__builtin_amdgcn_perm(t[1][j >> 1], t[0][j >> 1], sel),
                                   __builtin_amdgcn_perm(t[3][j >> 1], t[2][j >> 1], sel),
                                   __builtin_amdgcn_perm(t[5][j >> 1], t[4][j >> 1], sel),
                                   __builtin_amdgcn_perm(t[7][j >> 1], t[6][j >> 1], sel)};
#pragma unroll
                for (int u = 0; u < kN; ++u)
                    oacc[u][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), pf[u][half],
                                                                         oacc[u][j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < kN; ++u)
            if (kWin ? sees(nan_lo, nan_hi, qpos[u] - 64 * x.kb, p.window, p.sinks - 64 * x.kb) : nan_at <= qpos[u]) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) oacc[u][j][e] = __builtin_nanf("");
            }
    };

    for (int i = 0; i < nb_w; i += 2) {
        xb = load_page(i + 1);
        __builtin_amdgcn_sched_barrier(0);
        compute(xa);
        xa = load_page(i + 2);
        if (i + 1 < nb_w) compute(xb);
    }

    // ---- the eight waves' results through LDS, 16 rows at a time ----
#pragma unroll
    for (int u = 0; u < kN; ++u) {
        float ls = l_run[u];
        ls += __shfl_xor(ls, 16, 64);
        ls += __shfl_xor(ls, 32, 64);
        if (u > 0) __syncthreads();
        // tile j, value i: dim 8 (4 g + i) + j of row n
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float* to = mo + (w * 16 + n) * kOStride4 + 8 * (4 * g + i);
            *reinterpret_cast<f32x4_t*>(to) = f32x4_t{oacc[u][0][i], oacc[u][1][i], oacc[u][2][i], oacc[u][3][i]};
            *reinterpret_cast<f32x4_t*>(to + 4) = f32x4_t{oacc[u][4][i], oacc[u][5][i], oacc[u][6][i], oacc[u][7][i]};
        }
        if (g == 0) {
            ml[(w * 16 + n) * 2 + 0] = m_run[u];
            ml[(w * 16 + n) * 2 + 1] = ls;
        }
        __syncthreads();
        const int lrow = tid >> 5;  // 16 rows x 32 threads, 4 dims each
        const int orow = r0 + 16 * u + lrow;
        const int d4 = (tid & 31) * 4;
        if (orow < R) {
            float mx = kNegInf;
#pragma unroll
            for (int v = 0; v < kWaves4; ++v) mx = fmaxf(mx, ml[(v * 16 + lrow) * 2]);
            const float m_use = mx == kNegInf ? 0.0f : mx;
            f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
            float wsum = 0.0f;
#pragma unroll
            for (int v = 0; v < kWaves4; ++v) {
                const float wv = __builtin_amdgcn_exp2f(ml[(v * 16 + lrow) * 2] - m_use);
                wsum += wv * ml[(v * 16 + lrow) * 2 + 1];
                acc += wv * *reinterpret_cast<const f32x4_t*>(mo + (v * 16 + lrow) * kOStride4 + d4);
            }
            // no key: zeros and -inf; a NaN sum stays
            const float inv = wsum == 0.0f ? 0.0f : 1.0f / wsum;
            const float lse2 = wsum == 0.0f ? kNegInf : m_use + __log2f(wsum);
            acc *= inv;
            const int ot = orow / G;
            const int hq = hk * G + orow - ot * G;
            if (nsplit == 1) {
                uint16_t* op = p.out.data + b * p.out.sb + (int64_t)ot * p.out.st + (int64_t)hq * p.out.sh + d4;
                *reinterpret_cast<bf16x4_t*>(op) = __builtin_convertvector(acc, bf16x4_t);
                if (p.lse && (tid & 31) == 0) p.lse[((int64_t)b * s.Hq + hq) * s.Lq + ot] = lse2 * 0.69314718055994531f;
            } else {
                const int64_t prow = ((int64_t)split * (s.B * s.Hkv) + row) * R + orow;
                *reinterpret_cast<f32x4_t*>(p.ws_o + prow * 128 + d4) = acc;
                if ((tid & 31) == 0) p.ws_lse[prow] = lse2;
            }
        }
    }
}

// How K and V are loaded: to stay in the caches (chunks and drafts of several tiles read them again), past them,
// or past them where no other request reads the item's pages.  Past them is faster even for small caches, as a
// model's layers take turns in what the last-level cache (256 MB) holds: one token over 4096 tokens, 80 caches
// in turn, 10.0 us kept, 9.0 past them; one cache again and again 8.6, 8.6; 131072 tokens, 4 caches in turn 34.8,
// 30.5, 64 requests of 4096, 3 caches 55.5, 50.5.  Slower only for one cache near that size again and again (64
// requests of 4096, 285 MB, 47.2, 48.9).
enum { kLoadsKept, kLoadsStreamed, kLoadsStreamedUnshared };
template <int kN, bool kTab, int kLoads, bool kWin = false>
__global__ __launch_bounds__(kWaves4 * 64) __attribute__((amdgpu_waves_per_eu(2))) void attn4_decode_kernel(Attn4Params p4) {
    __shared__ __attribute__((aligned(16))) float mo[kWaves4 * 16 * kOStride4];
    __shared__ float ml[kWaves4 * 16 * 2];
    Item it;
    if (!find_item(p4.a, kN == 1 ? 1 : p4.a.ntiles, &it)) return;
    it.row = __builtin_amdgcn_readfirstlane(it.row);
    it.b = __builtin_amdgcn_readfirstlane(it.b);
    it.split = __builtin_amdgcn_readfirstlane(it.split);
    it.tile = __builtin_amdgcn_readfirstlane(it.tile);
    if (kLoads == kLoadsStreamed ||
        (kLoads == kLoadsStreamedUnshared && !shares_pages(p4.a, it, p4.k.page_table, p4.k.pts)))
        decode4_item<kN, kTab, true, kWin>(p4, it, mo, ml);
    else
        decode4_item<kN, kTab, false, kWin>(p4, it, mo, ml);
}

// ---------------------------------------------------------------------------------------
// Chunks, and drafts with many packed rows: 256 packed rows a workgroup, 32 a wave, with the products and
// the software pipeline of the bf16 kernel: the scores of the next block run beside the softmax of this one,
// then its PV product beside the next block's row max, instruction by instruction (fused).
// A block's codes go from memory to registers (16 bytes a thread: waves 0-3 a group of a token of K, waves
// 4-7 8 dims of four tokens of V), through 16 conversions to bf16 and into LDS in the bf16 kernel's places,
// between the MFMAs of the PV product.  Rings of four K and four V blocks in LDS, K of block j in place
// j & 3 and V in place (j + 1) & 3; slot j writes K of j + 3 and V of j + 2 (one place for all waves)
// and loads the codes of the blocks after those.
// Bound by the matrix cores and their power, as the bf16 kernel: 2048 queries over 34816 dense keys (32 Q / 8 KV
// heads) 913-950 us where bf16 pages take 876-909, 1.2 PFLOP/s.  A loop without the pipeline took 1095.
// kTab: block lists come from the per-row table; otherwise they are the identity (drafts).
constexpr int kPlace4 = 64 * 256;     // K or V rows of one block in LDS
constexpr int kVRing4 = 4 * kPlace4;  // LDS byte offset of the V ring

template <int N>
struct Int4C {
    static constexpr int value = N;
};

template <bool kTab, bool kWin = false>
__global__ __launch_bounds__(kNW * 64) __attribute__((amdgpu_waves_per_eu(2))) void attn4_fwd_kernel(Attn4Params p4) {
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * kVRing4];
    // by block modulo 4 and group of dims: the first key in the block with a NaN value (masked blocks), kWin: a
    // bit for every key with one
    __shared__ int vnan[4][4];
    __shared__ uint32_t vbits[4][4][2];
    __shared__ int late[kNW];
    const AttnParams& p = p4.a;
    const Shape& s = p.s;
    Item it;
    if (!find_item(p, p.ntiles, &it)) return;
    const int row = __builtin_amdgcn_readfirstlane(it.row);
    const int b = __builtin_amdgcn_readfirstlane(it.b);
    const int split = __builtin_amdgcn_readfirstlane(it.split);
    const int tile = __builtin_amdgcn_readfirstlane(it.tile);
    const int hk = row - b * s.Hkv;
    const int nsplit = p.sp[b];
    const int G = s.G;
    const int qpos0 = p.qpos0[b];
    const int nkb = p.nkb[b];
    const int rows_total = p.rows_total;
    const int r0 = tile * kBM;
    const int t_first = r0 / G;
    const int t_last = min(r0 + kBM - 1, rows_total - 1) / G;
    const int32_t* tab = kTab ? p.table + (int64_t)row * p.table_stride : nullptr;
    const int lim = (qpos0 + t_last) >> 6;  // last block the tile can see
    const int kv_tokens = qpos0 + s.Lq;
    const int first_q = qpos0 + t_first;  // blocks that reach past it are masked
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l = tid & 63;
    const int h = l >> 5;
    const int n = l & 31;

    int qpos;
    bf16x8_t qf[8];
    {
        const int qrow = r0 + 32 * w + n;
        const bool qvalid = qrow < rows_total;
        const int qt = qvalid ? qrow / G : 0;
        const int qg = qvalid ? qrow - qt * G : 0;
        qpos = qpos0 + qt;
        const uint16_t* qp = p.q.data + b * p.q.sb + (int64_t)qt * p.q.st + (int64_t)(hk * G + qg) * p.q.sh + 8 * h;
#pragma unroll
        for (int ds = 0; ds < 8; ++ds) {
            const u32x4_t z = {0u, 0u, 0u, 0u};
            qf[ds] = qvalid ? *reinterpret_cast<const bf16x8_t*>(qp + 16 * ds) : __builtin_bit_cast(bf16x8_t, z);
        }
    }
    const WindowList win(first_q, qpos0 + t_last, p.window, p.sinks);
    if (kWin) {
        if (tid < 32) (&vbits[0][0][0])[tid] = 0;
    } else if (tid < 16) {
        vnan[tid >> 2][tid & 3] = 64;
    }
    // entries up to the last one that the tile can see
    int n_vis = kTab ? 0 : kWin ? win.total : min(nkb, lim + 1);
    if (kTab) {
        for (int end = min(max(sload(p.counts + row), 0), s.cap); end > 0; end -= 64) {
            const int e = end - 1 - l;
            const uint64_t seen = __ballot(e >= 0 && min(max(tab[max(e, 0)], 0), nkb - 1) <= lim);
            if (seen != 0) {
                n_vis = end - (__ffsll(static_cast<unsigned long long>(seen)) - 1);
                break;
            }
        }
    }
    const int chunk = (n_vis + nsplit - 1) / nsplit;
    const int e0 = min(n_vis, split * chunk);
    const int nblk = min(n_vis, e0 + chunk) - e0;
    // blocks before the first masked one; a list's order is not relied on: every wave looks through an eighth
    const int whole = (first_q + 1) >> 6;  // blocks [0, whole) hold no key past the tile's first query
    int n_un = min(max((kWin ? win.full : whole) - e0, 0), nblk);
    if (kTab) {
        int first = nblk;
        for (int at = 64 * w; at < nblk; at += 64 * kNW) {
            const int id = at + l < nblk ? tab[e0 + at + l] : 0;
            const uint64_t hit = __ballot(at + l < nblk && min(max(id, 0), nkb - 1) >= whole);
            if (hit != 0) {
                first = at + __ffsll(static_cast<unsigned long long>(hit)) - 1;
                break;
            }
        }
        if (l == 0) late[w] = first;
    }

    f32x16_t oacc[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int j = 0; j < 16; ++j) oacc[dt][j] = 0.0f;
    float m_run = kNegInf;
    float l_run = 0.0f;
    float m_neg = 0.0f;  // -m_run, 0 while a row has seen no key

    // ---- the pages of the list's blocks, 64 entries at a time, one per lane (past its end: the last entry) ----
    const bool is_v = w >= 4;
    const Kv4Addr& kv = is_v ? p4.v : p4.k;
    const int32_t* pt = kv.page_table + (int64_t)row * kv.pts;
    int cur_page = 0, next_page = 0;
    auto load_pages = [&](int c) {
        const int e = e0 + min(64 * c + l, nblk - 1);
        const int id = kTab ? min(max(tab[e], 0), nkb - 1) : kWin ? win.block(e) : e;
        next_page = static_cast<int>(clamp_page(pt[id], kv.max_page));
    };
    auto id_of = [&](int i) { return kTab ? min(max(sload(tab + e0 + i), 0), nkb - 1) : kWin ? win.block(e0 + i) : e0 + i; };
    // ---- a block's codes: memory -> registers (of this wave's cache; i asked for in ascending order) ----
    const int u = tid & 255;
    const int st_t = is_v ? 4 * (u >> 4) : u >> 2;  // token (of V: the first of four)
    const int st_c = is_v ? u & 15 : 4 * (u & 3);   // 16-byte chunk of the row in LDS (of K: the first of four)
    const int sc_off = is_v ? v4_scale(st_t, st_c >> 2) : k4_scale(st_t, u & 3) & ~3;  // the word with the byte(s)
    struct Codes {
        u32x4_t code;
        uint32_t scale;
    };
    auto fetch = [&](int i) {
        if ((i & 63) == 0) {
            cur_page = next_page;
            load_pages((i >> 6) + 1);
        }
        Codes x;
        const uint8_t* page = kv.data + (int64_t)__builtin_amdgcn_readlane(cur_page, i & 63) * kv.stride;
        x.code = load16(page + 16 * u);
        x.scale = *reinterpret_cast<const uint32_t*>(page + sc_off);
        return x;
    };
    // ---- registers -> bf16 rows in LDS ----
    //   K: 16-byte chunk c of row r sits at chunk c ^ (r & 15), V: at chunk c ^ 4 (r & 3)
    // (chunk or row i of a thread's four: bits flipped and bytes added to the first one's address)
    const int to = is_v ? kVRing4 + st_t * 256 + st_c * 16 : st_t * 256 + (st_c ^ (st_t & 15)) * 16;
    const int to_flip = is_v ? 64 : 16, to_add = is_v ? 256 : 0;
    // Before a block's conversions: K's one scale byte to all four words' places; of V's blocks from the first
    // masked one on the values that no query may see become zero, and NaN, which goes to the rows that see it
    // after the product.
    auto settle = [&](Codes& x, int block) {
        if (!is_v) {
            x.scale = ((x.scale >> (8 * w)) & 0xffu) * 0x01010101u;  // K's token 16 w + l / 4
        } else if (block >= n_un) {
            const int first = 64 * id_of(min(block, nblk - 1)) + st_t;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool bad = ((x.scale >> (8 * i)) & 0xffu) == kScaleNan;
                const bool there = first + i < kv_tokens;
                if (kWin && bad && there) atomicOr(&vbits[block & 3][st_c >> 2][(st_t + i) >> 5], 1u << ((st_t + i) & 31));
                if (!kWin && bad && there) atomicMin(&vnan[block & 3][st_c >> 2], st_t + i);
                if (bad || !there) {
                    x.code[i] = 0;
                    x.scale &= ~(0xffu << (8 * i));
                }
            }
        }
    };
    auto put = [&](const Codes& x, int place, int i) {
        *reinterpret_cast<u32x4_t*>(smem + ((to ^ (to_flip * i)) + to_add * i) + place * kPlace4) = decode_row(x.code[i], scale_of(x.scale, i));
    };
    // slot j writes this wave's block j + lead (K: j + 3, V: j + 2) to place (j + 3) & 3
    const int lead = is_v ? 2 : 3;
    Codes held;  // the codes that the next slot writes
    auto stage = [&](int j) {
        settle(held, j + lead);
#pragma unroll
        for (int i = 0; i < 4; ++i) put(held, (j + 3) & 3, i);
        held = fetch(j + lead + 1);
    };

    const float sl2 = p.scale_log2;
    // Fragment addresses, as in the bf16 kernel: K rows swap23(n) (+32), 16 bytes at d = 16 ds + 8 h; V^T by
    // transposing reads of 8 bytes at row 16 s4 + 8 h + 4 hh + (l & 15) / 4, d = 32 dt + 16 ((l >> 4) & 1) + 4 (l & 3).
    const int k_r = swap23(n);
    int k_off[8];
#pragma unroll
    for (int ds = 0; ds < 8; ++ds) k_off[ds] = k_r * 256 + (((2 * ds + h) ^ (k_r & 15)) * 16);
    const int v_rq = (l & 15) >> 2;
    const int v_x = 2 * ((l >> 4) & 1) + ((l & 3) >> 1);
    int v_off[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) v_off[dt] = kVRing4 + (8 * h + v_rq) * 256 + (4 * (dt ^ v_rq) + v_x) * 16 + (l & 1) * 8;
    const i16x4_t ones = {0x3f80, 0x3f80, 0x3f80, 0x3f80};
    auto add_weights = [&](uint32_t w0, uint32_t w1, f32x4_t acc) {
        const u32x2_t ww = {w0, w1};
        return __builtin_amdgcn_mfma_f32_4x4x4bf16_1k(ones, __builtin_bit_cast(i16x4_t, ww), acc, 0, 0, 0);
    };
    f32x16_t sc[2];  // scores of the block whose softmax comes next (32 keys each)
    auto k_frag = [&](int base, int i) {
        return *reinterpret_cast<const bf16x8_t*>(smem + base + k_off[i >> 1] + (i & 1) * 8192);
    };
    auto v_frag = [&](int base, int i) {  // A operand of PV MFMA i: 16-key step i / 4, 32-d tile i % 4
        const uint8_t* vp = smem + base + v_off[i & 3] + (i >> 2) * 4096;
        const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(to_lds_v4(vp));
        const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(to_lds_v4(vp + 1024));
        return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto scores = [&](int kbase) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int j = 0; j < 16; ++j) sc[kt][j] = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(kbase, i), qf[i >> 1], sc[i & 1], 0, 0, 0);
    };
    auto mask = [&](int kb) {
        const int vis = qpos - 64 * kb - 8 * h;
        const int past = kWin ? vis - p.window : 0, sink = kWin ? p.sinks - 64 * kb - 8 * h : 0;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int key = kt * 32 + 16 * (e >> 3) + 4 * ((e >> 2) & 1) + (e & 3);
                if (key > vis || (kWin && key <= past && key >= sink)) sc[kt][e] = kNegInf;
            }
    };
    auto rise = [&](float mx) {
        float alpha = 1.0f;
        if (mx > m_run + kRescale) {
            alpha = __builtin_amdgcn_exp2f(m_run - mx);  // 0 when m_run = -inf
            m_run = mx;
            m_neg = -mx;
            l_run *= alpha;
        }
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) oacc[dt][e] *= alpha;
    };
    auto block_max = [&]() {
        float mx = kNegInf;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, sc[kt][e]);
        mx = xor32_max(mx) * sl2;
        if (__ballot(mx > m_run + kRescale)) rise(mx);
    };
    auto finish = [&](int j, int kb) {
        bf16x8_t pf[4];
        f32x4_t rs = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s4 = 0; s4 < 4; ++s4) {
            f32x8_t pv8;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                pv8[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s4 >> 1][8 * (s4 & 1) + i], sl2, m_neg));
            pf[s4] = __builtin_convertvector(pv8, bf16x8_t);
            const u32x4_t w4 = __builtin_bit_cast(u32x4_t, pf[s4]);
            rs = add_weights(w4[0], w4[1], rs);
            rs = add_weights(w4[2], w4[3], rs);
        }
        l_run += rs[0];
        const int vbase = ((j + 1) & 3) * kPlace4;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            oacc[i & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v_frag(vbase, i), pf[i >> 2], oacc[i & 3], 0, 0, 0);
        if (j >= n_un) {
#pragma unroll
            for (int dt = 0; dt < 4; ++dt) {
                const int at = kWin ? 64 : vnan[j & 3][dt];
                if (kWin ? sees(vbits[j & 3][dt][0], vbits[j & 3][dt][1], qpos - 64 * kb, p.window, p.sinks - 64 * kb)
                         : at < 64 && 64 * kb + at <= qpos)
#pragma unroll
                    for (int e = 0; e < 16; ++e) oacc[dt][e] = __builtin_nanf("");
            }
        }
    };
    // ---- KV loop ----
    // Slot j computes the scores of block j + 1 and the PV product of block j.  The barrier of slot j stands
    // for: K of block j + 2 and V of block j + 1 are in LDS, and every wave has read K of block j + 1 and V
    // of block j - 1.
    auto mid_slot = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's writes
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    constexpr int kAhead = 4;   // K fragments in flight ahead of their MFMA
    constexpr int kVAhead = 3;  // V fragments
    bf16x8_t kf[16];
    // As in the bf16 kernel: the pins fix the order of the instructions in groups of one MFMA, a fragment read
    // and the stages of one weight, so no instruction of a group waits for another.
    auto fused = [&](f32x16_t(&sc)[2], f32x16_t(&sn)[2], auto place, int j) {
        constexpr int R = decltype(place)::value;
        constexpr int kK = ((R + 1) & 3) * kPlace4, kV = ((R + 1) & 3) * kPlace4, kN = ((R + 2) & 3) * kPlace4;
        bf16x8_t vf[16];
        uint32_t pw[16];  // packed weights, two per word
        float y[33], x[34];
        f32x4_t rs = {0.0f, 0.0f, 0.0f, 0.0f};
        auto weight = [&](int e) {  // e = 0 .. 34
            if (e >= 6 && (e & 3) == 2) rs = add_weights(pw[(e - 6) >> 1], pw[((e - 6) >> 1) + 1], rs);
            if (e >= 3 && (e & 1) && e < 34) {
                const f32x2_t pr = {x[e - 3], x[e - 2]};
                pw[(e - 3) >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pr, bf16x2_t));
            }
            if (e >= 1 && e <= 32) x[e - 1] = __builtin_amdgcn_exp2f(y[e - 1]);
            if (e < 32) y[e] = __builtin_fmaf(sc[e >> 4][e & 15], sl2, m_neg);
        };
        auto pf = [&](int s4) {
            const u32x4_t v = {pw[4 * s4], pw[4 * s4 + 1], pw[4 * s4 + 2], pw[4 * s4 + 3]};
            return __builtin_bit_cast(bf16x8_t, v);
        };
        const f32x16_t zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
        constexpr int kEarly = 6;  // groups with two stages
        int e = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i + kAhead < 16) kf[i + kAhead] = k_frag(kK, i + kAhead);
            if (i >= 16 - kVAhead) vf[i - 16 + kVAhead] = v_frag(kV, i - 16 + kVAhead);
            sn[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i], qf[i >> 1], i < 2 ? zero : sn[i & 1], 0, 0, 0);
            weight(e++);
            if (i < kEarly) weight(e++);
            asm volatile("" : "+v"(sn[i & 1]), "+v"(y[e - 1]), "+v"(x[e - 2]), "+v"(rs), "+v"(sc[e >> 4]) : : "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
        mid_slot();
        __builtin_amdgcn_s_setprio(1);
        settle(held, j + lead);
        float mx = kNegInf;
        bool up = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i + kVAhead < 16) vf[i + kVAhead] = v_frag(kV, i + kVAhead);
            if (i >= 16 - kAhead) kf[i - 16 + kAhead] = k_frag(kN, i - 16 + kAhead);
            oacc[i & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i], pf(i >> 2), oacc[i & 3], 0, 0, 0);
            if (e < 35) {
                weight(e++);
                if (e < 33) asm volatile("" : "+v"(y[e - 1]) : : "memory");
                if (e < 34) asm volatile("" : "+v"(x[e - 2]) : : "memory");
                asm volatile("" : "+v"(rs), "+v"(sc[1]) : : "memory");
            }
            if (i >= 4 && i < 12) {  // the row max of the next block's 32 scores
                const int v = i - 4;
#pragma unroll
                for (int q = 0; q < 4; ++q) mx = fmaxf(mx, sn[v >> 2][4 * (v & 3) + q]);
            }
            if (i == 12) mx = xor32_max(mx) * sl2;
            if (i == 13) up = __ballot(mx > m_run + kRescale) != 0;
            if (i == 14) l_run += rs[0];
            asm volatile("" : "+v"(oacc[i & 3]), "+v"(mx), "+v"(l_run) : : "memory");
            if (i >= 1 && i <= 10 && (i - 1) % 3 == 0) put(held, (R + 3) & 3, (i - 1) / 3);
            if (i == 11) held = fetch(j + lead + 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        if (up) rise(mx);
    };

    if (nblk > 0) {
        load_pages(0);
        Codes c0 = fetch(0), c1 = fetch(1);
        __syncthreads();  // vnan, late
        if (kTab) {
            n_un = nblk;
#pragma unroll
            for (int i = 0; i < kNW; ++i) n_un = min(n_un, late[i]);
            n_un = __builtin_amdgcn_readfirstlane(n_un);
        }
        settle(c0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) put(c0, is_v ? 1 : 0, i);
        if (!is_v) {
            settle(c1, 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) put(c1, 1, i);
            c1 = fetch(2);
        }
        held = c1;
        mid_slot();  // K of blocks 0 and 1, V of block 0
        scores(0);
        if (n_un == 0) mask(id_of(0));
        block_max();
        stage(-1);
        int j = 0;
        f32x16_t sn[2];
        if (j + 2 < n_un) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) kf[i] = k_frag(kPlace4, i);
        }
        // four slots a round: the ring places are constants and the scores change places without copies
        for (; j + 4 < n_un; j += 4) {
            fused(sc, sn, Int4C<0>{}, j);
            fused(sn, sc, Int4C<1>{}, j + 1);
            fused(sc, sn, Int4C<2>{}, j + 2);
            fused(sn, sc, Int4C<3>{}, j + 3);
        }
        if (j + 2 < n_un) {
            fused(sc, sn, Int4C<0>{}, j);
            fused(sn, sc, Int4C<1>{}, j + 1);
            j += 2;
        }
        for (; j < nblk; ++j) {  // the next block is masked, or there is none
            finish(j, id_of(j));
            if (j + 1 < nblk) {
                scores(((j + 1) & 3) * kPlace4);
                const int kb = id_of(j + 1);
                if (kWin ? j + 1 >= n_un : 64 * kb + 63 > first_q) mask(kb);
                block_max();
                mid_slot();
                // read last for block j - 1, written next for j + 3
                if (kWin) {
                    if (tid < 8) vbits[(j + 3) & 3][tid >> 1][tid & 1] = 0;
                } else if (tid < 4) {
                    vnan[(j + 3) & 3][tid] = 64;
                }
                stage(j);
            }
        }
    }

    // ---- epilogue (the row's place computed again: kept, it would take registers from the loop) ----
    l_run += __shfl_xor(l_run, 32, 64);
    int tid2 = threadIdx.x;
    asm volatile("" : "+v"(tid2));
    const int qrow = r0 + 32 * (tid2 >> 6) + (tid2 & 31);
    if (qrow < rows_total) {
        const int qt = qrow / G, qg = qrow - qt * G, h = (tid2 >> 5) & 1;
        // no key: zeros and -inf; a NaN sum stays
        const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
        const float lse2 = l_run == 0.0f ? kNegInf : (m_run == kNegInf ? 0.0f : m_run) + __log2f(l_run);
        const int hq = hk * G + qg;
        const int64_t prow = ((int64_t)split * (s.B * s.Hkv) + row) * rows_total + qrow;
        uint16_t* op = p.out.data + b * p.out.sb + (int64_t)qt * p.out.st + (int64_t)hq * p.out.sh;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int jq = 0; jq < 4; ++jq) {
                const int d0 = dt * 32 + 8 * jq + 4 * h;
                f32x4_t o4;
#pragma unroll
                for (int i = 0; i < 4; ++i) o4[i] = oacc[dt][4 * jq + i] * inv;
                if (nsplit == 1)
                    *reinterpret_cast<bf16x4_t*>(op + d0) = __builtin_convertvector(o4, bf16x4_t);
                else
                    *reinterpret_cast<f32x4_t*>(p.ws_o + prow * 128 + d0) = o4;
            }
        if (h == 0) {
            if (nsplit != 1)
                p.ws_lse[prow] = lse2;
            else if (p.lse)
                p.lse[((int64_t)b * s.Hq + hq) * s.Lq + qt] = lse2 * 0.69314718055994531f;
        }
    }
}

// What a merge reads of a launch (all of the attention's arguments, 3.6 KB, take the host 0.3 to 0.6 us longer).
struct Merge4Params {
    Shape s;
    SeqAddr out;
    float* lse;
    const float* ws_o;
    const float* ws_lse;
    int rows_total;
    int32_t sp[CA_MAX_BATCH];
};

// The joins weigh every split, those of weight 0 too: one without keys holds zeros, and a NaN sum stays NaN however
// little its split weighs, as it does within a split.

// Merge of many splits of few rows: four groups of 32 threads share a row, each a quarter of its splits, so
// that the partials' loads go out in one or two rounds where 32 threads take them in up to eight.
__global__ __launch_bounds__(128) void attn4_merge_kernel(Merge4Params p) {
    __shared__ f32x4_t part[3][32];
    const Shape& s = p.s;
    const int64_t rows_all = (int64_t)s.B * s.Hkv * p.rows_total;
    const int64_t gid = blockIdx.x;
    const int row = static_cast<int>(gid / p.rows_total);
    const int r = static_cast<int>(gid - (int64_t)row * p.rows_total);
    const int b = row / s.Hkv;
    const int hk = row - b * s.Hkv;
    const int nsplit = p.sp[b];
    if (nsplit == 1) return;  // the attention kernel wrote this request's rows
    const int lane = threadIdx.x & 31;
    const int grp = threadIdx.x >> 5;
    constexpr int kAtOnce = 8;
    // group grp's splits: grp, grp + 4, ...; their partials are loaded before the weights are known
    const float* wo = p.ws_o + gid * 128 + 4 * lane;
    f32x4_t o[kAtOnce];
    auto load = [&](int sp0) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int sp = sp0 + grp + 4 * i;
            o[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (sp < nsplit) o[i] = *reinterpret_cast<const f32x4_t*>(wo + (int64_t)sp * rows_all * 128);
        }
    };
    const float ls0 = lane < nsplit ? p.ws_lse[(int64_t)lane * rows_all + gid] : kNegInf;
    const float ls1 = lane + 32 < nsplit ? p.ws_lse[(int64_t)(lane + 32) * rows_all + gid] : kNegInf;
    load(0);
    float mx = fmaxf(ls0, ls1);
#pragma unroll
    for (int i = 16; i >= 1; i >>= 1) mx = fmaxf(mx, __shfl_xor(mx, i, 32));
    const float m_use = mx == kNegInf ? 0.0f : mx;
    const float w0 = __builtin_amdgcn_exp2f(ls0 - m_use), w1 = __builtin_amdgcn_exp2f(ls1 - m_use);
    float wsum = w0 + w1;
#pragma unroll
    for (int i = 16; i >= 1; i >>= 1) wsum += __shfl_xor(wsum, i, 32);
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int sp0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int sp = sp0 + grp + 4 * i;  // the same in all 32 threads
            const float wa = __shfl(w0, sp & 31, 32), wb = __shfl(w1, sp & 31, 32);
            const float wt = sp >= nsplit ? 0.0f : sp < 32 ? wa : wb;
            acc += wt * o[i];
        }
        sp0 += 4 * kAtOnce;
        if (sp0 >= nsplit) break;
        load(sp0);
    }
    if (grp > 0) part[grp - 1][lane] = acc;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int i = 0; i < 3; ++i) acc += part[i][lane];
    acc *= wsum == 0.0f ? 0.0f : 1.0f / wsum;  // no key: zeros and -inf; a NaN sum stays
    const int t = r / s.G;
    const int hq = hk * s.G + r - t * s.G;
    uint16_t* op = p.out.data + b * p.out.sb + (int64_t)t * p.out.st + (int64_t)hq * p.out.sh + 4 * lane;
    *reinterpret_cast<bf16x4_t*>(op) = __builtin_convertvector(acc, bf16x4_t);
    if (p.lse && lane == 0)
        p.lse[((int64_t)b * s.Hq + hq) * s.Lq + t] = wsum == 0.0f ? kNegInf : (m_use + __log2f(wsum)) * 0.69314718055994531f;
}

// Merge of few splits of many rows: 16 threads a row, 8 dims each.  Bound by memory (a row of a split is 516
// bytes, read once): 2 splits of 32768 rows (42 MB) 9.8 us, 12.1 in the bf16 kernels' merge.
__global__ __launch_bounds__(256) void attn4_merge_rows_kernel(Merge4Params p) {
    const Shape& s = p.s;
    const int64_t rows_all = (int64_t)s.B * s.Hkv * p.rows_total;
    const int64_t gid = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (gid >= rows_all) return;
    const int row = static_cast<int>(gid / p.rows_total);
    const int r = static_cast<int>(gid - (int64_t)row * p.rows_total);
    const int b = row / s.Hkv;
    const int hk = row - b * s.Hkv;
    const int nsplit = p.sp[b];
    if (nsplit == 1) return;  // the attention kernel wrote this request's rows
    const int d = 8 * (threadIdx.x & 15);
    const float* wo = p.ws_o + gid * 128 + d;
    constexpr int kAtOnce = 2;
    f32x4_t o[kAtOnce][2];
    auto load = [&](int sp0) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (sp0 + i < nsplit) {
                const f32x4_t* at = reinterpret_cast<const f32x4_t*>(wo + (int64_t)(sp0 + i) * rows_all * 128);
                o[i][0] = __builtin_nontemporal_load(at);
                o[i][1] = __builtin_nontemporal_load(at + 1);
            }
        }
    };
    load(0);
    float mx = kNegInf;
    for (int sp = 0; sp < nsplit; ++sp) mx = fmaxf(mx, p.ws_lse[(int64_t)sp * rows_all + gid]);
    const float m_use = mx == kNegInf ? 0.0f : mx;
    f32x4_t acc[2] = {f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}};
    float wsum = 0.0f;
    for (int sp0 = 0;;) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if (sp0 + i < nsplit) {
                const float wt = __builtin_amdgcn_exp2f(p.ws_lse[(int64_t)(sp0 + i) * rows_all + gid] - m_use);
                wsum += wt;
                acc[0] += wt * o[i][0];
                acc[1] += wt * o[i][1];
            }
        }
        sp0 += kAtOnce;
        if (sp0 >= nsplit) break;
        load(sp0);
    }
    const float inv = wsum == 0.0f ? 0.0f : 1.0f / wsum;  // no key: zeros and -inf; a NaN sum stays
    const int t = r / s.G;
    const int hq = hk * s.G + r - t * s.G;
    uint16_t* op = p.out.data + b * p.out.sb + (int64_t)t * p.out.st + (int64_t)hq * p.out.sh + d;
    f32x8_t v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = acc[i >> 2][i & 3] * inv;
    *reinterpret_cast<bf16x8_t*>(op) = __builtin_convertvector(v, bf16x8_t);
    if (p.lse && d == 0)
        p.lse[((int64_t)b * s.Hq + hq) * s.Lq + t] = wsum == 0.0f ? kNegInf : (m_use + __log2f(wsum)) * 0.69314718055994531f;
}

}  // namespace

// Which kernel: tiles of 16 or 32 rows whose waves take blocks on their own, or of 256 rows whose waves share
// them.  A workgroup takes 0.9 us for 32 rows x four blocks and 1.3 us for 256 x one, so the small tiles do
// less up to 160 rows, and beyond do 1.4 times the work but start and end 6 to 12 us earlier, need no merge
// where their tiles alone fill the CUs, and waste fewer rows.  They win up to 12 blocks of 256 rows for every
// CU (all blocks counted; 32 Q / 8 KV heads, small tiles and large): 64 queries over 16 + 1 blocks 13.4, 21.3 us;
// 256 over 8 + 4 11.7, 26.8; 256 over 64 + 4 (8.5 blocks a CU) 26.5, 41; 256 over 256 + 4 (32.5) 78.4, 75.3,
// with 30 % kept 32.7, 42.5; 512 over 128 + 8 (34) 87.5, 77.2, with 30 % kept 43.6, 43.0.  (Not always: 300 over
// 40 + 5 with 28 / 4 heads, 6.3 blocks a CU, 39.3, 33.3.)
// Under a window lists are short and tiles many: a round of 256 small tiles takes 7.3 us and 0.3 us a block, tiles of 256 rows
// what they take of bf16 pages and 5 us (2021 queries under 71, 24 Q / 6 KV heads, small and large, 51.7, 22.7 us; 397 of 5
// requests under 131, 32 / 8, 77.7, 52.6; 1000 under 1024, 8 / 8, 14.4, 39.1; 512 under 4096, 32 / 8, 54.6, 55.9).
AttnTiling attn4_tiling(const Shape& s, const PastBlocks& pb, const int32_t* kv_len, int window, int sinks) {
    const bool dense = kv_len != nullptr;
    const int rows = s.Lq * s.G;
    int32_t qpos0[CA_MAX_BATCH], nkb[CA_MAX_BATCH];
    attn_positions(s, pb, kv_len, qpos0, nkb);
    bool small = rows <= 160;
    if (window == 0) {
        double blocks = 0.0;  // of 256 rows
        for (int b = 0; b < s.B; ++b) blocks += (double)s.Hkv * ((rows + kBM - 1) / kBM) * nkb[b];
        small = small || blocks <= 12.0 * 256;
    } else if (!small) {
        int most = 1, most_small = 1, splits;
        for (int b = 0; b < s.B; ++b) {
            most = max(most, attn_window_blocks(s, kBM, qpos0[b], window, sinks));
            most_small = max(most_small, attn_window_blocks(s, 32, qpos0[b], window, sinks));
        }
        const double items = (double)s.B * s.Hkv * ((rows + 31) / 32);
        const int c = max(1, static_cast<int>(256 / items));
        const double us = ceil(items * c / 256) * (7.3 + 0.3 * ((most_small + c - 1) / c)) + (c > 1 ? 4.0 + 1.9e-4 * s.B * s.Hkv * rows * c : 0.0);
        small = us < attn_window_us(s, kBM, most, kMaxDecodeSplits, &splits) + 5.0;
    }
    if (small)
        return AttnTiling{dense && rows <= 16 ? 16 : 32, true, true, !dense, 0, dense ? 32 : kMaxPrefillSplits};
    AttnTiling t = attn_tiling(s, dense, false);
    t.steps = true;
    t.window = window > 0;
    return t;
}

hipError_t launch_attn4(const AttnArgs& a, const Kv4Addr& k, const Kv4Addr& v, hipStream_t stream) {
    Attn4Params p;
    SplitPlan plan;
    const AttnTiling tiling = attn4_tiling(a.s, a.pb, a.kv_len, a.window, a.sinks);
    attn_fill(a, tiling, &p.a, &plan);
    p.a.ws_unsplit = nullptr;  // a launch with splits keeps them
    p.k = k;
    p.v = v;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(plan.per_xcd * 8), dim3(kNW * 64), 0, stream, p); };
    static_assert(kNW == kWaves4, "one workgroup size");
    if (a.window > 0)
        tiling.tile_rows == 16   ? launch(attn4_decode_kernel<1, false, kLoadsStreamed, true>)
        : tiling.tile_rows == 32 ? launch(attn4_decode_kernel<2, false, kLoadsKept, true>)
                                 : launch(attn4_fwd_kernel<false, true>);
    else if (a.table)
        tiling.streams ? launch(attn4_decode_kernel<2, true, kLoadsKept>) : launch(attn4_fwd_kernel<true>);
    else if (tiling.tile_rows == 16)
        a.s.B > 1 ? launch(attn4_decode_kernel<1, false, kLoadsStreamedUnshared>)
                  : launch(attn4_decode_kernel<1, false, kLoadsStreamed>);
    else if (tiling.tile_rows == 32)
        launch(attn4_decode_kernel<2, false, kLoadsKept>);
    else
        launch(attn4_fwd_kernel<false>);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || plan.max <= 1) return e;
    const int64_t rows_all = (int64_t)a.s.B * a.s.Hkv * p.a.rows_total;
    // By rows and splits, with 128, 16 and (the bf16 kernels' merge) 32 threads a row: 32 splits of 32 rows 4.0,
    // 22.1 us, 16 of 2048 5.4, 10.8; 2 of 32768 32.9, 10.0, 12.1; 12 of 4800 in a launch of 68.5 us with 32 74.1
    // with 16.
    if (rows_all > 4096 && plan.max > 4) return launch_attn_merge(p.a, true, stream);
    Merge4Params m{a.s, p.a.out, p.a.lse, p.a.ws_o, p.a.ws_lse, p.a.rows_total, {}};
    for (int b = 0; b < CA_MAX_BATCH; ++b) m.sp[b] = p.a.sp[b];
    if (rows_all <= 4096)
        hipLaunchKernelGGL(attn4_merge_kernel, dim3(static_cast<unsigned>(rows_all)), dim3(128), 0, stream, m);
    else
        hipLaunchKernelGGL(attn4_merge_rows_kernel, dim3(static_cast<unsigned>((rows_all + 15) / 16)), dim3(256), 0, stream, m);
    return hipGetLastError();
}

}  // namespace ca
