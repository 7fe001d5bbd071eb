// The pages of a KV cache: appends to and reads from pages held in 4 bits (the format is in ca_kv4.h),
// and copies of whole pages of any kind.  All are bound by memory, and by the launch where they are small.

#include "ca_kernels.h"
#include "ca_kv4.h"

namespace ca {
namespace {

typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4p_t __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------
// Append: a thread quantises 8 dims of a token of K and of V, so the 4 lanes of a quad share a group's
// scale and 16 lanes hold a token of a head.  Rows (b, t, h) run over heads first, as the new tokens
// lie in memory.  The codes go through v_cvt_scalef32_pk_fp4_bf16, which rounds to nearest even.
struct Kv4Rows {
    int L, H;
    int64_t rows;  // B * L * H
    int32_t start[CA_MAX_BATCH];
};

struct Append4Params {
    Kv4Rows r;
    SeqAddr k_new, v_new;
    Kv4Addr k, v;
};

__device__ __forceinline__ uint32_t max_quad(uint32_t a) {
    a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0xb1, 0xf, 0xf, true));  // quad_perm [1, 0, 3, 2]
    return max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x4e, 0xf, 0xf, true));  // quad_perm [2, 3, 0, 1]
}

__device__ __forceinline__ uint32_t encode8(u16x8_t x, uint32_t* byte) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = max(a, (uint32_t)x[i] & 0x7fffu);
    *byte = scale_byte(max_quad(a));
    if (*byte == kScaleNan) return 0;
    const float s = __uint_as_float(*byte << 23);
    typedef __bf16 bf16x8v_t __attribute__((ext_vector_type(8)));
    const bf16x8v_t v = __builtin_bit_cast(bf16x8v_t, x);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_shufflevector(v, v, 0, 1), s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_shufflevector(v, v, 2, 3), s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_shufflevector(v, v, 4, 5), s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_shufflevector(v, v, 6, 7), s, 3);
}

// (b, t, h) and the position of row i
struct RowAt {
    int b, t, h, pos;
};
__device__ __forceinline__ RowAt row_at(const Kv4Rows& r, int64_t i) {
    const uint32_t bt = static_cast<uint32_t>(i) / static_cast<uint32_t>(r.H);
    RowAt a;
    a.h = static_cast<int>(static_cast<uint32_t>(i) - bt * r.H);
    a.b = bt / static_cast<uint32_t>(r.L);
    a.t = bt - a.b * r.L;
    a.pos = r.start[a.b] + a.t;
    return a;
}

__global__ __launch_bounds__(256) void append4_kernel(Append4Params p) {
    const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (i >= p.r.rows) return;
    const int m = threadIdx.x & 15;  // dims 8 m .. 8 m + 7
    const RowAt a = row_at(p.r, i);
    const int64_t row = (int64_t)a.b * p.r.H + a.h;
    const int kb = a.pos >> 6, t = a.pos & 63;
    const u16x8_t kx = *reinterpret_cast<const u16x8_t*>(p.k_new.data + a.b * p.k_new.sb + a.t * p.k_new.st +
                                                         a.h * p.k_new.sh + 8 * m);
    const u16x8_t vx = *reinterpret_cast<const u16x8_t*>(p.v_new.data + a.b * p.v_new.sb + a.t * p.v_new.st +
                                                         a.h * p.v_new.sh + 8 * m);
    // a page outside the pool is no page: nothing is written for it
    const int32_t kp = p.k.page_table[row * p.k.pts + kb], vp = p.v.page_table[row * p.v.pts + kb];
    uint32_t kbyte, vbyte;
    const uint32_t kc = encode8(kx, &kbyte), vc = encode8(vx, &vbyte);
    if (kp >= 0 && kp <= p.k.max_page) {
        uint8_t* page = p.k.data + kp * p.k.stride;
        *reinterpret_cast<uint32_t*>(page + k4_code(t, 8 * m)) = kc;
        if ((m & 3) == 0) page[k4_scale(t, m >> 2)] = static_cast<uint8_t>(kbyte);
    }
    if (vp >= 0 && vp <= p.v.max_page) {
        uint8_t* page = p.v.data + vp * p.v.stride;
        *reinterpret_cast<uint32_t*>(page + v4_code(t, 8 * m)) = vc;
        if ((m & 3) == 0) page[v4_scale(t, m >> 2)] = static_cast<uint8_t>(vbyte);
    }
}

// ---------------------------------------------------------------------------------------
// Read back: [B, H, L, 128] bf16 values of tokens start[b] .. start[b] + L - 1, 8 dims a thread.
struct Gather4Params {
    Kv4Rows r;
    Kv4Addr k, v;
    uint16_t* k_out;  // nullable, as v_out
    uint16_t* v_out;
};

__device__ __forceinline__ u32x4p_t decode8(const uint8_t* page, int code, int scale) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(page + code);
    const float s = scale_of<0>(page[scale]);
    return u32x4p_t{decode2<0>(w, s), decode2<1>(w, s), decode2<2>(w, s), decode2<3>(w, s)};
}

__global__ __launch_bounds__(256) void gather4_kernel(Gather4Params p) {
    const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (i >= p.r.rows) return;
    const int m = threadIdx.x & 15;
    // rows (b, h, t) here: the output's order
    const uint32_t row = static_cast<uint32_t>(i) / static_cast<uint32_t>(p.r.L);
    const int t0 = static_cast<int>(static_cast<uint32_t>(i) - row * p.r.L);
    const int b = row / static_cast<uint32_t>(p.r.H);
    const int pos = p.r.start[b] + t0;
    const int kb = pos >> 6, t = pos & 63;
    if (p.k_out != nullptr) {
        const int64_t kp = clamp_page(p.k.page_table[row * p.k.pts + kb], p.k.max_page);
        const u32x4p_t kx = decode8(p.k.data + kp * p.k.stride, k4_code(t, 8 * m), k4_scale(t, m >> 2));
        *reinterpret_cast<u32x4p_t*>(p.k_out + i * kD + 8 * m) = kx;
    }
    if (p.v_out != nullptr) {
        const int64_t vp = clamp_page(p.v.page_table[row * p.v.pts + kb], p.v.max_page);
        const u32x4p_t vx = decode8(p.v.data + vp * p.v.stride, v4_code(t, 8 * m), v4_scale(t, m >> 2));
        *reinterpret_cast<u32x4p_t*>(p.v_out + i * kD + 8 * m) = vx;
    }
}

// ---------------------------------------------------------------------------------------
// Copies of pages.  The ids of up to kCopyPairs pages travel in the launch's arguments: no upload, nothing
// to wait for, and a captured graph holds them.  (Up to kFewPairs in fewer arguments: a call for 32 pages 9.5
// us with 3.8 KB of them, 9.2 so.)  More are read from device memory where the caller has put them there,
// else copied in several launches.  A thread moves 16 bytes.  Bound by memory: 9001 4-bit pages (157 MB read
// and written) of two pools 36.4 us with four such pieces a thread, 30.2 with one and stores past the caches
// (5.2 TB/s); 2300 bf16 pages (151 MB) 34.9 and 26.1.  Few pages, such as those that a decode step is about
// to read, are stored to stay in the caches.
constexpr int kCopyPairs = 448;  // 3.5 KB of the 4 KB of arguments
constexpr int kFewPairs = 64;
constexpr int kCopyThreads = 256;

template <int kPairs>  // 0: by id
struct CopyParams {
    PagePool pool[CA_MAX_POOLS];
    const int32_t* ids;  // by id: n sources, then n destinations
    uint32_t pages;      // by id: nothing is copied from or to an id that is not below
    int n;
    int32_t src[kPairs > 0 ? kPairs : 1];
    int32_t dst[kPairs > 0 ? kPairs : 1];
};
static_assert(sizeof(CopyParams<kCopyPairs>) <= 4096, "the arguments of a launch");

template <int kPairs>
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(CopyParams<kPairs> p) {
    constexpr bool kById = kPairs == 0;
    const PagePool pool = p.pool[blockIdx.y];
    const uint32_t units = static_cast<uint32_t>(pool.bytes >> 4);
    // the workgroup's first unit (64 bits) by uniform arithmetic, the thread's from there
    const uint64_t first = (uint64_t)blockIdx.x * kCopyThreads;
    const uint64_t pair0 = first / units;
    const uint32_t u = static_cast<uint32_t>(first - pair0 * units) + threadIdx.x;
    const uint32_t k = u / units;
    const uint64_t pair = pair0 + k;
    if (pair >= (uint64_t)p.n) return;
    const int64_t off = (int64_t)(u - k * units) * 16;
    const int32_t src = kById ? p.ids[pair] : p.src[pair];
    const int32_t dst = kById ? p.ids[p.n + pair] : p.dst[pair];
    if (kById && (static_cast<uint32_t>(src) >= p.pages || static_cast<uint32_t>(dst) >= p.pages)) return;
    const u32x4p_t v = *reinterpret_cast<const u32x4p_t*>(pool.data + src * pool.stride + off);
    u32x4p_t* to = reinterpret_cast<u32x4p_t*>(pool.data + dst * pool.stride + off);
    if (kById)
        __builtin_nontemporal_store(v, to);
    else
        *to = v;
}

Kv4Rows rows_of(int B, int L, int H, const int32_t* start) {
    Kv4Rows r;
    r.L = L;
    r.H = H;
    r.rows = (int64_t)B * L * H;
    for (int b = 0; b < CA_MAX_BATCH; ++b) r.start[b] = b < B ? start[b] : 0;
    return r;
}

}  // namespace

hipError_t launch_append4(int B, int L, int H, const int32_t* start, const SeqAddr& k_new, const SeqAddr& v_new,
                          const Kv4Addr& k, const Kv4Addr& v, hipStream_t stream) {
    Append4Params p{rows_of(B, L, H, start), k_new, v_new, k, v};
    hipLaunchKernelGGL(append4_kernel, dim3(static_cast<unsigned>((p.r.rows + 15) / 16)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_gather4(int B, int L, int H, const int32_t* start, const Kv4Addr* k, const Kv4Addr* v,
                          uint16_t* k_out, uint16_t* v_out, hipStream_t stream) {
    const Kv4Addr none{};
    Gather4Params p{rows_of(B, L, H, start), k != nullptr ? *k : none, v != nullptr ? *v : none,
                    k != nullptr ? k_out : nullptr, v != nullptr ? v_out : nullptr};
    hipLaunchKernelGGL(gather4_kernel, dim3(static_cast<unsigned>((p.r.rows + 15) / 16)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_copy_pages(const PagePool* pools, int n_pools, const int32_t* src, const int32_t* dst, int n,
                             const int32_t* ids, uint32_t pages, hipStream_t stream) {
    int64_t most = 0;
    for (int i = 0; i < n_pools; ++i)
        if (pools[i].bytes > most) most = pools[i].bytes;
    auto launch = [&](auto params, auto kernel, int at, int count) {
        for (int i = 0; i < n_pools; ++i) params.pool[i] = pools[i];
        params.ids = ids;
        params.pages = pages;
        params.n = count;
        if (sizeof(params.src) > sizeof(int32_t)) {
            for (int i = 0; i < count; ++i) {
                params.src[i] = src[at + i];
                params.dst[i] = dst[at + i];
            }
        }
        const int64_t blocks = ((most >> 4) * count + kCopyThreads - 1) / kCopyThreads;
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks), n_pools), dim3(kCopyThreads), 0, stream, params);
        return hipGetLastError();
    };
    if (n <= kFewPairs) return launch(CopyParams<kFewPairs>(), copy_pages_kernel<kFewPairs>, 0, n);
    if (ids != nullptr && n > kCopyPairs) return launch(CopyParams<0>(), copy_pages_kernel<0>, 0, n);
    for (int at = 0; at < n; at += kCopyPairs) {
        const hipError_t e = launch(CopyParams<kCopyPairs>(), copy_pages_kernel<kCopyPairs>, at, min(kCopyPairs, n - at));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace ca
