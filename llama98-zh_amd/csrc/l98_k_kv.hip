// Rows into and out of the paged key-value cache, and copies of its pages.
//
// A Q8 row is the engine's kind: groups of 32, scale max|x| / 127, codes
// rounded half to even (d_q8_round), stored as code + 128 in the order that
// the matrix instructions of the attention read (include/llama98_hip.h).  All three kernels only move bytes: their bound is HBM.
#include <limits.h>

#include "l98_devmath.h"
#include "l98_kv.h"

#define KV_THREADS 256

template <class T> __device__ __forceinline__ float kv_f32(T x) { return (float)x; }

// E consecutive elements at x; vec: x is aligned to the E elements' size
// (at most 16 bytes a load).
template <class T, int E>
__device__ __forceinline__ void kv_load(const T *x, bool vec, float *o) {
    constexpr int N = 16 / sizeof(T) < E ? 16 / sizeof(T) : E;     // elements of a load
    typedef T vt __attribute__((ext_vector_type(N)));
    if (vec) {
#pragma unroll
        for (int i = 0; i < E; i += N) {
            const vt t = *reinterpret_cast<const vt *>(x + i);
#pragma unroll
            for (int u = 0; u < N; u++) o[i + u] = (float)t[u];
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i++) o[i] = (float)x[i];
    }
}
template <class T, int E>
__device__ __forceinline__ void kv_store(T *x, bool vec, const float *v) {
    constexpr int N = 16 / sizeof(T) < E ? 16 / sizeof(T) : E;
    typedef T vt __attribute__((ext_vector_type(N)));
    if (vec) {
#pragma unroll
        for (int i = 0; i < E; i += N) {
            vt t;
#pragma unroll
            for (int u = 0; u < N; u++) t[u] = (T)v[i + u];
            *reinterpret_cast<vt *>(x + i) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; i++) x[i] = (T)v[i];
    }
}

// A row of one head of K or V belongs to 16 lanes, E = D / 16 elements each:
// of K (and of a bf16 row) the lane's own consecutive dimensions, of a Q8 V
// row the dimensions t * 16 + lane, so that either way a lane's E codes lie
// together in the page.
struct KvUnit {
    int lane, which, head, row;          // which: 0 K, 1 V; row: of the arrays, -1 for none
    const unsigned char *page;           // null: the position has no page
    int off;                             // its row in the page
};
__device__ __forceinline__ KvUnit kv_unit(const KvPages &p, const KvSeqs &b) {
    KvUnit u;
    u.lane = threadIdx.x & 15;
    const KvSeq s = kv_seq(b, blockIdx.y, p.shift);
    const long long i = (long long)blockIdx.x * (KV_THREADS / 16) + (threadIdx.x >> 4);
    const int per = 2 * p.hk;
    const int j = (int)(i / per), w = (int)(i % per);
    u.which = w & 1;
    u.head = w >> 1;
    const int r = s.r0 + j, pos = s.pos0 + j;
    u.row = j < s.n && j < b.max_rows && (unsigned)r < (unsigned)b.n_rows ? r : -1;
    u.page = nullptr;
    u.off = 0;
    if (u.row >= 0 && pos >= 0 && pos < s.len) {
        const int id = b.table[blockIdx.y * b.stride + (pos >> p.shift)];
        if ((unsigned)id < (unsigned)p.n_pages) u.page = kv_page(p, id);
        u.off = pos & ((1 << p.shift) - 1);
    }
    return u;
}
// offsets in a page's block: a row's numbers (es bytes each), and its scale of group g
template <int D>
__device__ __forceinline__ long long kv_at(const KvPages &p, const KvUnit &u, int es) {
    return ((((long long)u.which * p.hk + u.head) << p.shift) + u.off) * D * es;
}
template <int D>
__device__ __forceinline__ long long kv_scale_at(const KvPages &p, const KvUnit &u, int g) {
    return (((long long)2 * p.hk << p.shift) * D) +
           ((((((long long)u.which * p.hk + u.head) * (D / 32)) + g) << p.shift) + u.off) * 4;
}

// q8_scale_inv with the factor 127 * (1 / max) instead of 127 / max: what a
// torch program that fills pages itself gets from 127.0 / max.  (Some of the
// factors differ in the last bit, and with them about one code in a million
// by one.)
__device__ __forceinline__ void kv_scale_inv(float amax, float *sg, float *inv) {
    float unused;
    q8_scale_inv(amax, sg, &unused);
    *inv = unused == 0.0f ? 0.0f : 127.0f * (1.0f / amax);
}

__device__ __forceinline__ uint32_t max_over(uint32_t v, int lanes) {    // over aligned groups of `lanes`
    for (int o = 1; o < lanes; o <<= 1) {
        const uint32_t y = __shfl_xor(v, o);
        v = y > v ? y : v;
    }
    return v;
}

template <class T, int D, bool Q8>
__global__ __launch_bounds__(KV_THREADS) void k_kv_append(KvPages p, KvSeqs b, KvRows k, KvRows v, int vec) {
    constexpr int E = D / 16;
    const KvUnit u = kv_unit(p, b);
    const KvRows &src = u.which ? v : k;
    float x[E];
#pragma unroll
    for (int i = 0; i < E; i++) x[i] = 0.0f;
    const bool live = u.page != nullptr;
    const T *s = (const T *)src.p + (live ? u.row * src.row + u.head * src.head : 0);
    if (!Q8) {
        if (!live) return;
        kv_load<T, E>(s + u.lane * E, vec, x);
        kv_store<__bf16, E>((__bf16 *)(u.page + kv_at<D>(p, u, 2)) + u.lane * E, true, x);
        return;
    }
    // the shuffles below take every lane of the wave
    if (live) {
        if (u.which == 0) {
            kv_load<T, E>(s + u.lane * E, vec, x);
        } else {
#pragma unroll
            for (int t = 0; t < E; t++) x[t] = (float)s[t * 16 + u.lane];
        }
    }
    uint32_t c[(E + 3) / 4] = {};
    float sg, inv;
    uint32_t am[E / 2];
#pragma unroll
    for (int g = 0; g < E / 2; g++) {
        const uint32_t a = u_from_f(x[2 * g]) & 0x7FFFFFFFu, e = u_from_f(x[2 * g + 1]) & 0x7FFFFFFFu;
        am[g] = a > e ? a : e;
    }
    if (u.which == 0) {
        uint32_t m = am[0];
#pragma unroll
        for (int g = 1; g < E / 2; g++) m = am[g] > m ? am[g] : m;
        m = max_over(m, 32 / E);
#pragma unroll
        for (int g = 0; g < E / 2; g++) am[g] = m;
    } else {
#pragma unroll
        for (int g = 0; g < E / 2; g++) am[g] = max_over(am[g], 16);
    }
#pragma unroll
    for (int g = 0; g < E / 2; g++) {
        kv_scale_inv(f_from_u(am[g]), &sg, &inv);
        if (live && (u.which == 0 ? g == 0 && u.lane % (32 / E) == 0 : u.lane == 0))
            *(float *)(u.page + kv_scale_at<D>(p, u, u.which == 0 ? u.lane * E / 32 : g)) = sg;
#pragma unroll
        for (int i = 2 * g; i < 2 * g + 2; i++) {
            int qi = d_q8_round(x[i] * inv);
            qi = qi > 127 ? 127 : qi;
            qi = qi < -127 ? -127 : qi;
            c[i / 4] |= (uint32_t)(qi + 128) << (8 * (i & 3));
        }
    }
    if (!live) return;
    // K: dimension c*32 + h*8 + j lies at byte h*(D/4) + c*8 + j
    const int d0 = u.lane * E;
    const int at = u.which ? d0 : ((d0 & 31) >> 3) * (D / 4) + (d0 >> 5) * 8 + (d0 & 7);
    unsigned char *o = const_cast<unsigned char *>(u.page) + kv_at<D>(p, u, 1) + at;
    if (E == 8) *(uint2 *)o = make_uint2(c[0], c[E == 8 ? 1 : 0]);
    else if (E == 4) *(uint32_t *)o = c[0];
    else *(uint16_t *)o = (uint16_t)c[0];
}

template <class T, int D, bool Q8>
__global__ __launch_bounds__(KV_THREADS) void k_kv_read(KvPages p, KvSeqs b, KvRows k, KvRows v, int vec) {
    constexpr int E = D / 16;
    const KvUnit u = kv_unit(p, b);
    if (u.row < 0) return;
    const KvRows &dst = u.which ? v : k;
    T *o = (T *)dst.p + (u.row * dst.row + u.head * dst.head);
    float x[E];
#pragma unroll
    for (int i = 0; i < E; i++) x[i] = 0.0f;
    if (!Q8) {
        if (u.page) kv_load<__bf16, E>((const __bf16 *)(u.page + kv_at<D>(p, u, 2)) + u.lane * E, true, x);
        kv_store<T, E>(o + u.lane * E, vec, x);
        return;
    }
    if (u.page) {
        const int d0 = u.lane * E;
        const int at = u.which ? d0 : ((d0 & 31) >> 3) * (D / 4) + (d0 >> 5) * 8 + (d0 & 7);
        const unsigned char *c = u.page + kv_at<D>(p, u, 1) + at;
        uint32_t w[(E + 3) / 4];
        if (E == 8) { const uint2 t = *(const uint2 *)c; w[0] = t.x; w[E == 8 ? 1 : 0] = t.y; }
        else if (E == 4) w[0] = *(const uint32_t *)c;
        else w[0] = *(const uint16_t *)c;
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int g = u.which ? i / 2 : d0 / 32;
            const float sg = *(const float *)(u.page + kv_scale_at<D>(p, u, g));
            x[i] = (float)((int)((w[i / 4] >> (8 * (i & 3))) & 255u) - 128) * sg;
        }
    }
    if (u.which == 0) {
        kv_store<T, E>(o + u.lane * E, vec, x);
    } else {
#pragma unroll
        for (int t = 0; t < E; t++) o[t * 16 + u.lane] = (T)x[t];
    }
}

// Whole pages, 16 bytes a lane and load, KV_COPY_UNROLL loads in flight (the
// index clamped instead of a branch around each load).
#define KV_COPY_UNROLL 4
template <int N>
__global__ __launch_bounds__(KV_THREADS) void k_kv_copy(unsigned char *data, long long page_bytes, KvMoves<N> m) {
    typedef uint32_t v4 __attribute__((ext_vector_type(4)));
    const v4 *s = (const v4 *)(data + m.src[blockIdx.y] * page_bytes);
    v4 *d = (v4 *)(data + m.dst[blockIdx.y] * page_bytes);
    const long long n = page_bytes / 16, i0 = (long long)blockIdx.x * (KV_THREADS * KV_COPY_UNROLL) + threadIdx.x;
    v4 x[KV_COPY_UNROLL];
#pragma unroll
    for (int u = 0; u < KV_COPY_UNROLL; u++) x[u] = s[i0 + u * KV_THREADS < n ? i0 + u * KV_THREADS : n - 1];
#pragma unroll
    for (int u = 0; u < KV_COPY_UNROLL; u++)
        if (i0 + u * KV_THREADS < n) d[i0 + u * KV_THREADS] = x[u];
}

// ---------------------------------------------------------- host glue ---

// every row's and head's run of `unit` elements can be loaded as a vector
static int kv_vec(const KvRows &r, int es, int unit) {
    const int b = es * unit < 16 ? es * unit : 16;
    return ((uintptr_t)r.p % b) == 0 && (r.row * es) % b == 0 && (r.head * es) % b == 0;
}

#define KV_ROWS_LAUNCH(K, T, DD, QQ)                                                                       \
    do {                                                                                                   \
        const int vec = kv_vec(k, sizeof(T), DD / 16) && kv_vec(v, sizeof(T), DD / 16);                    \
        hipLaunchKernelGGL((K<T, DD, QQ>), grid, dim3(KV_THREADS), 0, st, p, b, k, v, vec);                \
    } while (0)
#define KV_ROWS_DISPATCH(K)                                                                                \
    const long long units = (long long)b.max_rows * p.hk * 2;                                              \
    const long long blocks = (units + KV_THREADS / 16 - 1) / (KV_THREADS / 16);                            \
    if (blocks > INT_MAX) return -1;                                                                       \
    const dim3 grid((unsigned)blocks, b.n_seq);                                                            \
    if (p.d == 32) KV_ROWS_D(K, 32);                                                                       \
    else if (p.d == 64) KV_ROWS_D(K, 64);                                                                  \
    else if (p.d == 128) KV_ROWS_D(K, 128);                                                                \
    else return -1;                                                                                        \
    return (int)hipGetLastError()
#define KV_ROWS_D(K, DD)                                                                                   \
    do {                                                                                                   \
        if (bf16) { if (q8) KV_ROWS_LAUNCH(K, __bf16, DD, true); else KV_ROWS_LAUNCH(K, __bf16, DD, false); } \
        else { if (q8) KV_ROWS_LAUNCH(K, float, DD, true); else KV_ROWS_LAUNCH(K, float, DD, false); }     \
    } while (0)

extern "C" int l98k_kv_append(const KvPages &p, int q8, const KvSeqs &b, const KvRows &k, const KvRows &v, int bf16,
                              hipStream_t st) {
    KV_ROWS_DISPATCH(k_kv_append);
}

extern "C" int l98k_kv_read(const KvPages &p, int q8, const KvSeqs &b, const KvRows &k, const KvRows &v, int bf16,
                            hipStream_t st) {
    KV_ROWS_DISPATCH(k_kv_read);
}

template <int N>
static int copy_some(unsigned char *data, long long page_bytes, const int *src, const int *dst, int n, hipStream_t st) {
    const long long per = (long long)KV_THREADS * KV_COPY_UNROLL * 16;
    KvMoves<N> m = {};
    for (int u = 0; u < n; u++) { m.src[u] = src[u]; m.dst[u] = dst[u]; }
    hipLaunchKernelGGL((k_kv_copy<N>), dim3((unsigned)((page_bytes + per - 1) / per), n), dim3(KV_THREADS), 0, st, data,
                       page_bytes, m);
    return (int)hipGetLastError();
}
// A launch's arguments hold at most 4 KB; a fork's few copies take a launch of
// few arguments.
extern "C" int l98k_kv_copy(unsigned char *data, long long page_bytes, const int *src, const int *dst, int n,
                            hipStream_t st) {
    if (n <= 16) return copy_some<16>(data, page_bytes, src, dst, n, st);
    for (int i = 0; i < n; i += 448) {
        const int rc = copy_some<448>(data, page_bytes, src + i, dst + i, n - i < 448 ? n - i : 448, st);
        if (rc) return rc;
    }
    return 0;
}
