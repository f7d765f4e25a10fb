// Rows into and out of the paged key-value cache, and copies of its pages.
//
// A Q8 row is the engine's kind: groups of 32, scale max|x| / 127, codes
// rounded half to even (d_q8_round), stored as code + 128 in the order that
// the matrix instructions of the attention read (include/llama98_hip.h).  All three kernels only move bytes: their bound is HBM.
#include <limits.h>

#include "l98_devmath.h"
#include "l98_kv.h"

#define KV_THREADS 256
// Four units a lane where one each would be more blocks than the chip holds at
// once, 8 on each of 256 CUs.
#define KV_ALL 2048

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

// A piece, the row of one head of K or V, belongs to 16 lanes, E = D / 16
// consecutive dimensions each.  A Q8 piece's codes are made that way too, and
// V's then change lanes through LDS: in the page lane n's E codes are the
// dimensions t * 16 + n.  A block's 16 groups of lanes take 16 rows, or with
// fewer rows several pieces of each, and U pieces one after the other whose
// loads are in flight together: a page has a head's rows side by side and of
// their scales a group's, and what a row needs (its page, its places) is found
// once.  (Appending 19,000 bf16 rows of 4 heads of 128, 61 MB: 17 us and reading
// them 13, where a large copy would take 12.  With each piece on its own 24 and
// 16: that is bound by the instructions that find its places.  With V read from
// the caller's rows in the page's order, two bytes a load, appending took 32.)
struct KvRow {
    int row;                             // of the arrays, -1 for none
    unsigned char *page;                 // null: the position has no page
    int off;                             // its row in the page
    int w0, step;                        // its first piece, and from one to the next; K's heads come before V's
};
// lr: log2 of a block's rows; parts: blocks of a row
__device__ __forceinline__ KvRow kv_row(const KvPages &p, const KvSeqs &b, int lr, unsigned parts, int U) {
    KvRow u;
    const KvSeq s = kv_seq(b, blockIdx.y, p.shift);
    const unsigned group = blockIdx.x / parts, slot = threadIdx.x >> 4;
    const long long j = ((long long)group << lr) + (slot & ((1u << lr) - 1));
    u.step = KV_THREADS / 16 >> lr;
    u.w0 = (int)(blockIdx.x - group * parts) * U * u.step + (int)(slot >> lr);
    const int r = s.r0 + (int)j, pos = s.pos0 + (int)j;
    u.row = j < s.n && j < b.max_rows && (unsigned)r < (unsigned)b.n_rows ? r : -1;
    u.page = nullptr;
    u.off = 0;
    if (u.row >= 0 && pos >= 0 && pos < s.len) {
        const int id = b.table[blockIdx.y * b.stride + (pos >> p.shift)];
        if ((unsigned)id < (unsigned)p.n_pages) u.page = const_cast<unsigned char *>(kv_page(p, id));
        u.off = pos & ((1 << p.shift) - 1);
    }
    return u;
}
// offsets in a page's block: piece w's numbers (es bytes each), and its scale of group g
template <int D>
__device__ __forceinline__ long long kv_at(const KvPages &p, int off, int w, int es) {
    return (((long long)w << p.shift) + off) * D * es;
}
template <int D>
__device__ __forceinline__ long long kv_scale_at(const KvPages &p, int off, int w, int g) {
    return (((long long)2 * p.hk << p.shift) * D) + ((((long long)w * (D / 32) + g) << p.shift) + off) * 4;
}
// where piece w of a row lies in the caller's arrays
template <class T>
__device__ __forceinline__ T *kv_place(const KvPages &p, const KvRows &k, const KvRows &v, int row, int w) {
    const bool second = w >= p.hk;
    return (T *)(second ? v.p : k.p) + (row * (second ? v.row : k.row) + (w - (second ? p.hk : 0)) * (second ? v.head : k.head));
}

// Scale and factor of a Q8 group: scale max * (1 / 127), factor 127 * (1 / max)
// (what a torch program that fills pages itself gets from 127.0 / max: against
// 127 / max some factors differ in the last bit, and with them about one code
// in a million by one).  A group of zeros, with NaN or too small: 1 and 0.
__device__ __forceinline__ void kv_scale_inv(float amax, float *sg, float *inv) {
    const float s = amax * (1.0f / 127.0f);
    const bool live = amax > 0.0f && !(s < 1.0e-30f);
    *sg = live ? s : 1.0f;
    *inv = live ? 127.0f * (1.0f / amax) : 0.0f;
}

__device__ __forceinline__ uint32_t max_over(uint32_t v, int lanes) {    // over aligned groups of `lanes`
    for (int o = 1; o < lanes; o <<= 1) {
        const uint32_t y = __shfl_xor(v, o);
        v = y > v ? y : v;
    }
    return v;
}

// E codes of a lane as they lie together, in the low bytes
template <int E> struct KvCodes {
    uint32_t w[(E + 3) / 4];
    __device__ __forceinline__ void load(const unsigned char *s) {
        if (E == 8) {
            const uint2 t = *(const uint2 *)s;
            w[0] = t.x;
            w[E == 8 ? 1 : 0] = t.y;
        } else if (E == 4) {
            w[0] = *(const uint32_t *)s;
        } else {
            w[0] = *(const uint16_t *)s;
        }
    }
    __device__ __forceinline__ void store(unsigned char *s) const {
        if (E == 8) *(uint2 *)s = make_uint2(w[0], w[E == 8 ? 1 : 0]);
        else if (E == 4) *(uint32_t *)s = w[0];
        else *(uint16_t *)s = (uint16_t)w[0];
    }
    __device__ __forceinline__ uint32_t operator[](int i) const { return (w[i / 4] >> (8 * (i & 3))) & 255u; }
};
// The lanes of a row are of one wave: what one of them wrote to LDS is there
// for the others behind this.
__device__ __forceinline__ void kv_lanes() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// K's dimension c*32 + h*8 + j lies at byte h*(D/4) + c*8 + j
template <int D> __device__ __forceinline__ int kv_k_byte(int d) { return ((d & 31) >> 3) * (D / 4) + (d >> 5) * 8 + (d & 7); }

template <class T, int D, bool Q8, int U>
__global__ __launch_bounds__(KV_THREADS) void k_kv_append(KvPages p, KvSeqs b, KvRows k, KvRows v, int vec, int lr, unsigned parts) {
    constexpr int E = D / 16, N = KV_THREADS / 16;
    __shared__ __align__(16) unsigned char rows[Q8 ? U : 1][Q8 ? N : 1][D];
    const KvRow u = kv_row(p, b, lr, parts, U);
    const int lane = threadIdx.x & 15, slot = threadIdx.x >> 4, d0 = lane * E;
    float x[U][E];
    // the shuffles below take every lane of the wave; one without a piece reads a row's first
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int w = u.w0 + i * u.step;
        kv_load<T, E>(kv_place<const T>(p, k, v, u.page ? u.row : 0, w < 2 * p.hk ? w : 0) + d0, vec, x[i]);
    }
    if (!Q8) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int w = u.w0 + i * u.step;
            if (u.page && w < 2 * p.hk) kv_store<__bf16, E>((__bf16 *)(u.page + kv_at<D>(p, u.off, w, 2)) + d0, true, x[i]);
        }
        return;
    }
    KvCodes<E> c[U];
    float sg[U];
#pragma unroll
    for (int i = 0; i < U; i++) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const uint32_t a = u_from_f(x[i][e]) & 0x7FFFFFFFu;
            m = a > m ? a : m;
        }
        m = max_over(m, 32 / E);
        float inv;
        kv_scale_inv(f_from_u(m), &sg[i], &inv);
        c[i] = KvCodes<E>();
        // x + 1.5 * 2^23 has x rounded half to even in its lowest byte, 128 more
        // is the sign bit turned.  |x * inv| < 127.5 where the factor is not 0;
        // where it is, all codes are 0 whatever x holds.
#pragma unroll
        for (int e = 0; e < E; e++) c[i].w[e / 4] |= (u_from_f(x[i][e] * inv + 12582912.0f) & 255u) << (8 * (e & 3));
#pragma unroll
        for (int e = 0; e < (E + 3) / 4; e++) c[i].w[e] = (inv == 0.0f ? 0u : c[i].w[e]) ^ 0x80808080u;
        c[i].store(rows[i][slot] + d0);
    }
    kv_lanes();
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int w = u.w0 + i * u.step;
        if (w >= p.hk) {
#pragma unroll
            for (int e = 0; e < (E + 3) / 4; e++) c[i].w[e] = 0;
#pragma unroll
            for (int t = 0; t < E; t++) c[i].w[t / 4] |= (uint32_t)rows[i][slot][t * 16 + lane] << (8 * (t & 3));
        }
        if (!u.page || w >= 2 * p.hk) continue;
        if (lane % (32 / E) == 0) *(float *)(u.page + kv_scale_at<D>(p, u.off, w, d0 / 32)) = sg[i];
        c[i].store(u.page + kv_at<D>(p, u.off, w, 1) + (w >= p.hk ? d0 : kv_k_byte<D>(d0)));
    }
}

template <class T, int D, bool Q8, int U>
__global__ __launch_bounds__(KV_THREADS) void k_kv_read(KvPages p, KvSeqs b, KvRows k, KvRows v, int vec, int lr, unsigned parts) {
    constexpr int E = D / 16, N = KV_THREADS / 16;
    __shared__ __align__(16) unsigned char rows[Q8 ? U : 1][Q8 ? N : 1][D];
    const KvRow u = kv_row(p, b, lr, parts, U);
    const int lane = threadIdx.x & 15, slot = threadIdx.x >> 4, d0 = lane * E;
    float x[U][E];
    if (!Q8) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int w = u.w0 + i * u.step;
#pragma unroll
            for (int e = 0; e < E; e++) x[i][e] = 0.0f;
            if (u.page && w < 2 * p.hk) kv_load<__bf16, E>((const __bf16 *)(u.page + kv_at<D>(p, u.off, w, 2)) + d0, true, x[i]);
        }
    } else {
        KvCodes<E> c[U];
        float sg[U];
        const unsigned char *page = u.page ? u.page : p.data;      // (without one: a row of page 0, not used)
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int w = u.w0 + i * u.step, a = w < 2 * p.hk ? w : 0;
            c[i].load(page + kv_at<D>(p, u.off, a, 1) + (a >= p.hk ? d0 : kv_k_byte<D>(d0)));
            sg[i] = *(const float *)(page + kv_scale_at<D>(p, u.off, a, d0 / 32));
        }
#pragma unroll
        for (int i = 0; i < U; i++)
            if (u.w0 + i * u.step >= p.hk)
#pragma unroll
                for (int t = 0; t < E; t++) rows[i][slot][t * 16 + lane] = (unsigned char)c[i][t];
        kv_lanes();
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (u.w0 + i * u.step >= p.hk) c[i].load(rows[i][slot] + d0);
#pragma unroll
            for (int e = 0; e < E; e++) x[i][e] = u.page ? (float)((int)c[i][e] - 128) * sg[i] : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int w = u.w0 + i * u.step;
        if (u.row >= 0 && w < 2 * p.hk) kv_store<T, E>(kv_place<T>(p, k, v, u.row, w) + d0, vec, x[i]);
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
        if (many) hipLaunchKernelGGL((K<T, DD, QQ, 4>), grid, dim3(KV_THREADS), 0, st, p, b, k, v, vec, lr, parts); \
        else hipLaunchKernelGGL((K<T, DD, QQ, 1>), grid, dim3(KV_THREADS), 0, st, p, b, k, v, vec, lr, parts); \
    } while (0)
#define KV_ROWS_DISPATCH(K)                                                                                \
    int lr = 0;                                                                                            \
    while (lr < 4 && 1 << lr < b.max_rows) lr++;                                                           \
    const long long groups = ((long long)b.max_rows + (1 << lr) - 1) >> lr;                                \
    const long long step = KV_THREADS / 16 >> lr, singly = (2LL * p.hk + step - 1) / step;                 \
    const bool many = groups * singly * b.n_seq > KV_ALL;                                                  \
    const unsigned parts = (unsigned)(many ? (singly + 3) / 4 : singly);                                   \
    const long long blocks = groups * parts;                                                               \
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
