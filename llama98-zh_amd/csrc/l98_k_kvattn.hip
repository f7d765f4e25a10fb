// Causal attention over the paged key-value cache.
//
// Few rows (k_kv_few): every key is read once for all query heads of its kv
// head, so the bound is HBM and the work is split over the keys: a block takes
// `chunk` keys of one (sequence, kv head, tile of 16 MT rows), its four waves
// 32 keys at a time in turn, and a second launch joins the blocks' partial
// results where there is more than one per row.  A row of a tile is a (new
// row, query head of the group) pair: m = new row * group + head.
//
// A wave computes S^T = K Q^T and O^T += V^T P^T with 16 x 16 x 32 matrix
// instructions, so that the probabilities of a lane's S^T (query lane & 15,
// keys 4 (lane >> 4) + i of each of the two 16-key tiles) are the second
// product's operand as they stand.  K and V go from memory to registers
// directly, one 32-key tile ahead of the one in use.
//
// Exactness.  Q8: the codes are exact in fp16 (as code * 2^-9: a byte u in an
// fp16's low bits is the subnormal u 2^-24, and one packed fma makes
// u 2^-9 - 128 2^-9 of it); a group's partial score is taken in fp32 and
// scaled there.  q is scaled by a power of two per row to below 2^15; a bf16
// row is then exact in fp16, an fp32 row goes as two fp16 parts (22 bits).
// The weights w = p * (V's scale of the group) are at most 2^15 (the running
// maximum M bounds s + log2(scale) - 15 instead of s; the sum runs in the same
// unit), in one fp16 for bf16 rows (a rounding of 2^-11, against 2^-8 of the
// output), two parts for fp32 rows.  bf16 caches: q and p in as many bf16
// parts as their types need: a bf16 q is exact, fp32 takes three (24 bits); p
// takes two for bf16 rows, three for fp32.
#include <limits.h>

#include <type_traits>

#include "l98_devmath.h"
#include "l98_kv.h"
#include "l98_kvattn.h"

#define FEW_THREADS 256
#define FEW_WAVES (FEW_THREADS / 64)
#define FEW_KEYS 32               // of one wave at a time

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// N parts of E whose sum is x to N times E's bits
template <class E, int N>
__device__ __forceinline__ void parts(float x, E *o) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        o[i] = (E)x;
        x -= (float)o[i];
    }
}

// The shape of the work for one (width, cache, row type).
template <int D, bool Q8, bool BF>
struct Few {
    static constexpr int NG = D / 32;                        // contractions of 32, and Q8 groups
    static constexpr int NT = D / 16;                        // 16-wide tiles of the output
    static constexpr int KB = Q8 ? D / 4 : D / 2;            // bytes of a key's K in a lane
    static constexpr int VB = Q8 ? D / 16 : D / 8;           // and of its V
    static constexpr int NQ = Q8 ? (BF ? 1 : 2) : (BF ? 1 : 3);
    static constexpr int NP = Q8 ? (BF ? 1 : 2) : (BF ? 2 : 3);
    static constexpr int KW = KB / 4, VW = VB < 4 ? 1 : VB / 4;
    using E = typename std::conditional<Q8, _Float16, __bf16>::type;
    using V8 = typename std::conditional<Q8, f16x8, bf16x8>::type;
    // a lane's operand element j of contraction c: this dimension of K and q
    static __device__ __forceinline__ int dim(int c, int h) { return Q8 ? c * 32 + h * 8 : h * (D / 4) + c * 8; }
};

// What a lane holds of 32 keys: K of key t*16 + (lane & 15), V of the eight
// keys t*16 + 4*(lane >> 4) + i, and 4 of the tile's Q8 scales.
template <int D, bool Q8, bool BF>
struct FewTile {
    using F = Few<D, Q8, BF>;
    uint32_t k[2][F::KW], v[8][F::VW];
    f32x4 sc[(2 * F::NG * FEW_KEYS) / 256 ? (2 * F::NG * FEW_KEYS) / 256 : 1];
    bool there[2];
};

template <int B>
__device__ __forceinline__ void load_bytes(const unsigned char *s, uint32_t *o) {
    if (B == 2) {
        o[0] = *(const uint16_t *)s;
    } else if (B == 4) {
        o[0] = *(const uint32_t *)s;
    } else if (B == 8) {
        const uint2 x = *(const uint2 *)s;
        o[0] = x.x;
        o[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < B / 16; i++) {
            const uint4 x = *(const uint4 *)(s + 16 * i);
            o[4 * i] = x.x;
            o[4 * i + 1] = x.y;
            o[4 * i + 2] = x.z;
            o[4 * i + 3] = x.w;
        }
    }
}

// The 32 keys from `key` on (a multiple of 32, below the sequence's end): both
// 16-key halves lie within one page each, whose bytes all exist, so positions
// past the length are read too (and masked where they are used).
template <int D, bool Q8, bool BF>
__device__ __forceinline__ void few_load(FewTile<D, Q8, BF> &T, const KvPages &p, const int *table, int pages, int kh,
                                         int key, int len) {
    using F = Few<D, Q8, BF>;
    const int lane = threadIdx.x & 63, n = lane & 15, h = lane >> 4, rows = 1 << p.shift;
    const int vo = p.hk << p.shift;                          // V's rows behind K's
    const unsigned char *pg[2];
    int off[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int k = key + 16 * t, at = k >> p.shift;
        const int id = at < pages ? table[at] : -1;
        T.there[t] = (unsigned)id < (unsigned)p.n_pages;
        pg[t] = kv_page(p, T.there[t] ? id : 0);
        off[t] = (kh << p.shift) + (k & (rows - 1));
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
        load_bytes<F::KB>(pg[t] + (off[t] + n) * (Q8 ? D : 2 * D) + h * F::KB, T.k[t]);
#pragma unroll
        for (int i = 0; i < 4; i++)
            load_bytes<F::VB>(pg[t] + (vo + off[t] + h * 4 + i) * (Q8 ? D : 2 * D) + n * F::VB, T.v[t * 4 + i]);
    }
    if (Q8) {
        // chunk x of the tile's 2 NG 32 / 4 scales: which, group, 4 keys
#pragma unroll
        for (int u = 0; u < (int)(sizeof(T.sc) / 16); u++) {
            const int x = u * 64 + lane, which = (x / (F::NG * 8)) & 1, g = (x / 8) % F::NG, k4 = (x & 7) * 4, t = k4 >> 4;
            const unsigned char *s = (t ? pg[1] : pg[0]) + 2 * vo * D +
                                     (((which * p.hk + kh) * F::NG + g) << p.shift) * 4 +
                                     (((key + k4) & (rows - 1)) * 4);
            T.sc[u] = *(const f32x4 *)s;
#pragma unroll
            for (int i = 0; i < 4; i++) T.sc[u][i] = key + k4 + i < len ? T.sc[u][i] : 0.0f;
        }
    }
}

__device__ __forceinline__ float max_h(float x) {            // over the four lanes of a query
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_h(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <int D, bool Q8, bool BF, int MT>
struct FewAcc {
    using F = Few<D, Q8, BF>;
    u32x4 q[MT][F::NG][F::NQ];
    f32x4 o[MT][F::NT];
    float m[MT], l[MT], cq[MT];
    int lim[MT];                                             // the row's keys: below this
};

// One tile of 32 keys.  masked: some row of the block's may not attend some
// of them, or they are not all there.
template <int D, bool Q8, bool BF, int MT>
__device__ __forceinline__ void few_tile(FewAcc<D, Q8, BF, MT> &A, FewTile<D, Q8, BF> &T, float *sc, int key, int len,
                                         bool masked) {
    using F = Few<D, Q8, BF>;
    using E = typename F::E;
    using V8 = typename F::V8;
    const int lane = threadIdx.x & 63, h = lane >> 4;
    f32x4 s[MT][2];
    if (Q8) {
        // the wave's own part of LDS: written whole, then read by every lane
#pragma unroll
        for (int u = 0; u < (int)(sizeof(T.sc) / 16); u++)
            if (u * 64 + lane < 2 * F::NG * 8) *(f32x4 *)(sc + (u * 64 + lane) * 4) = T.sc[u];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    float top[MT];
#pragma unroll
    for (int t = 0; t < 2; t++) {
#pragma unroll
        for (int m = 0; m < MT; m++) s[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < F::NG; c++) {
            u32x4 kx;
            if (Q8) {
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const uint32_t x = T.k[t][2 * c + w];
                    kx[2 * w] = codes2(0, x, 0x0c010c00u);
                    kx[2 * w + 1] = codes2(0, x, 0x0c030c02u);
                }
                const f32x4 ks = *(const f32x4 *)(sc + c * FEW_KEYS + t * 16 + h * 4);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    f32x4 part = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < F::NQ; i++) part = mfma(as<V8>(kx), as<V8>(A.q[m][c][i]), part);
#pragma unroll
                    for (int i = 0; i < 4; i++) s[m][t][i] = __builtin_fmaf(part[i], ks[i], s[m][t][i]);
                }
            } else {
#pragma unroll
                for (int w = 0; w < 4; w++) kx[w] = T.k[t][4 * c + w];
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < F::NQ; i++) s[m][t] = mfma(as<V8>(kx), as<V8>(A.q[m][c][i]), s[m][t]);
            }
        }
    }
    // scores in units of log2, masked; the largest of the row and, for Q8, of V's scales with it
#pragma unroll
    for (int m = 0; m < MT; m++) {
        float mx = ninf();
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[m][t][i] *= A.cq[m];
                if (masked && !(T.there[t] && key + t * 16 + h * 4 + i < A.lim[m])) s[m][t][i] = ninf();
                mx = fmaxf(mx, s[m][t][i]);
            }
        top[m] = mx;
    }
    float vmax[8];
    if (Q8) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            f32x4 x = *(const f32x4 *)(sc + F::NG * FEW_KEYS + t * 16 + h * 4);
#pragma unroll
            for (int g = 1; g < F::NG; g++) {
                const f32x4 y = *(const f32x4 *)(sc + (F::NG + g) * FEW_KEYS + t * 16 + h * 4);
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = fmaxf(x[i], y[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) vmax[t * 4 + i] = x[i];
        }
    }
    bool same = true;
    float keep[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) {
        float mt = max_h(top[m]);
        if (Q8) {
            // 2^ex > every V scale that the row attends; M = s + ex - 15
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = !masked || (T.there[i >> 2] && key + (i >> 2) * 16 + h * 4 + (i & 3) < A.lim[m]);
                x = fmaxf(x, in ? vmax[i] : 0.0f);
            }
            x = max_h(x);
            mt += (float)((int)(u_from_f(x) >> 23) - 126 - 15);
        }
        const float mn = fmaxf(A.m[m], mt), mu = mn == ninf() ? 0.0f : mn;
        keep[m] = kv_exp2(A.m[m] - mu);
        same = same && mn == A.m[m];
        A.m[m] = mn;
        float l = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[m][t][i] = kv_exp2(s[m][t][i] - mu);
                l += s[m][t][i];
            }
        A.l[m] = __builtin_fmaf(A.l[m], keep[m], l);
    }
    if (!__all(same)) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int d = 0; d < F::NT; d++) A.o[m][d] *= keep[m];
    }
    if (!Q8 && masked) {
        // A key that some row may not attend must not reach it as 0 * NaN: its
        // V becomes zero; where it has a value that is not finite, the rows
        // that attend it get NaN by their sum instead.
#pragma unroll
        for (int i = 0; i < 8; i++) {
            bool bad = false;
#pragma unroll
            for (int w = 0; w < F::VW; w++)
                bad = bad || (T.v[i][w] & 0x7F80u) == 0x7F80u || (T.v[i][w] & 0x7F800000u) == 0x7F800000u;
            const bool any = ((__ballot(bad) >> (16 * h)) & 0xFFFFull) != 0;
            const int k = key + (i >> 2) * 16 + h * 4 + (i & 3);
            const bool drop = any || k >= len || !T.there[i >> 2];
#pragma unroll
            for (int w = 0; w < F::VW; w++) T.v[i][w] = drop ? 0u : T.v[i][w];
#pragma unroll
            for (int m = 0; m < MT; m++)
                if (any && T.there[i >> 2] && k < A.lim[m]) A.l[m] = __builtin_nanf("");
        }
    }
    if (Q8) {
#pragma unroll
        for (int g = 0; g < F::NG; g++) {
            u32x4 w[MT][F::NP];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const f32x4 vs = *(const f32x4 *)(sc + (F::NG + g) * FEW_KEYS + t * 16 + h * 4);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    E e[4][F::NP];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = s[m][t][i] * vs[i];
                        // a scale that is not finite, of a key that the row may not attend
                        if (masked && !(T.there[t] && key + t * 16 + h * 4 + i < A.lim[m])) x = 0.0f;
                        parts<E, F::NP>(x, e[i]);
                    }
#pragma unroll
                    for (int k = 0; k < F::NP; k++) {
                        w[m][k][2 * t] = pack2(e[0][k], e[1][k]);
                        w[m][k][2 * t + 1] = pack2(e[2][k], e[3][k]);
                    }
                }
            }
#pragma unroll
            for (int d = 2 * g; d < 2 * g + 2; d++) {
                u32x4 vx;
                constexpr uint32_t base = 0x0c040c00u;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    vx[i] = codes2(T.v[2 * i + 1][d / 4], T.v[2 * i][d / 4], base + (uint32_t)(d & 3) * 0x00010001u);
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int k = 0; k < F::NP; k++) A.o[m][d] = mfma(as<V8>(vx), as<V8>(w[m][k]), A.o[m][d]);
            }
        }
    } else {
        u32x4 w[MT][F::NP];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int t = 0; t < 2; t++) {
                E e[4][F::NP];
#pragma unroll
                for (int i = 0; i < 4; i++) parts<E, F::NP>(s[m][t][i], e[i]);
#pragma unroll
                for (int k = 0; k < F::NP; k++) {
                    w[m][k][2 * t] = pack2(e[0][k], e[1][k]);
                    w[m][k][2 * t + 1] = pack2(e[2][k], e[3][k]);
                }
            }
#pragma unroll
        for (int d = 0; d < F::NT; d++) {
            u32x4 vx;
#pragma unroll
            for (int i = 0; i < 4; i++)
                vx[i] = __builtin_amdgcn_perm(T.v[2 * i + 1][d / 2], T.v[2 * i][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int k = 0; k < F::NP; k++) A.o[m][d] = mfma(as<V8>(vx), as<V8>(w[m][k]), A.o[m][d]);
        }
    }
}

template <int D, bool Q8, bool BF, int MT>
__global__ __launch_bounds__(FEW_THREADS, D == 128 && MT == 2 ? 1 : 2) void k_kv_few(KvPages p, KvSeqs b, KvRows q, KvRows out, int heads, int group,
                                                           float scale2, int chunk, int tiles, KvParts w) {
    using F = Few<D, Q8, BF>;
    using E = typename F::E;
    using T = typename std::conditional<BF, __bf16, float>::type;
    constexpr int ROWS = 16 * MT, SC = 2 * F::NG * FEW_KEYS;
    __shared__ float so[FEW_WAVES * ROWS * D];               // the loop's scales, then the waves' results
    __shared__ float sm[FEW_WAVES][ROWS], sl[FEW_WAVES][ROWS];
    static_assert(SC * FEW_WAVES <= FEW_WAVES * ROWS * D, "the scales fit");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, h = lane >> 4;
    // splits of a tile next to each other, the tiles with the most keys first
    const int seq = blockIdx.y, split = blockIdx.x % w.splits, y = blockIdx.x / w.splits;
    const int kh = y % p.hk, tile = tiles - 1 - y / p.hk;
    const KvSeq s = kv_seq(b, seq, p.shift);
    const int nr = s.n < b.max_rows ? s.n : b.max_rows;
    if ((long long)tile * ROWS >= (long long)nr * group) return;
    const int j_first = tile * ROWS / group;
    int j_last = (tile * ROWS + ROWS - 1) / group;
    j_last = j_last < nr ? j_last : nr - 1;
    int end = s.pos0 + j_last + 1;                           // of the tile's keys
    end = end < s.len ? end : s.len;
    const int k0 = split * chunk;
    int k1 = k0 + chunk;
    k1 = k1 < end ? k1 : end;
    const int *table = b.table + seq * b.stride;

    FewAcc<D, Q8, BF, MT> A;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int row = tile * ROWS + m * 16 + n, j = row / group, r = s.r0 + j;
        const bool on = j < nr && (unsigned)r < (unsigned)b.n_rows;
        const T *src = (const T *)q.p + (on ? r * q.row + (kh * group + row % group) * q.head : 0);
        A.lim[m] = on ? (s.pos0 + j + 1 < s.len ? s.pos0 + j + 1 : s.len) : 0;
        A.m[m] = ninf();
        A.l[m] = 0.0f;
#pragma unroll
        for (int d = 0; d < F::NT; d++) A.o[m][d] = f32x4{0, 0, 0, 0};
        float x[F::NG][8];
        uint32_t big = 0;
#pragma unroll
        for (int c = 0; c < F::NG; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c][i] = on ? (float)src[F::dim(c, h) + i] : 0.0f;
                const uint32_t a = u_from_f(x[c][i]) & 0x7FFFFFFFu;
                big = a > big ? a : big;
            }
        A.cq[m] = scale2;
        int e = 0;
        if (Q8) {
            uint32_t y = __shfl_xor(big, 16);
            big = y > big ? y : big;
            y = __shfl_xor(big, 32);
            big = y > big ? y : big;
            e = (int)(big >> 23) - 127 - 14;                 // the row's largest to [2^14, 2^15)
            A.cq[m] = __builtin_amdgcn_ldexpf(scale2, e + 9);
        }
#pragma unroll
        for (int c = 0; c < F::NG; c++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                E lo[F::NQ], hi[F::NQ];
                parts<E, F::NQ>(Q8 ? __builtin_amdgcn_ldexpf(x[c][i], -e) : x[c][i], lo);
                parts<E, F::NQ>(Q8 ? __builtin_amdgcn_ldexpf(x[c][i + 1], -e) : x[c][i + 1], hi);
#pragma unroll
                for (int k = 0; k < F::NQ; k++) A.q[m][c][k][i / 2] = pack2(lo[k], hi[k]);
            }
    }
    // keys below this are attended by every row of the tile
    int all = s.pos0 + j_first + 1;
    all = all < s.len ? all : s.len;
    float *sc = so + wave * SC;
    const int step = FEW_WAVES * FEW_KEYS;
    int key = k0 + wave * FEW_KEYS;
    if (key < k1) {
        FewTile<D, Q8, BF> t0, t1;
        few_load<D, Q8, BF>(t0, p, table, b.pages, kh, key, s.len);
        for (;;) {
            const bool m0 = key + FEW_KEYS > all || !(t0.there[0] && t0.there[1]);
            const int next = key + step;
            if (next < k1) few_load<D, Q8, BF>(t1, p, table, b.pages, kh, next, s.len);
            few_tile<D, Q8, BF, MT>(A, t0, sc, key, s.len, m0);
            if (next >= k1) break;
            key = next + step;
            const bool m1 = next + FEW_KEYS > all || !(t1.there[0] && t1.there[1]);
            if (key < k1) few_load<D, Q8, BF>(t0, p, table, b.pages, kh, key, s.len);
            few_tile<D, Q8, BF, MT>(A, t1, sc, next, s.len, m1);
            if (key >= k1) break;
        }
    }
    // the four waves' results: scaled to the block's maximum, summed in wave order
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const float l = sum_h(A.l[m]);
        if (h == 0) {
            sm[wave][m * 16 + n] = A.m[m];
            sl[wave][m * 16 + n] = l;
        }
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; m++) {
        float mx = ninf();
#pragma unroll
        for (int x = 0; x < FEW_WAVES; x++) mx = fmaxf(mx, sm[x][m * 16 + n]);
        const float f = kv_exp2(A.m[m] - (mx == ninf() ? 0.0f : mx));
        float *o = so + (wave * ROWS + m * 16 + n) * D;
#pragma unroll
        for (int d = 0; d < F::NT; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[Q8 ? d * 16 + h * 4 + i : (h * 4 + i) * F::NT + d] = A.o[m][d][i] * f;
    }
    __syncthreads();
    constexpr int PER = FEW_THREADS / ROWS, DT = D / PER;    // threads of a row, dimensions of a thread
    const int m = threadIdx.x / PER, d0 = threadIdx.x % PER * DT;
    const int row = tile * ROWS + m, j = row / group, r = s.r0 + j, head = kh * group + row % group;
    if (j >= nr || (unsigned)r >= (unsigned)b.n_rows) return;
    float mx = ninf(), l = 0.0f, x[DT];
#pragma unroll
    for (int y = 0; y < FEW_WAVES; y++) mx = fmaxf(mx, sm[y][m]);
#pragma unroll
    for (int y = 0; y < FEW_WAVES; y++) l += sl[y][m] * kv_exp2(sm[y][m] - (mx == ninf() ? 0.0f : mx));
#pragma unroll
    for (int i = 0; i < DT; i++) {
        x[i] = 0.0f;
#pragma unroll
        for (int y = 0; y < FEW_WAVES; y++) x[i] += so[(y * ROWS + m) * D + d0 + i];
        if (Q8) x[i] *= 512.0f;                              // the codes' 2^-9
    }
    if (w.splits == 1) {
        T *dst = (T *)out.p + r * out.row + head * out.head + d0;
#pragma unroll
        for (int i = 0; i < DT; i++) dst[i] = (T)(l == 0.0f ? 0.0f : x[i] / l);
        return;
    }
    const long long at = ((long long)r * heads + head) * w.splits + split;
    if (d0 == 0) {
        w.ml[2 * at] = mx;
        w.ml[2 * at + 1] = l;
    }
    if (mx != ninf())
#pragma unroll
        for (int i = 0; i < DT; i++) w.o[at * D + d0 + i] = x[i];
}

// out = sum over splits of 2^(M_s - M) o_s / sum of 2^(M_s - M) l_s, in split
// order within a lane and then over the lanes: one block per (row, head).
#define JOIN_THREADS 256
template <int D, bool BF>
__global__ __launch_bounds__(JOIN_THREADS) void k_kv_join(KvSeqs b, KvRows out, int heads, KvParts w) {
    using T = typename std::conditional<BF, __bf16, float>::type;
    constexpr int L = D / 4, G = JOIN_THREADS / L;           // lanes of a split, splits at a time
    __shared__ float so[G][D], sl[G], sm[JOIN_THREADS / 64];
    const int j = blockIdx.x / heads, head = blockIdx.x % heads, seq = blockIdx.y, tid = threadIdx.x;
    const int r0 = b.row0[seq], nr = b.row0[seq + 1] - r0, r = r0 + j;
    if (j >= nr || (unsigned)r >= (unsigned)b.n_rows) return;
    const long long at = ((long long)r * heads + head) * w.splits;
    float mx = ninf();
    for (int i = tid; i < w.splits; i += JOIN_THREADS) mx = fmaxf(mx, w.ml[2 * (at + i)]);
    for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
    if ((tid & 63) == 0) sm[tid >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < JOIN_THREADS / 64; i++) mx = fmaxf(mx, sm[i]);
    const int g = tid / L, d = tid % L * 4;
    f32x4 acc = {0, 0, 0, 0};
    float l = 0.0f;
    for (int i = g; i < w.splits; i += G) {
        const float mi = w.ml[2 * (at + i)];
        if (mi == ninf()) continue;                          // no keys: its o is not written
        const float f = kv_exp2(mi - mx);
        l += w.ml[2 * (at + i) + 1] * f;
        acc += *(const f32x4 *)(w.o + (at + i) * D + d) * f;
    }
    *(f32x4 *)&so[g][d] = acc;
    if (d == 0) sl[g] = l;
    __syncthreads();
    if (tid < D) {
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int i = 0; i < G; i++) {
            x += so[i][tid];
            y += sl[i];
        }
        ((T *)out.p + r * out.row + head * out.head)[tid] = (T)(y == 0.0f ? 0.0f : x / y);
    }
}

// ---------------------------------------------------------- host glue ---

namespace {

// How a call's work is cut.  rows: of a block's tile; tiles: of a sequence and
// kv head; chunk: keys of a block; splits: blocks of a tile.
KvPlan plan(const KvPages &p, const KvSeqs &b, int heads, int bf16) {
    KvPlan x;
    const long long rows = (long long)b.max_rows * (heads / p.hk);
    x.many = bf16 && rows > 128;
    int unit, least;
    long long want;
    if (x.many) {
        x.rows = (long long)b.n_seq * p.hk * ((rows + 255) / 256) >= 256 ? 256 : 128;
        unit = 64;
        least = 512;
        want = 256;
    } else {
        x.rows = rows <= 16 ? 16 : 32;
        unit = FEW_WAVES * FEW_KEYS;
        least = 256;
        want = 768;
    }
    x.tiles = (int)((rows + x.rows - 1) / x.rows);
    const long long base = (long long)b.n_seq * p.hk * x.tiles;
    long long splits = (want + base - 1) / base;
    const long long most = (b.max_len + least - 1) / least;
    splits = splits < most ? splits : most;
    splits = splits > 1 ? splits : 1;
    const long long chunk = ((b.max_len + splits - 1) / splits + unit - 1) / unit * unit;
    x.chunk = (int)(chunk > unit ? chunk : unit);
    x.splits = (int)(((long long)b.max_len + x.chunk - 1) / x.chunk);
    x.splits = x.splits > 1 ? x.splits : 1;
    return x;
}

template <int D, bool Q8, bool BF>
int few(const KvPages &p, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads, float scale2, const KvPlan &x,
        const KvParts &w, hipStream_t st) {
    const dim3 grid((unsigned)((long long)x.splits * p.hk * x.tiles), b.n_seq);
    if (x.rows == 16)
        hipLaunchKernelGGL((k_kv_few<D, Q8, BF, 1>), grid, dim3(FEW_THREADS), 0, st, p, b, q, o, heads, heads / p.hk,
                           scale2, x.chunk, x.tiles, w);
    else
        hipLaunchKernelGGL((k_kv_few<D, Q8, BF, 2>), grid, dim3(FEW_THREADS), 0, st, p, b, q, o, heads, heads / p.hk,
                           scale2, x.chunk, x.tiles, w);
    return (int)hipGetLastError();
}

template <int D>
int attend(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads, int bf16, float scale,
           void *ws, hipStream_t st) {
    const KvPlan x = plan(p, b, heads, bf16);
    KvParts w;
    w.splits = x.splits;
    w.o = (float *)ws;
    w.ml = w.o + (long long)b.n_rows * heads * x.splits * D;
    const float scale2 = scale * 1.44269504088896341f;
    const long long blocks = (long long)x.splits * p.hk * x.tiles, joins = (long long)b.max_rows * heads;
    if (blocks > INT_MAX || joins > INT_MAX) return -1;
    int rc;
    if (x.many) rc = l98k_kv_many(p, q8, b, q, o, heads, scale2, x, w, st);
    else if (q8) rc = bf16 ? few<D, true, true>(p, b, q, o, heads, scale2, x, w, st)
                           : few<D, true, false>(p, b, q, o, heads, scale2, x, w, st);
    else rc = bf16 ? few<D, false, true>(p, b, q, o, heads, scale2, x, w, st)
                   : few<D, false, false>(p, b, q, o, heads, scale2, x, w, st);
    if (rc || x.splits == 1) return rc;
    if (bf16) hipLaunchKernelGGL((k_kv_join<D, true>), dim3((unsigned)joins, b.n_seq), dim3(JOIN_THREADS), 0, st, b, o, heads, w);
    else hipLaunchKernelGGL((k_kv_join<D, false>), dim3((unsigned)joins, b.n_seq), dim3(JOIN_THREADS), 0, st, b, o, heads, w);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" long long l98k_kv_attend_ws(const KvPages &p, int, const KvSeqs &b, int heads, int bf16) {
    const KvPlan x = plan(p, b, heads, bf16);
    return x.splits == 1 ? 0 : (long long)b.n_rows * heads * x.splits * (p.d + 2) * 4;
}

extern "C" int l98k_kv_attend(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads,
                              int bf16, float scale, void *ws, hipStream_t st) {
    if (p.d == 32) return attend<32>(p, q8, b, q, o, heads, bf16, scale, ws, st);
    if (p.d == 64) return attend<64>(p, q8, b, q, o, heads, bf16, scale, ws, st);
    if (p.d == 128) return attend<128>(p, q8, b, q, o, heads, bf16, scale, ws, st);
    return -1;
}
