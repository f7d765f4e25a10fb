// Causal attention over the paged key-value cache.
//
// Few rows (k_kv_few): every key is read once for all query heads of its kv
// head, so the bound is HBM and the work is split over the keys: a block takes
// `chunk` keys of one (sequence, kv head, tile of 16 MT rows), its four waves
// 32 keys at a time in turn, and a second launch joins the blocks' partial
// results where there is more than one per row.  A row of a tile is a (new
// row, query head of the group) pair: m = new row * group + head.  Measured
// (16 heads over 4, width 128): 8 rows at 250,015 keys of Q8 64 us, 4.4 TB/s;
// one row each of 100 sequences of 1 to 5000 keys in bf16 113 us, 4.7 TB/s; 4
// fp32 rows each of 32 sequences of 256 to 2048 keys 18 us, of which a block's
// start is a third.  512 fp32 rows at 4096 are bound by their registers and
// vector instructions: 80 us.
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
// maximum is of s + log2(scale); the sum runs in the same unit), in one fp16
// for bf16 rows (a rounding of 2^-12, against the output's 2^-9), two parts
// for fp32 rows.  bf16 caches: q and p in as many bf16 parts as their types
// need: a bf16 q is exact, fp32 takes three (24 bits); p takes two for bf16
// rows, three for fp32.
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

// What a lane holds of a tile of 32 keys: K of key t*16 + (lane & 15), V of the
// eight keys t*16 + 4*(lane >> 4) + i, and 4 of the tile's Q8 scales.
template <int D, bool Q8, bool BF>
struct FewTile {
    using F = Few<D, Q8, BF>;
    uint32_t k[2][F::KW], v[8][F::VW];
    f32x4 sc;
};

// The pages of a tile's two 16-key halves, which each lie within one: all its
// bytes exist, so positions past the length are read too, and masked where
// they are used.
struct FewPages {
    int id[2];
};
__device__ __forceinline__ FewPages few_pages(const KvPages &p, const int *table, int pages, int key) {
    FewPages x;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        const int at = (key + 16 * t) >> p.shift;
        x.id[t] = at < pages ? table[at] : -1;
    }
    return x;
}

// The addresses of a kv head's tiles: uniform ones per tile half, and what is
// the lane's own.
template <int D, bool Q8, bool BF>
struct FewAddr {
    using F = Few<D, Q8, BF>;
    static constexpr uint32_t ROW = Q8 ? D : 2 * D;
    uint32_t head, v, scales;              // of the page's block: this head's K, V behind K, the scales
    uint32_t lane_k, lane_v, lane_s;
    bool second;                           // the lane's scales belong to the second half

    __device__ __forceinline__ FewAddr(const KvPages &p, int kh) {
        const uint32_t lane = threadIdx.x & 63, n = lane & 15, h = lane >> 4;
        head = ((uint32_t)kh << p.shift) * ROW;
        v = ((uint32_t)p.hk << p.shift) * ROW;
        scales = 2 * v;
        lane_k = n * ROW + h * F::KB;
        lane_v = h * 4 * ROW + n * F::VB;
        // lane x: 4 keys' scales, x = (which * NG + group) * 8 + key / 4
        const uint32_t which = (lane / (F::NG * 8)) & 1, g = (lane / 8) % F::NG, k4 = (lane & 7) * 4;
        second = k4 >= 16;
        lane_s = ((((which * p.hk + kh) * F::NG + g) << p.shift) + (k4 & 15)) * 4;
    }
    __device__ __forceinline__ const unsigned char *base(const KvPages &p, const FewPages &x, int t) const {
        return kv_page(p, (unsigned)x.id[t] < (unsigned)p.n_pages ? x.id[t] : 0);
    }
    __device__ __forceinline__ uint32_t at(const KvPages &p, int key, int t) const {
        return (uint32_t)((key + 16 * t) & ((1 << p.shift) - 1));
    }
    __device__ __forceinline__ void load_k(FewTile<D, Q8, BF> &T, const KvPages &p, const FewPages &x, int key) const {
#pragma unroll
        for (int t = 0; t < 2; t++) load_bytes<F::KB>(base(p, x, t) + (head + at(p, key, t) * ROW) + lane_k, T.k[t]);
    }
    __device__ __forceinline__ void load_v(FewTile<D, Q8, BF> &T, const KvPages &p, const FewPages &x, int key) const {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const unsigned char *s = base(p, x, t) + (v + head + at(p, key, t) * ROW);
#pragma unroll
            for (int i = 0; i < 4; i++) load_bytes<F::VB>(s + i * ROW + lane_v, T.v[t * 4 + i]);
        }
        if (Q8) {
            const unsigned char *s0 = base(p, x, 0) + (scales + at(p, key, 0) * 4), *s1 = base(p, x, 1) + (scales + at(p, key, 1) * 4);
            T.sc = *(const f32x4 *)((second ? s1 : s0) + lane_s);
        }
    }
};

__device__ __forceinline__ float max_h(float x) {            // over the four lanes of a query
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_h(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// the largest of the wave's words, by DPP: over rows of 16, then over the rows
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t x) {
    auto step = [&](uint32_t y) { x = y > x ? y : x; };
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true));   // row_shr:1
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, true));   // row_bcast:15 into rows 1, 3
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, true));   // row_bcast:31 into rows 2, 3
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// eight consecutive numbers; without a branch around each load, or they would
// be waited for one by one
template <class T>
__device__ __forceinline__ void load8(const T *s, int vec, float *x) {
    typedef T vt __attribute__((ext_vector_type(16 / sizeof(T))));
    constexpr int N = 16 / sizeof(T);
    if (vec) {
#pragma unroll
        for (int i = 0; i < 8; i += N) {
            const vt t = *reinterpret_cast<const vt *>(s + i);
#pragma unroll
            for (int u = 0; u < N; u++) x[i + u] = (float)t[u];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)s[i];
    }
}

#define FEW_NONE -3.0e38f         // the running maximum of a row without keys
template <int D, bool Q8, bool BF, int MT>
struct FewAcc {
    using F = Few<D, Q8, BF>;
    u32x4 q[MT][F::NG][F::NQ];
    f32x4 o[MT][F::NT];
    float m[MT], l[MT], cq[MT];
    int lim[MT];                                             // the row's keys: below this
    bool huge;                                               // some m is
};
__device__ __forceinline__ bool few_huge(float m) { return fabsf(m) > 0x1p20f && m != FEW_NONE; }

// The scores of a tile, s[m][t][i] of query (lane & 15) and key t*16 + 4*(lane >> 4) + i.
template <int D, bool Q8, bool BF, int MT>
__device__ __forceinline__ void few_scores(const FewAcc<D, Q8, BF, MT> &A, const FewTile<D, Q8, BF> &T, const float *sc,
                                           f32x4 (&s)[MT][2]) {
    using F = Few<D, Q8, BF>;
    using V8 = typename F::V8;
    const int h = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int t = 0; t < 2; t++) s[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < F::NG; c++) {
        f32x4 part[MT][2], ks[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            u32x4 kx;
            if (Q8) {
                ks[t] = *(const f32x4 *)(sc + c * FEW_KEYS + t * 16 + h * 4);
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    kx[2 * w] = codes2(0, T.k[t][2 * c + w], 0x0c010c00u);
                    kx[2 * w + 1] = codes2(0, T.k[t][2 * c + w], 0x0c030c02u);
                }
            } else {
#pragma unroll
                for (int w = 0; w < 4; w++) kx[w] = T.k[t][4 * c + w];
            }
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if (Q8) part[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < F::NQ; i++) {
                    if (Q8) part[m][t] = mfma(as<V8>(kx), as<V8>(A.q[m][c][i]), part[m][t]);
                    else s[m][t] = mfma(as<V8>(kx), as<V8>(A.q[m][c][i]), s[m][t]);
                }
            }
        }
        if (Q8)
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[m][t][i] = __builtin_fmaf(part[m][t][i], ks[t][i], s[m][t][i]);
    }
}

// Softmax of a tile's scores and the products with V.  there: which halves
// have a page; masked: some row may not attend some of the keys, or they are
// not all there.
template <int D, bool Q8, bool BF, int MT>
__device__ __forceinline__ void few_values(FewAcc<D, Q8, BF, MT> &A, FewTile<D, Q8, BF> &T, float *sc,
                                           f32x4 (&s)[MT][2], int key, int len, bool there0, bool there1, bool masked,
                                           float vex) {
    using F = Few<D, Q8, BF>;
    using E = typename F::E;
    using V8 = typename F::V8;
    const int lane = threadIdx.x & 63, h = lane >> 4;
    // Q8 weights are p * (V's scale): 2^ex > every scale that the row attends
    // of the tile (vex: all of them), and s + ex bounds their logarithm.  They
    // may reach 2^15; a raise of the running maximum brings them to 2^11.
    // bf16: p up to 2^8, and to 1.
    constexpr float ROOM = Q8 ? 15.0f : 8.0f, DROP = Q8 ? 11.0f : 0.0f;
    float cand[MT];
    bool up = false;
    if (masked) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
            float vx = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int k = (i >> 2) * 16 + h * 4 + (i & 3);
                const bool in = (i < 4 ? there0 : there1) && key + k < A.lim[m];
                s[m][i >> 2][i & 3] = in ? s[m][i >> 2][i & 3] : ninf();
                if (Q8)
#pragma unroll
                    for (int g = 0; g < F::NG; g++) {
                        const float v = sc[(F::NG + g) * FEW_KEYS + k];
                        const bool bad = (u_from_f(v) & 0x7F800000u) == 0x7F800000u;
                        if (in && bad) A.l[m] = __builtin_nanf("");
                        vx = fmaxf(vx, in && !bad ? v : 0.0f);
                    }
            }
            cand[m] = Q8 ? (float)((int)(u_from_f(vx) >> 23) - 126) : 0.0f;
        }
        if (Q8) {
            // A scale that is not finite becomes zero, so that it does not reach the
            // rows that may not attend its key as 0 * NaN; those that attend it have
            // NaN by their sum.
            if (lane < 2 * F::NG * 8 && lane >= F::NG * 8) {
                f32x4 v = *(f32x4 *)(sc + lane * 4);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = (u_from_f(v[i]) & 0x7F800000u) == 0x7F800000u ? 0.0f : v[i];
                *(f32x4 *)(sc + lane * 4) = v;
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    } else {
#pragma unroll
        for (int m = 0; m < MT; m++) cand[m] = vex;
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
        float mx = s[m][0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[m][i >> 2][i & 3]);
        cand[m] = mx * A.cq[m] + cand[m];                    // (rounded in two steps, as below)
        up = up || cand[m] > A.m[m] + ROOM;
    }
    if (__any(up)) {
        // each row by itself: its bits must not depend on the tile's other rows
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const float c = max_h(cand[m]);
            const bool mine = c > A.m[m] + ROOM;
            const float f = mine ? kv_exp2(A.m[m] - (c - DROP)) : 1.0f;
            A.m[m] = mine ? c - DROP : A.m[m];
            A.l[m] *= f;
#pragma unroll
            for (int d = 0; d < F::NT; d++) A.o[m][d] *= f;
        }
        bool any = false;
#pragma unroll
        for (int m = 0; m < MT; m++) any = any || few_huge(A.m[m]);
        A.huge = __any(any);
    }
#pragma unroll
    for (int m = 0; m < MT; m++) {
        float c = A.cq[m], mu = A.m[m];
        // Of scores so large that the maximum's rounding is no small difference
        // the products are rounded like it.
        if (A.huge) {
            const bool big = few_huge(mu);
#pragma unroll
            for (int i = 0; i < 8; i++) s[m][i >> 2][i & 3] = big ? s[m][i >> 2][i & 3] * c - mu : s[m][i >> 2][i & 3];
            c = big ? 1.0f : c;
            mu = big ? 0.0f : mu;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            s[m][i >> 2][i & 3] = kv_exp2(__builtin_fmaf(s[m][i >> 2][i & 3], c, -mu));
            A.l[m] += s[m][i >> 2][i & 3];
        }
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
            const bool any = ((__ballot(bad) >> (16 * h)) & 0xFFFFull) != 0, there = i < 4 ? there0 : there1;
            const int k = key + (i >> 2) * 16 + h * 4 + (i & 3);
            const bool drop = any || k >= len || !there;
#pragma unroll
            for (int w = 0; w < F::VW; w++) T.v[i][w] = drop ? 0u : T.v[i][w];
#pragma unroll
            for (int m = 0; m < MT; m++)
                if (any && there && k < A.lim[m]) A.l[m] = __builtin_nanf("");
        }
    }
    u32x4 w[MT][F::NP];
    auto weights = [&](const f32x4 (&vs)[2]) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const int t = i >> 2, e = i & 3;
                float a = s[m][t][e], b = s[m][t][e + 1];
                if (Q8) {
                    a *= vs[t][e];
                    b *= vs[t][e + 1];
                }
                uint32_t x[F::NP];
                parts2<E, F::NP>(a, b, x);
#pragma unroll
                for (int k = 0; k < F::NP; k++) w[m][k][i / 2] = x[k];
            }
    };
    auto product = [&](int d, const u32x4 &vx) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int k = 0; k < F::NP; k++) A.o[m][d] = mfma(as<V8>(vx), as<V8>(w[m][k]), A.o[m][d]);
    };
    if (Q8) {
#pragma unroll
        for (int g = 0; g < F::NG; g++) {
            f32x4 vs[2];
#pragma unroll
            for (int t = 0; t < 2; t++) vs[t] = *(const f32x4 *)(sc + (F::NG + g) * FEW_KEYS + t * 16 + h * 4);
            weights(vs);
#pragma unroll
            for (int d = 2 * g; d < 2 * g + 2; d++) {
                u32x4 vx;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    vx[i] = codes2(T.v[2 * i + 1][d / 4], T.v[2 * i][d / 4], 0x0c040c00u + (uint32_t)(d & 3) * 0x00010001u);
                product(d, vx);
            }
        }
    } else {
        const f32x4 one[2] = {};
        weights(one);
#pragma unroll
        for (int d = 0; d < F::NT; d++) {
            u32x4 vx;
#pragma unroll
            for (int i = 0; i < 4; i++)
                vx[i] = __builtin_amdgcn_perm(T.v[2 * i + 1][d / 2], T.v[2 * i][d / 2], d & 1 ? 0x07060302u : 0x05040100u);
            product(d, vx);
        }
    }
}

template <int D, bool Q8, bool BF, int MT>
__global__ __launch_bounds__(FEW_THREADS, 2) void k_kv_few(KvPages p, KvSeqs b, KvRows q, KvRows out, int heads, int group,
                                                           float scale2, int chunk, int tiles, int vec, KvParts w) {
    using F = Few<D, Q8, BF>;
    using E = typename F::E;
    using T = typename std::conditional<BF, __bf16, float>::type;
    constexpr int ROWS = 16 * MT, SC = 2 * F::NG * FEW_KEYS;
    __shared__ __align__(16) float so[FEW_WAVES * ROWS * D]; // the loop's scales, then the waves' results
    __shared__ float sm[FEW_WAVES][ROWS], sl[FEW_WAVES][ROWS];
    static_assert(SC <= ROWS * D, "the scales fit");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, h = lane >> 4;
    // The later splits, which a short sequence does not have, come last: blocks
    // are dealt to the CUs in turn, and with a sequence's splits next to each
    // other some got three with keys and others none (32 sessions of 256 to
    // 2048 keys: the median block took 13 us, the last 20).  Within a split the
    // tiles with the most keys first.
    int y = blockIdx.x;
    const int seq = y % b.n_seq;
    y /= b.n_seq;
    const int kh = y % p.hk;
    y /= p.hk;
    const int tile = tiles - 1 - y % tiles, split = y / tiles;
    const int k0 = split * chunk, step = FEW_WAVES * FEW_KEYS;
    int key = k0 + wave * FEW_KEYS;
    const int *table = b.table + seq * b.stride;
    FewPages pg = few_pages(p, table, b.pages, key);         // (beside the lengths' loads)
    const KvSeq s = kv_seq(b, seq, p.shift);
    const int nr = s.n < b.max_rows ? s.n : b.max_rows;
    if ((long long)tile * ROWS >= (long long)nr * group) return;
    const int j_first = tile * ROWS / group;
    int j_last = (tile * ROWS + ROWS - 1) / group;
    j_last = j_last < nr ? j_last : nr - 1;
    int end = s.pos0 + j_last + 1;                           // of the tile's keys
    end = end < s.len ? end : s.len;
    int k1 = k0 + chunk;
    k1 = k1 < end ? k1 : end;
    if (k0 >= k1 && w.splits > 1) {                          // no keys: the join skips this part
        const int row = tile * ROWS + threadIdx.x, j = row / group, r = s.r0 + j;
        if (threadIdx.x < ROWS && j < nr && (unsigned)r < (unsigned)b.n_rows) {
            const long long at = ((long long)r * heads + kh * group + row % group) * w.splits + split;
            *(float2 *)(w.ml + 2 * at) = make_float2(ninf(), 0.0f);
        }
        return;
    }

    const FewAddr<D, Q8, BF> addr(p, kh);
    FewTile<D, Q8, BF> tl;
    if (key < k1) {
        addr.load_k(tl, p, pg, key);
        addr.load_v(tl, p, pg, key);
    }

    FewAcc<D, Q8, BF, MT> A;
#pragma unroll
    for (int m = 0; m < MT; m++) {
        const int row = tile * ROWS + m * 16 + n, j = row / group, r = s.r0 + j;
        const bool on = j < nr && (unsigned)r < (unsigned)b.n_rows;
        const T *src = (const T *)q.p + (on ? r * q.row + (kh * group + row % group) * q.head : 0);
        A.lim[m] = on ? (s.pos0 + j + 1 < s.len ? s.pos0 + j + 1 : s.len) : 0;
        A.m[m] = FEW_NONE;
        A.l[m] = 0.0f;
        A.huge = false;
#pragma unroll
        for (int d = 0; d < F::NT; d++) A.o[m][d] = f32x4{0, 0, 0, 0};
        float x[F::NG][8];
        uint32_t big = 0;
#pragma unroll
        for (int c = 0; c < F::NG; c++)
            load8(src + F::dim(c, h), vec, x[c]);
#pragma unroll
        for (int c = 0; c < F::NG; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c][i] = on ? x[c][i] : 0.0f;
                const uint32_t a = u_from_f(x[c][i]) & 0x7FFFFFFFu;
                big = a > big ? a : big;
            }
        // a negative scale turns q around, so that the factor of the scores is
        // not negative; nor zero, so that -inf stays what it is
        A.cq[m] = fabsf(scale2);
        float unit = scale2 < 0.0f ? -1.0f : 1.0f;
        if (Q8) {
            uint32_t y = __shfl_xor(big, 16);
            big = y > big ? y : big;
            y = __shfl_xor(big, 32);
            big = y > big ? y : big;
            const int e = (int)(big >> 23) - 127 - 14;       // the row's largest to [2^14, 2^15)
            A.cq[m] = __builtin_amdgcn_ldexpf(A.cq[m], e + 9);
#pragma unroll
            for (int c = 0; c < F::NG; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) x[c][i] = __builtin_amdgcn_ldexpf(x[c][i], -e);
        }
        A.cq[m] = fmaxf(A.cq[m], 1e-37f);
#pragma unroll
        for (int c = 0; c < F::NG; c++)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                uint32_t y[F::NQ];
                parts2<E, F::NQ>(x[c][i] * unit, x[c][i + 1] * unit, y);
#pragma unroll
                for (int k = 0; k < F::NQ; k++) A.q[m][c][k][i / 2] = y[k];
            }
    }
    // keys below this are attended by every row of the tile
    int all = s.pos0 + j_first + 1;
    all = all < s.len ? all : s.len;
    float *sc = so + wave * ROWS * D;
    while (key < k1) {
        const int next = key + step;
        const bool there0 = (unsigned)pg.id[0] < (unsigned)p.n_pages, there1 = (unsigned)pg.id[1] < (unsigned)p.n_pages;
        const bool masked = key + FEW_KEYS > all || !there0 || !there1;
        float vex = 0.0f;
        if (Q8) {
            // the wave's own part of LDS: written whole, then read by every lane
            if (masked) {
                const int k4 = key + (lane & 7) * 4;
#pragma unroll
                for (int i = 0; i < 4; i++) tl.sc[i] = k4 + i < s.len ? tl.sc[i] : 0.0f;
            }
            if (lane < 2 * F::NG * 8) *(f32x4 *)(sc + lane * 4) = tl.sc;
            if (!masked) {
                const float x = fmaxf(fmaxf(tl.sc[0], tl.sc[1]), fmaxf(tl.sc[2], tl.sc[3]));
                vex = (float)((int)(wave_max_bits(lane >= F::NG * 8 && lane < 2 * F::NG * 8 ? u_from_f(x) : 0u) >> 23) - 126);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        // the last turn loads its own tile again, without a branch: registers
        // that are loaded on one of two paths came out of the compiler
        // overwritten before their last use
        const int ahead = next < k1 ? next : key;
        pg = few_pages(p, table, b.pages, ahead);
        f32x4 x[MT][2];
        few_scores<D, Q8, BF, MT>(A, tl, sc, x);
        addr.load_k(tl, p, pg, ahead);
        few_values<D, Q8, BF, MT>(A, tl, sc, x, key, s.len, there0, there1, masked, vex);
        addr.load_v(tl, p, pg, ahead);
        key = next;
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
        float mx = FEW_NONE;
#pragma unroll
        for (int x = 0; x < FEW_WAVES; x++) mx = fmaxf(mx, sm[x][m * 16 + n]);
        const float f = kv_exp2(A.m[m] - mx);
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
    float mx = FEW_NONE, l = 0.0f, x[DT];
#pragma unroll
    for (int y = 0; y < FEW_WAVES; y++) mx = fmaxf(mx, sm[y][m]);
#pragma unroll
    for (int y = 0; y < FEW_WAVES; y++) l += sl[y][m] * kv_exp2(sm[y][m] - mx);
#pragma unroll
    for (int i = 0; i < DT; i++) {
        x[i] = 0.0f;
#pragma unroll
        for (int y = 0; y < FEW_WAVES; y++) x[i] += so[(y * ROWS + m) * D + d0 + i];
        if (Q8) x[i] *= 512.0f;                              // the codes' 2^-9
    }
    if (w.splits == 1) {
        T *dst = (T *)out.p + r * out.row + head * out.head + d0;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < DT; i++) dst[i] = (T)(x[i] * inv);
        return;
    }
    const long long at = ((long long)r * heads + head) * w.splits + split;
    if (d0 == 0) {
        w.ml[2 * at] = mx == FEW_NONE && l == l ? ninf() : mx;   // (scores that are all NaN leave mx, and are not no keys)
        w.ml[2 * at + 1] = l;
    }
    if (mx != FEW_NONE)
#pragma unroll
        for (int i = 0; i < DT; i++) w.o[at * D + d0 + i] = x[i];
}

// out = sum over splits of 2^(M_s - M) o_s / sum of 2^(M_s - M) l_s, in split
// order within a lane and then over the lanes: one block per (row, head).
#define JOIN_THREADS 256
#define JOIN_MOST 1024            // splits
template <int D, bool BF>
__global__ __launch_bounds__(JOIN_THREADS) void k_kv_join(KvSeqs b, KvRows out, int heads, KvParts w) {
    using T = typename std::conditional<BF, __bf16, float>::type;
    constexpr int L = D / 4, G = JOIN_THREADS / L, U = 4;    // lanes of a split, splits at a time, loads in flight
    __shared__ __align__(16) float so[G][D];
    __shared__ float sf[JOIN_MOST], sl[JOIN_THREADS / 64], sm[JOIN_THREADS / 64];
    const int j = blockIdx.x / heads, head = blockIdx.x % heads, seq = blockIdx.y, tid = threadIdx.x;
    const int r0 = b.row0[seq], nr = b.row0[seq + 1] - r0, r = r0 + j;
    if (j >= nr || (unsigned)r >= (unsigned)b.n_rows) return;
    const long long at = ((long long)r * heads + head) * w.splits;
    float m[JOIN_MOST / JOIN_THREADS], l[JOIN_MOST / JOIN_THREADS], mx = ninf(), sum = 0.0f;
#pragma unroll
    for (int u = 0; u < JOIN_MOST / JOIN_THREADS; u++) {
        const int i = tid + u * JOIN_THREADS;
        const float2 x = i < w.splits ? *(const float2 *)(w.ml + 2 * (at + i)) : make_float2(ninf(), 0.0f);
        m[u] = x.x;
        l[u] = x.y;
        mx = fmaxf(mx, x.x);
    }
    for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
    if ((tid & 63) == 0) sm[tid >> 6] = mx;
    __syncthreads();
    for (int i = 0; i < JOIN_THREADS / 64; i++) mx = fmaxf(mx, sm[i]);
#pragma unroll
    for (int u = 0; u < JOIN_MOST / JOIN_THREADS; u++) {
        const int i = tid + u * JOIN_THREADS;
        const float f = m[u] == ninf() ? 0.0f : kv_exp2(m[u] - mx);
        if (i < w.splits) sf[i] = m[u] == ninf() ? -1.0f : f;      // -1: no keys, its o is not written
        sum += m[u] == ninf() ? 0.0f : l[u] * f;
    }
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
    if ((tid & 63) == 0) sl[tid >> 6] = sum;
    __syncthreads();
    const int g = tid / L, d = tid % L * 4;
    f32x4 acc = {0, 0, 0, 0};
    for (int i0 = g; i0 < w.splits; i0 += U * G) {
        f32x4 x[U];
        float f[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * G < w.splits ? i0 + u * G : i0;
            f[u] = i0 + u * G < w.splits ? sf[i] : -1.0f;
            x[u] = *(const f32x4 *)(w.o + (at + i) * D + d);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] += f[u] == -1.0f ? 0.0f : x[u][e] * f[u];
    }
    *(f32x4 *)&so[g][d] = acc;
    __syncthreads();
    if (tid < D) {
        float x = 0.0f, y = 0.0f;
#pragma unroll
        for (int i = 0; i < G; i++) x += so[i][tid];
#pragma unroll
        for (int i = 0; i < JOIN_THREADS / 64; i++) y += sl[i];
        ((T *)out.p + r * out.row + head * out.head)[tid] = (T)(y == 0.0f ? 0.0f : x / y);
    }
}

// The same for up to JOIN_FEW splits, whose parts a wave's registers hold at
// once: one wave per (row, head), four of them in a block, without a barrier (4
// rows of 32 sequences in 4 parts: 3.6 us, a block each 4.4; one row in 123
// parts takes 4.6 by a block).
#define JOIN_FEW 16
template <int D, bool BF>
__global__ __launch_bounds__(256) void k_kv_join_few(KvSeqs b, KvRows out, int heads, KvParts w) {
    using T = typename std::conditional<BF, __bf16, float>::type;
    constexpr int E = D >= 64 ? D / 64 : 1;                  // dimensions of a lane
    const long long x = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int j = (int)(x / heads), head = (int)(x % heads), seq = blockIdx.y, lane = threadIdx.x & 63;
    const int r0 = b.row0[seq], nr = b.row0[seq + 1] - r0, r = r0 + j;
    if (j >= nr || j >= b.max_rows || (unsigned)r >= (unsigned)b.n_rows) return;
    const long long at = ((long long)r * heads + head) * w.splits;
    const int d = lane * E < D ? lane * E : 0;
    float o[JOIN_FEW][E];
#pragma unroll
    for (int i = 0; i < JOIN_FEW; i++)                       // (of a split without keys: of any content, not used)
#pragma unroll
        for (int e = 0; e < E; e++) o[i][e] = i < w.splits ? w.o[(at + i) * D + d + e] : 0.0f;
    const float2 ml = lane < w.splits ? *(const float2 *)(w.ml + 2 * (at + lane)) : make_float2(ninf(), 0.0f);
    float mx = ml.x;
#pragma unroll
    for (int y = 1; y < JOIN_FEW; y <<= 1) mx = fmaxf(mx, __shfl_xor(mx, y));
    const float f = ml.x == ninf() ? 0.0f : kv_exp2(ml.x - mx);
    float l = ml.x == ninf() ? 0.0f : ml.y * f, acc[E] = {};
#pragma unroll
    for (int y = 1; y < JOIN_FEW; y <<= 1) l += __shfl_xor(l, y);
    l = __shfl(l, 0);
#pragma unroll
    for (int i = 0; i < JOIN_FEW; i++) {
        const float g = __shfl(f, i), m = __shfl(ml.x, i);
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] += m == ninf() ? 0.0f : o[i][e] * g;
    }
    if (lane * E >= D) return;
    T *dst = (T *)out.p + r * out.row + head * out.head + d;
#pragma unroll
    for (int e = 0; e < E; e++) dst[e] = (T)(l == 0.0f ? 0.0f : acc[e] / l);
}

// ---------------------------------------------------------- host glue ---

namespace {

// How a call's work is cut.  rows: of a block's tile; tiles: of a sequence and
// kv head; chunk: keys of a block; splits: blocks of a tile.
KvPlan plan(const KvPages &p, const KvSeqs &b, int heads, int bf16) {
    KvPlan x;
    const long long rows = (long long)b.max_rows * (heads / p.hk);
    // The prompts' kernels where there is enough to do for their large blocks and
    // two launches: above 256 rows, and 2^18 (32-row tile, key) pairs.  Measured
    // (4 kv heads, Q8, width 128, few rows' kernels : prompts'): below, 128 new
    // rows of 4 heads alone 11 : 17 us, 512 of them 17 : 27, 256 of them at 2000
    // keys 33 : 37, 256 each of 4 sequences 17 : 21; above, 384 at 2000 keys 46 :
    // 39, 384 each of 4 sequences 27 : 25, 512 each 36 : 29, at 2000 keys 108 : 89;
    // 64 new rows of 32 sequences at 4000 keys (256 rows) 175 : 239.
    const long long few = (long long)b.n_seq * p.hk * ((rows + 31) / 32);
    x.many = bf16 && rows > 256 && (double)few * b.max_len > 262144.0;
    // A block takes 512 keys or more: less costs more in starting and joining
    // than it gives (300 keys of one session: 6.9 us in one block per head, 5.8
    // and 3.1 for the join in two).
    const int unit = x.many ? 64 : FEW_WAVES * FEW_KEYS, least = 512;
    // Blocks of 256 rows where they fill the chip, else of 128 (4 prompts of 512
    // tokens, 4 kv heads of 128: 128 blocks of 256 rows 30.2 us, 256 of 128 29.4; of
    // 1024 tokens 256 blocks 49, 512 of 128 rows 55; of 4096 tokens 317 and 499).
    if (x.many) x.rows = (long long)b.n_seq * p.hk * ((rows + 255) / 256) >= 256 ? 256 : 128;
    else x.rows = rows <= 16 ? 16 : 32;
    x.tiles = (int)((rows + x.rows - 1) / x.rows);
    const long long base = (long long)b.n_seq * p.hk * x.tiles;
    // Blocks wanted: 256 of many rows, which have a CU each.  Of few rows two per
    // CU for one sequence (8 rows at 250,015 keys: 256 blocks 72 us, 492 63, 980
    // 74), but no splits where the tiles alone fill the chip (512 fp32 rows at
    // 4096, 256 tiles: 80 us, with two splits 74 and 12 for the join); four for
    // several, whose lengths differ (100 sessions of 1 to 5000 keys: 800 blocks
    // 122 us, 1200 110, 2400 109).
    const long long want = x.many ? 256 : b.n_seq > 1 ? 1024 : base >= 256 ? base : 512;
    long long splits = (want + base - 1) / base;
    const long long most = (b.max_len + least - 1) / least;
    splits = splits < most ? splits : most;
    splits = splits < JOIN_MOST ? splits : JOIN_MOST;
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
    const int es = BF ? 2 : 4, vec = (uintptr_t)q.p % 16 == 0 && q.row * es % 16 == 0 && q.head * es % 16 == 0;
    const dim3 grid((unsigned)((long long)x.splits * p.hk * x.tiles * b.n_seq));
    if (x.rows == 16)
        hipLaunchKernelGGL((k_kv_few<D, Q8, BF, 1>), grid, dim3(FEW_THREADS), 0, st, p, b, q, o, heads, heads / p.hk,
                           scale2, x.chunk, x.tiles, vec, w);
    else
        hipLaunchKernelGGL((k_kv_few<D, Q8, BF, 2>), grid, dim3(FEW_THREADS), 0, st, p, b, q, o, heads, heads / p.hk,
                           scale2, x.chunk, x.tiles, vec, w);
    return (int)hipGetLastError();
}

template <int D>
int attend(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads, int bf16, float scale,
           void *ws, hipStream_t st) {
    const KvPlan x = plan(p, b, heads, bf16);
    KvParts w;
    w.splits = x.splits;
    w.o = (float *)((char *)ws + (x.many ? l98k_kv_many_ws(p, b) : 0));
    w.ml = w.o + (long long)b.n_rows * heads * x.splits * D;
    const float scale2 = scale * 1.44269504088896341f;
    const long long blocks = (long long)x.splits * p.hk * x.tiles * b.n_seq, joins = (long long)b.max_rows * heads;
    if (blocks > INT_MAX || joins > INT_MAX) return -1;
    int rc;
    if (x.many) rc = l98k_kv_many(p, q8, b, q, o, heads, scale2, x, w, ws, st);
    else if (q8) rc = bf16 ? few<D, true, true>(p, b, q, o, heads, scale2, x, w, st)
                           : few<D, true, false>(p, b, q, o, heads, scale2, x, w, st);
    else rc = bf16 ? few<D, false, true>(p, b, q, o, heads, scale2, x, w, st)
                   : few<D, false, false>(p, b, q, o, heads, scale2, x, w, st);
    if (rc || x.splits == 1) return rc;
#define JOIN_LAUNCH(K, BF, N) \
    hipLaunchKernelGGL((K<D, BF>), dim3((unsigned)(N), b.n_seq), dim3(JOIN_THREADS), 0, st, b, o, heads, w)
    if (x.splits <= JOIN_FEW) {
        if (bf16) JOIN_LAUNCH(k_kv_join_few, true, (joins + 3) / 4);
        else JOIN_LAUNCH(k_kv_join_few, false, (joins + 3) / 4);
    } else {
        if (bf16) JOIN_LAUNCH(k_kv_join, true, joins);
        else JOIN_LAUNCH(k_kv_join, false, joins);
    }
    return (int)hipGetLastError();
}

}  // namespace

extern "C" long long l98k_kv_attend_ws(const KvPages &p, int, const KvSeqs &b, int heads, int bf16) {
    const KvPlan x = plan(p, b, heads, bf16);
    return (x.many ? l98k_kv_many_ws(p, b) : 0) + (x.splits == 1 ? 0 : (long long)b.n_rows * heads * x.splits * (p.d + 2) * 4);
}

extern "C" int l98k_kv_attend(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads,
                              int bf16, float scale, void *ws, hipStream_t st) {
    if (p.d == 32) return attend<32>(p, q8, b, q, o, heads, bf16, scale, ws, st);
    if (p.d == 64) return attend<64>(p, q8, b, q, o, heads, bf16, scale, ws, st);
    if (p.d == 128) return attend<128>(p, q8, b, q, o, heads, bf16, scale, ws, st);
    return -1;
}
