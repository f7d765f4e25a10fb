// Causal attention of many new rows over the paged key-value cache, bf16 rows.
//
// The bound is the matrix cores: a block takes 32 NW rows of one (sequence, kv
// head), 32 for each of its waves, and goes over the keys in tiles of 64 that
// all waves share.  A tile comes from its pages into registers one tile ahead
// and from there, converted, into one of two LDS buffers: K as [key][dim], V
// transposed as [dim][key], 16-byte chunks permuted so that the fragments'
// reads are free of bank conflicts.  S^T = K Q^T and O^T += V^T P^T by 32 x 32 x
// 16 instructions: a lane's S^T (query lane & 31) is the second product's
// operand as it stands, with V's keys in the order 0-3, 8-11, 4-7, 12-15 of
// each 16.
//
// Q8 goes through fp16: q scaled per row by a power of two (exact for bf16), K
// and V as code * scale * 2^(6 - E) with E of the tile's largest scale (K) and
// of the largest so far (V; the sums are rescaled when it grows), two roundings
// of 2^-11 against the output's 2^-8; numbers below 2^-27 of the largest lose
// bits.  bf16 caches are used as they are.  Weights are rounded to the same 16
// bits, and their sum, in fp32, is of the rounded ones.
//
// The running maximum is raised only where a tile exceeds it by 2^8 (weights
// stay below 2^8): the sums are rescaled a few times per row instead of once
// per tile.
#include <limits.h>

#include <type_traits>

#include "l98_devmath.h"
#include "l98_kv.h"
#include "l98_kvattn.h"

#define MANY_KEYS 64

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {   // packed fp16 product
    f16x2 x, y;
    __builtin_memcpy(&x, &a, 4);
    __builtin_memcpy(&y, &b, 4);
    x = x * y;
    uint32_t r;
    __builtin_memcpy(&r, &x, 4);
    return r;
}
__device__ __forceinline__ float finite_or_0(float x) {
    return (u_from_f(x) & 0x7F800000u) == 0x7F800000u ? 0.0f : x;
}
__device__ __forceinline__ int exp_above(uint32_t bits) { return (int)(bits >> 23) - 126; }   // 2^this > the float >= 0
// the wave's largest of each half of x, in both halves of the result: by DPP, over rows of 16, then over the rows
__device__ __forceinline__ uint32_t wave_max2(uint32_t x) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    auto step = [&](uint32_t y) {
        u16x2 p, q;
        __builtin_memcpy(&p, &x, 4);
        __builtin_memcpy(&q, &y, 4);
        p = __builtin_elementwise_max(p, q);
        __builtin_memcpy(&x, &p, 4);
    };
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true));   // row_shr:1
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true));
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, true));   // row_bcast:15 into rows 1, 3
    step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, true));   // row_bcast:31 into rows 2, 3
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
// c + the two fp16 or bf16 numbers of x
template <class E> __device__ __forceinline__ float add2(uint32_t x, float c);
template <> __device__ __forceinline__ float add2<_Float16>(uint32_t x, float c) {
    f16x2 v;
    __builtin_memcpy(&v, &x, 4);
    return __builtin_amdgcn_fdot2(v, (f16x2){(_Float16)1.0f, (_Float16)1.0f}, c, false);
}
template <> __device__ __forceinline__ float add2<__bf16>(uint32_t x, float c) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x2 v;
    __builtin_memcpy(&v, &x, 4);
    return __builtin_amdgcn_fdot2_f32_bf16(v, (bf16x2){(__bf16)1.0f, (__bf16)1.0f}, c, false);
}

// A 64-key tile's share of a thread, on its way from the pages to LDS.
template <int D, bool Q8, int NT>
struct Stage {
    static constexpr int ES = Q8 ? 1 : 2;
    static constexpr int KROW = D * ES / 16;                 // 16-byte units of a K row
    static constexpr int VROW = D / 4;                       // 4-number units of a V row
    static constexpr int KT = MANY_KEYS * KROW, VT = MANY_KEYS / 4 * VROW;
    static constexpr int KU = (KT + NT - 1) / NT, VU = (VT + NT - 1) / NT;
    static constexpr int G = D / 32;
    static constexpr int SG = D == 32 ? 1 : 2;               // groups of a V unit's four bytes
    u32x4 k[KU];
    uint32_t v[VU][4][ES];
    float ks[Q8 ? KU : 1][2];
    f32x4 vs[Q8 ? VU : 1][SG];
    f32x4 kall, vall;                                        // this lane's share of all the tile's scales
    uint32_t hole;                                           // bit i: keys 16 i .. of the tile have no page
};

// The pages of a tile's four 16-key quarters (uniform: scalar loads).
struct ManyPages {
    int id[4];
    uint32_t hole;
};
__device__ __forceinline__ ManyPages many_pages(const KvPages &p, const int *table, int pages, int key) {
    ManyPages x;
    x.hole = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int at = (key + 16 * i) >> p.shift, id = at < pages ? table[at] : -1;
        const bool there = (unsigned)id < (unsigned)p.n_pages;
        if (!there) x.hole |= 1u << i;
        x.id[i] = there ? id : 0;
    }
    return x;
}

template <int D, bool Q8, int NT>
__device__ __forceinline__ void many_load(Stage<D, Q8, NT> &S, const KvPages &p, const ManyPages &pg, int kh, int key) {
    using T = Stage<D, Q8, NT>;
    const uint32_t rows = 1u << p.shift, vo = (uint32_t)p.hk << p.shift, tid = threadIdx.x, at0 = (uint32_t)key & (rows - 1);
    const uint32_t unit = (uint32_t)(p.page_bytes >> 4), scales = 2 * vo * D, head = (uint32_t)kh << p.shift;
    S.hole = pg.hole;
    const uint32_t id0 = pg.id[0], id1 = pg.id[1], id2 = pg.id[2], id3 = pg.id[3];
    auto page = [=](uint32_t k) {                            // of the tile's key k
        const uint32_t a = k & 16 ? id1 : id0, c = k & 16 ? id3 : id2, id = k & 32 ? c : a;
        return p.data + (((uint64_t)id * unit) << 4);
    };
    auto row = [&](uint32_t k) { return (at0 + k) & (rows - 1); };
#pragma unroll
    for (int u = 0; u < T::KU; u++) {
        const uint32_t x = u * NT + tid, k = x / T::KROW % MANY_KEYS, c = x % T::KROW;
        const unsigned char *pk = page(k);
        S.k[u] = *(const u32x4 *)(pk + ((head + row(k)) * (D * T::ES) + c * 16));
        if (Q8) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t g = (2 * c + i) % T::G;       // chunk h G + g holds 8 numbers of group g
                S.ks[u][i] = *(const float *)(pk + (scales + (((kh * T::G + g) << p.shift) + row(k)) * 4));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < T::VU; u++) {
        const uint32_t x = u * NT + tid, k = x / T::VROW * 4 % MANY_KEYS, c = x % T::VROW;
        const unsigned char *pv = page(k), *s = pv + ((vo + head + row(k)) * (D * T::ES) + c * 4 * T::ES);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (Q8) {
                S.v[u][i][0] = *(const uint32_t *)(s + i * (D * T::ES));
            } else {
                const uint2 y = *(const uint2 *)(s + i * (D * T::ES));
                S.v[u][i][0] = y.x;
                S.v[u][i][T::ES - 1] = y.y;
            }
        }
        if (Q8) {
            const uint32_t g = D == 32 ? 0 : (4 * c) % (D / 16) / 2;         // byte n (D/16) + t: group t / 2
#pragma unroll
            for (int i = 0; i < T::SG; i++)
                S.vs[u][i] = *(const f32x4 *)(pv + (scales + ((((p.hk + kh) * T::G + g + i) << p.shift) + row(k)) * 4));
        }
    }
    if (Q8) {
        // every wave over all of the tile's scales, so that all know the same exponents
        const uint32_t lane = tid & 63, k = (lane & 15) * 4, g = (lane >> 4) % T::G;
        const unsigned char *s = page(k) + (scales + (((kh * T::G + g) << p.shift) + row(k)) * 4);
        S.kall = *(const f32x4 *)s;
        S.vall = *(const f32x4 *)(s + (vo * T::G) * 4);
    }
}

// Exponents above the tile's K and V scales, of the keys that exist.
template <int D, bool Q8, int NT>
__device__ __forceinline__ void many_exps(Stage<D, Q8, NT> &S, int key, int len, bool masked, int &ek, int &ev) {
    if (masked) {
        const int k = (threadIdx.x & 15) * 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = key + k + i < len && !(S.hole >> (k >> 4) & 1);
            S.kall[i] = in ? finite_or_0(S.kall[i]) : 0.0f;
            S.vall[i] = in ? finite_or_0(S.vall[i]) : 0.0f;
        }
    }
    const float a = fmaxf(fmaxf(S.kall[0], S.kall[1]), fmaxf(S.kall[2], S.kall[3]));
    const float c = fmaxf(fmaxf(S.vall[0], S.vall[1]), fmaxf(S.vall[2], S.vall[3]));
    const uint32_t x = wave_max2(__builtin_amdgcn_perm(u_from_f(a), u_from_f(c), 0x07060302u));
    ek = exp_above(x & 0xFFFF0000u);
    ev = exp_above(x << 16);
}

// 16-byte chunk c of row r (of CH chunks) in LDS: rows of less than 256 bytes
// share the banks, so the permutation changes with every 256 bytes
template <int CH>
__device__ __forceinline__ int chunk_at(int r, int c) {
    return r * CH + (c ^ (CH >= 16 ? r & 15 : (r / (16 / CH)) & (CH - 1)));
}

template <int D>
struct ManyLds {
    uint16_t k[2][MANY_KEYS * D], v[2][MANY_KEYS * D];
    uint32_t bad[3][2];                                      // keys of a masked tile whose V is not finite, by tile % 3
};

template <int D, bool Q8, int NT>
__device__ __forceinline__ void many_store(Stage<D, Q8, NT> &S, ManyLds<D> &L, int buf, int turn, int key, int len, bool masked,
                                           int ek, int ev) {
    using T = Stage<D, Q8, NT>;
    const int tid = threadIdx.x;
#pragma unroll
    for (int u = 0; u < T::KU; u++) {
        const int x = u * NT + tid;
        const int k = x / T::KROW, c = x % T::KROW;
        if (T::KT % NT && x >= T::KT) break;
        if (Q8) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float f = __builtin_amdgcn_ldexpf(S.ks[u][i], 15 - ek);
                const uint32_t ff = pack2<_Float16>(f, f);
                u32x4 o;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    o[2 * w] = mul2(codes2(0, S.k[u][2 * i + w], 0x0c010c00u), ff);
                    o[2 * w + 1] = mul2(codes2(0, S.k[u][2 * i + w], 0x0c030c02u), ff);
                }
                *(u32x4 *)&L.k[buf][chunk_at<D / 8>(k, 2 * c + i) * 8] = o;
            }
        } else {
            *(u32x4 *)&L.k[buf][chunk_at<D / 8>(k, c) * 8] = S.k[u];
        }
    }
#pragma unroll
    for (int u = 0; u < T::VU; u++) {
        const int x = u * NT + tid;
        if (T::VT % NT && x >= T::VT) break;
        const int k = x / T::VROW * 4, c = x % T::VROW;
        if (masked) {
            const bool hole = S.hole >> (k >> 4) & 1;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                bool bad = false;
                const bool gone = hole || key + k + i >= len;
                if (Q8) {
#pragma unroll
                    for (int g = 0; g < T::SG; g++) bad = bad || (u_from_f(S.vs[u][g][i]) & 0x7F800000u) == 0x7F800000u;
#pragma unroll
                    for (int g = 0; g < T::SG; g++) S.vs[u][g][i] = gone || bad ? 0.0f : S.vs[u][g][i];
                } else {
#pragma unroll
                    for (int w = 0; w < T::ES; w++)
                        bad = bad || (S.v[u][i][w] & 0x7F80u) == 0x7F80u || (S.v[u][i][w] & 0x7F800000u) == 0x7F800000u;
#pragma unroll
                    for (int w = 0; w < T::ES; w++) S.v[u][i][w] = gone || bad ? 0u : S.v[u][i][w];
                }
                if (bad && !gone) atomicOr(&L.bad[turn][(k + i) >> 5], 1u << ((k + i) & 31));
            }
        }
        // the quad's place: 0-3, 8-11, 4-7, 12-15 of each 16 keys
        const int r = (k >> 2) & 3, slot = (k >> 4) * 16 + ((r & 1) * 2 + (r >> 1)) * 4;
        uint32_t f[T::SG][2];
        if (Q8) {
#pragma unroll
            for (int g = 0; g < T::SG; g++)
#pragma unroll
                for (int w = 0; w < 2; w++)
                    f[g][w] = pack2<_Float16>(__builtin_amdgcn_ldexpf(S.vs[u][g][2 * w], 15 - ev),
                                              __builtin_amdgcn_ldexpf(S.vs[u][g][2 * w + 1], 15 - ev));
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int pos = 4 * c + e;
            uint2 o;
            int dim;
            if (Q8) {
                dim = pos % (D / 16) * 16 + pos / (D / 16);
                const int g = T::SG == 1 ? 0 : e >> 1;
                const uint32_t sel = 0x0c040c00u + (uint32_t)e * 0x00010001u;
                o.x = mul2(codes2(S.v[u][1][0], S.v[u][0][0], sel), f[g][0]);
                o.y = mul2(codes2(S.v[u][3][0], S.v[u][2][0], sel), f[g][1]);
            } else {
                dim = pos;
                const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                constexpr int H = T::ES - 1;
                o.x = __builtin_amdgcn_perm(S.v[u][1][e >> 1 ? H : 0], S.v[u][0][e >> 1 ? H : 0], sel);
                o.y = __builtin_amdgcn_perm(S.v[u][3][e >> 1 ? H : 0], S.v[u][2][e >> 1 ? H : 0], sel);
            }
            *(uint2 *)&L.v[buf][chunk_at<8>(dim, slot >> 3) * 8 + (slot & 7)] = o;
        }
    }
}

template <int D, bool Q8, int NW>
__global__ __launch_bounds__(NW * 64, 2) void k_kv_many(KvPages p, KvSeqs b, KvRows q, KvRows out, int heads, int group,
                                                        float scale2, int chunk, int tiles, int vec, KvParts w) {
    using E = typename std::conditional<Q8, _Float16, __bf16>::type;
    using V8 = typename std::conditional<Q8, f16x8, bf16x8>::type;
    constexpr int NT = NW * 64, ROWS = NW * 32, KK = D / 16, DT = D / 32;
    __shared__ __align__(16) ManyLds<D> L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int seq = blockIdx.y, split = blockIdx.x % w.splits, y = blockIdx.x / w.splits;
    const int kh = y % p.hk, tile = tiles - 1 - y / p.hk;
    const KvSeq s = kv_seq(b, seq, p.shift);
    const int nr = s.n < b.max_rows ? s.n : b.max_rows;
    if ((long long)tile * ROWS >= (long long)nr * group) return;
    auto end_of = [&](int row) {                             // keys of the rows up to `row`
        int j = row / group;
        j = j < nr ? j : nr - 1;
        const int e = s.pos0 + j + 1;
        return e < s.len ? e : s.len;
    };
    const int k0 = split * chunk;
    int k1 = k0 + chunk, wend = end_of(tile * ROWS + wave * 32 + 31);
    const int end = end_of(tile * ROWS + ROWS - 1), all = end_of(tile * ROWS);
    k1 = k1 < end ? k1 : end;
    wend = wend < k1 ? wend : k1;
    const int *table = b.table + seq * b.stride;

    const int row = tile * ROWS + wave * 32 + n, j = row / group, head = kh * group + row % group, r = s.r0 + j;
    const bool on = j < nr && (unsigned)r < (unsigned)b.n_rows;
    const int lim = on ? end_of(row) : 0;
    // a negative scale turns q around, so that the factor of the scores is not negative
    float cq = fabsf(scale2);
    V8 qf[KK];
    {
        const __bf16 *src = (const __bf16 *)q.p + (on ? r * q.row + head * q.head : 0);
        float x[KK][8];
        uint32_t big = 0;
#pragma unroll
        for (int c = 0; c < KK; c++) {
            const int at = 2 * c + h;                        // chunk of 8 in the order of K's rows
            const int d0 = Q8 ? (at % (D / 32)) * 32 + at / (D / 32) * 8 : at * 8;
            bf16x8 t;
            if (vec) {
                t = on ? *(const bf16x8 *)(src + d0) : bf16x8{};
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = on ? src[d0 + i] : (__bf16)0.0f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c][i] = scale2 < 0.0f ? -(float)t[i] : (float)t[i];
                const uint32_t a = u_from_f(x[c][i]) & 0x7FFFFFFFu;
                big = a > big ? a : big;
            }
        }
        int e = 0;
        if (Q8) {
            const uint32_t o = __shfl_xor(big, 32);
            big = o > big ? o : big;
            e = (int)(big >> 23) - 127 - 14;
            cq = __builtin_amdgcn_ldexpf(cq, e - 6);         // K comes with 2^(6 - ek)
        }
#pragma unroll
        for (int c = 0; c < KK; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) qf[c][i] = (E)(Q8 ? __builtin_amdgcn_ldexpf(x[c][i], -e) : x[c][i]);
    }
    f32x16 o[DT] = {};
    float m = ninf(), l = 0.0f;
    int ek = 0, ev = -1000;                                  // exponents of the tile in LDS

    if (k0 < k1) {
        if (threadIdx.x < 6) L.bad[threadIdx.x >> 1][threadIdx.x & 1] = 0;
        __syncthreads();
        int evn = ev, ekn = 0;
        auto bounds = [&](Stage<D, Q8, NT> &S, int key, bool masked) {
            if (!Q8) return;
            int x;
            many_exps<D, Q8, NT>(S, key, s.len, masked, ekn, x);
            evn = evn > x ? evn : x;
        };
        Stage<D, Q8, NT> S;
        ManyPages pg = many_pages(p, table, b.pages, k0);
        bool masked = k0 + MANY_KEYS > all || pg.hole, next_masked;
        many_load<D, Q8, NT>(S, p, pg, kh, k0);
        uint32_t hole = S.hole;
        bounds(S, k0, masked);
        many_store<D, Q8, NT>(S, L, 0, 0, k0, s.len, masked, ekn, evn);
        pg = many_pages(p, table, b.pages, k0 + MANY_KEYS < k1 ? k0 + MANY_KEYS : k0);
        __syncthreads();
        for (int key = k0, buf = 0, turn = 0; key < k1; key += MANY_KEYS, buf ^= 1) {
            const int next = key + MANY_KEYS, turn1 = turn == 2 ? 0 : turn + 1;
            // the flags of the tile before this one, which nobody reads or sets in this turn
            if (threadIdx.x < 2) L.bad[turn == 0 ? 2 : turn - 1][threadIdx.x] = 0;
            if (Q8 && evn != ev) {                           // the V scales' unit grew
                if (ev != -1000) {
                    const float f = __builtin_amdgcn_ldexpf(1.0f, ev - evn);
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] *= f;
                }
                ev = evn;
            }
            ek = ekn;
            // (the last turn loads its own tile again, without a branch)
            many_load<D, Q8, NT>(S, p, pg, kh, next < k1 ? next : key);
            pg = many_pages(p, table, b.pages, next + MANY_KEYS < k1 ? next + MANY_KEYS : key);
            if (key < wend) {
                f32x16 st[2] = {};
#pragma unroll
                for (int c = 0; c < KK; c++)
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const u32x4 a = *(const u32x4 *)&L.k[buf][chunk_at<D / 8>(t * 32 + n, 2 * c + h) * 8];
                        st[t] = mfma32(as<V8>(a), qf[c], st[t]);
                    }
                float c = Q8 ? __builtin_amdgcn_ldexpf(cq, ek) : cq;
                c = fmaxf(c, 1e-37f);                        // -inf * c stays -inf at a scale of zero
                float mx = ninf();
                if (masked) {
                    // (the lane's half taken out first, so that what is compared with is constant:
                    // it would be kept in 64 registers through the whole loop)
                    const uint32_t bad0 = L.bad[turn][0] >> (h * 4), bad1 = L.bad[turn][1] >> (h * 4);
                    const int left = lim - key - h * 4;
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const int k = (i >> 2) * 8 + (i & 3);
                            const bool in = t * 32 + k < left && !(hole >> (2 * t + (i >> 3)) & 1);
                            if (in && ((t ? bad1 : bad0) >> k & 1)) l = __builtin_nanf("");
                            st[t][i] = in ? st[t][i] : ninf();
                        }
                }
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) mx = fmaxf(mx, st[t][i]);
                mx = fmaxf(mx, __shfl_xor(mx, 32)) * c;
                // each row by itself: its bits must not depend on the wave's other rows
                const bool up = mx > m + 8.0f;
                if (__any(up)) {
                    const float mn = up ? mx : m, f = up ? kv_exp2(m - mn) : 1.0f;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] *= f;
                    m = mn;
                }
                const float mu = m == ninf() ? 0.0f : m;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        st[t][i] = kv_exp2(__builtin_fmaf(st[t][i], c, -mu));
                    }
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        u32x4 pw;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            pw[i] = pack2<E>(st[t][u * 8 + 2 * i], st[t][u * 8 + 2 * i + 1]);
                            l = add2<E>(pw[i], l);
                        }
#pragma unroll
                        for (int d = 0; d < DT; d++) {
                            const u32x4 a = *(const u32x4 *)&L.v[buf][chunk_at<8>(d * 32 + n, (t * 2 + u) * 2 + h) * 8];
                            o[d] = mfma32(as<V8>(a), as<V8>(pw), o[d]);
                        }
                    }
            }
            if (next < k1) {
                hole = S.hole;
                next_masked = next + MANY_KEYS > all || hole;
                bounds(S, next, next_masked);
                many_store<D, Q8, NT>(S, L, buf ^ 1, turn1, next, s.len, next_masked, ekn, evn);
                masked = next_masked;
            }
            turn = turn1;
            __syncthreads();
        }
    }
    l += __shfl_xor(l, 32);
    if (!on) return;
    if (Q8) {
        const float f = __builtin_amdgcn_ldexpf(1.0f, ev == -1000 ? 0 : ev - 6);
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= f;
    }
    if (w.splits == 1) {
        __bf16 *dst = (__bf16 *)out.p + r * out.row + head * out.head;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d0 = d * 32 + (i >> 2) * 8 + h * 4;
                uint2 t;
                t.x = pack2<__bf16>(o[d][i] * inv, o[d][i + 1] * inv);
                t.y = pack2<__bf16>(o[d][i + 2] * inv, o[d][i + 3] * inv);
                if (vec) {
                    *(uint2 *)(dst + d0) = t;
                } else {
                    uint16_t *x = (uint16_t *)dst + d0;
                    x[0] = (uint16_t)t.x, x[1] = (uint16_t)(t.x >> 16), x[2] = (uint16_t)t.y, x[3] = (uint16_t)(t.y >> 16);
                }
            }
        return;
    }
    const long long at = ((long long)r * heads + head) * w.splits + split;
    if (h == 0) {
        w.ml[2 * at] = m;
        w.ml[2 * at + 1] = l;
    }
    if (m != ninf())
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(f32x4 *)(w.o + at * D + d * 32 + (i >> 2) * 8 + h * 4) =
                    f32x4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
}

// ---------------------------------------------------------- host glue ---

static bool aligned16(const KvRows &r) {
    return ((uintptr_t)r.p % 16) == 0 && r.row % 8 == 0 && r.head % 8 == 0;
}

template <int D, bool Q8>
static int many(const KvPages &p, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads, float scale2,
                const KvPlan &x, const KvParts &w, hipStream_t st) {
    const int vec = aligned16(q) && aligned16(o);
    const dim3 grid((unsigned)((long long)x.splits * p.hk * x.tiles), b.n_seq);
    if (x.rows == 128)
        hipLaunchKernelGGL((k_kv_many<D, Q8, 4>), grid, dim3(256), 0, st, p, b, q, o, heads, heads / p.hk, scale2, x.chunk,
                           x.tiles, vec, w);
    else
        hipLaunchKernelGGL((k_kv_many<D, Q8, 8>), grid, dim3(512), 0, st, p, b, q, o, heads, heads / p.hk, scale2, x.chunk,
                           x.tiles, vec, w);
    return (int)hipGetLastError();
}

extern "C" int l98k_kv_many(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads,
                            float scale2, const KvPlan &x, const KvParts &w, hipStream_t st) {
#define MANY_D(DD)                                                                  \
    if (p.d == DD)                                                                  \
        return q8 ? many<DD, true>(p, b, q, o, heads, scale2, x, w, st)             \
                  : many<DD, false>(p, b, q, o, heads, scale2, x, w, st)
    MANY_D(32);
    MANY_D(64);
    MANY_D(128);
    return -1;
}
