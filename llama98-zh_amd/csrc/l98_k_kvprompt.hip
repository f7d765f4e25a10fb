// Causal attention of many new rows over the paged key-value cache, bf16 rows.
//
// Two launches.  k_kv_tiles turns each (sequence, kv head)'s keys into tiles of
// 64 in the workspace, as the second one has them in LDS: K as [key][dim], V
// transposed as [dim][key], in 16 bits, 16-byte chunks permuted so that the
// fragments' reads are free of bank conflicts.  It reads the cache once and
// writes 4 dim bytes per key, where each of the blocks below would convert all
// of its keys again (a 16,384-token prompt, 4 kv heads of 128, Q8: 64 times;
// with the conversion in the second kernel its waves issued 230 vector and 87
// scalar instructions per tile beside the 32 matrix ones, and took 1.23 ms).
//
// The tiles too are put together in LDS and stored from there in 16-byte pieces
// (V's 8-byte pieces of 64 rows a store straight to memory: 24,752 keys 27 us, so
// 18, and 17 and 13 for 16,384; the floors are 15 and 10).
//
// k_kv_many: the bound is the matrix cores (a 16,384-token prompt, 16 heads over
// 4 of width 128, Q8: 1.10 ms, 1.0 PFLOP/s; the matrix cores are busy in 48% of
// its cycles, at the 2.0 GHz that the power limit leaves).  A block takes 32 NW rows of one
// (sequence, kv head), 32 for each of its waves, and all waves share the tiles,
// which are loaded straight into LDS two tiles ahead.  S^T = K Q^T and O^T += V^T
// P^T by 32 x 32 x 16 instructions: a lane's S^T (query lane & 31) is the second
// product's operand as it stands, with V's keys in the order 0-3, 8-11, 4-7,
// 12-15 of each 16.
//
// Q8 goes through fp16: q scaled per row by a power of two (exact for bf16), K
// and V as code * (scale * 2^(8 - E)) with E of the tile's largest scale, so two
// roundings of 2^-12 against the output's 2^-9 (the fp16 number 1024 + u is u
// in the low bits of 1024's; less 1152 it is the code).  The sums are in units
// of a V tile's 2^E, rescaled when a tile's is larger or less than 2^-4 of it.
// Scales of down to 2^-22 of their tile's largest are held to full precision,
// smaller ones with an error of 2^-33 of it.  A key behind a row may be of any
// size, and must not take the row's own out of the range: where a tile that
// some row attends in part has a V so much larger than its first key's, where
// the error of K's numbers would show in the scores, and where the tiles' V
// scales differ by 2^60, the block computes its rows again from the pages in
// fp32 (many_slowly: 4096 rows of which all do take 36 ms instead of 0.15).
// bf16 caches are used as they are.  Weights are rounded to the same 16 bits,
// and their sum, in fp32, is of the rounded ones.
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
__device__ __forceinline__ float finite_or_0(float x) {
    return (u_from_f(x) & 0x7F800000u) == 0x7F800000u ? 0.0f : x;
}
__device__ __forceinline__ int exp_above(uint32_t bits) { return (int)(bits >> 23) - 126; }   // 2^this > the float >= 0
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
    f32x4 both[2];                                           // this lane's share of all the tile's scales
};

// The pages of a tile's four 16-key quarters (uniform).
struct ManyPages {
    uint32_t id[4];
    uint32_t hole;                                           // bit i: keys 16 i .. of the tile have no page
};
__device__ __forceinline__ ManyPages many_pages(const KvPages &p, const int *table, int pages, int key) {
    ManyPages x;
    x.hole = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int at = (key + 16 * i) >> p.shift, id = at < pages ? table[at] : -1;
        const bool there = (unsigned)id < (unsigned)p.n_pages;
        if (!there) x.hole |= 1u << i;
        x.id[i] = there ? (uint32_t)id : 0u;
    }
    return x;
}
// Where the tile's key k (the thread's own) has something that lies `lane`
// bytes into the page's block for key 0 and `step` bytes further for each key.
__device__ __forceinline__ const unsigned char *many_at(const KvPages &p, const ManyPages &pg, int key, uint32_t k,
                                                        uint32_t lane, uint32_t step) {
    const uint32_t unit = (uint32_t)(p.page_bytes >> 4), rows = 1u << p.shift, at0 = (uint32_t)key & (rows - 1);
    const uint32_t id0 = pg.id[0], id1 = pg.id[1], id2 = pg.id[2], id3 = pg.id[3];
    const uint32_t a = k & 16 ? id1 : id0, c = k & 16 ? id3 : id2, id = k & 32 ? c : a;
    return p.data + (((uint64_t)id * unit) << 4) + (lane + ((at0 + k) & (rows - 1)) * step);
}

template <int D, bool Q8, int NT>
__device__ __forceinline__ void many_load(Stage<D, Q8, NT> &S, const KvPages &p, const ManyPages &pg, int kh, int key) {
    using T = Stage<D, Q8, NT>;
    const uint32_t tid = threadIdx.x, head = ((uint32_t)kh << p.shift) * (D * T::ES), vo = ((uint32_t)p.hk << p.shift) * (D * T::ES);
#pragma unroll
    for (int u = 0; u < T::KU; u++) {
        const uint32_t x = u * NT + tid, k = x / T::KROW % MANY_KEYS, c = x % T::KROW;
        S.k[u] = *(const u32x4 *)many_at(p, pg, key, k, head + c * 16, D * T::ES);
    }
#pragma unroll
    for (int u = 0; u < T::VU; u++) {
        const uint32_t x = u * NT + tid, k = x / T::VROW * 4 % MANY_KEYS, c = x % T::VROW;
        const unsigned char *s = many_at(p, pg, key, k, vo + head + c * 4 * T::ES, D * T::ES);
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
    }
}

// The Q8 scales of the tile that S holds: the thread's own, and its share of
// all of them (every wave over all of the tile's, so that all know the same
// exponents: lanes 0-31 K's, 32-63 V's).
template <int D, bool Q8, int NT>
__device__ __forceinline__ void many_scales(Stage<D, Q8, NT> &S, const KvPages &p, const ManyPages &pg, int kh, int key) {
    using T = Stage<D, Q8, NT>;
    if (!Q8) return;
    const uint32_t tid = threadIdx.x, scales = 2 * ((uint32_t)p.hk << p.shift) * D;
    // group g: of K kh G + g, of V behind all of K's
    auto scale = [&](uint32_t g, uint32_t k) { return many_at(p, pg, key, k, scales + (g << p.shift) * 4, 4); };
#pragma unroll
    for (int u = 0; u < T::KU; u++) {
        const uint32_t x = u * NT + tid, k = x / T::KROW % MANY_KEYS, c = x % T::KROW;
        // chunk h G + g holds 8 numbers of group g
#pragma unroll
        for (int i = 0; i < 2; i++) S.ks[u][i] = *(const float *)scale(kh * T::G + (2 * c + i) % T::G, k);
    }
#pragma unroll
    for (int u = 0; u < T::VU; u++) {
        const uint32_t x = u * NT + tid, k = x / T::VROW * 4 % MANY_KEYS, c = x % T::VROW;
        const uint32_t g = D == 32 ? 0 : (4 * c) % (D / 16) / 2;             // byte n (D/16) + t: group t / 2
#pragma unroll
        for (int i = 0; i < T::SG; i++) S.vs[u][i] = *(const f32x4 *)scale((p.hk + kh) * T::G + g + i, k);
    }
    // 64 keys of G groups over 32 lanes, 8 of them each
    const uint32_t lane = tid & 31, k = (lane & 7) * 8, g = (lane >> 3) % T::G + (tid & 32 ? p.hk + kh : kh) * T::G;
    const unsigned char *s = scale(g, k);
    S.both[0] = *(const f32x4 *)s;
    S.both[1] = *(const f32x4 *)(s + 16);
}

// Exponents above the tile's K and V scales, of the keys that exist, and
// whether fp16 numbers of that unit are too coarse: bit 0, for the smallest
// scale of K; bit 1, for the first key's of V (a row that attends some of the
// tile attends that one, so what it attends is no smaller).
#define MANY_NONE (-126)                                     // no scale, or none above 2^-126
#define MANY_RANGE 22
template <int D, bool Q8, int NT>
__device__ __forceinline__ void many_exps(Stage<D, Q8, NT> &S, uint32_t hole, int key, int len, int &ek, int &ev, uint32_t &wide) {
    const int k = (threadIdx.x & 7) * 8;
    uint32_t x = 0, y = 0;                                   // the largest, and the smallest above 0 taken from TOP
    constexpr uint32_t TOP = 0x7F800000u;
    const int first = (__ffs((int)~hole) - 1) * 16;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const bool in = key + k + i < len && !(hole >> (k >> 4) & 1);
        const uint32_t v = in ? u_from_f(fmaxf(finite_or_0(S.both[i >> 2][i & 3]), 0.0f)) : 0u;
        const uint32_t w = v && (!(threadIdx.x & 32) || k + i == first) ? TOP - v : 0u;
        x = v > x ? v : x;
        y = w > y ? w : y;
    }
    // over each 32 lanes, into the last of them: by DPP, over rows of 16, then into the odd rows
    auto over = [](uint32_t &x) {
        auto step = [&](uint32_t o) { x = o > x ? o : x; };
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, true));   // row_shr:1
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, true));
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, true));
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, true));
        step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, true));   // row_bcast:15 into rows 1, 3
    };
    over(x);
    over(y);
    ek = exp_above((uint32_t)__builtin_amdgcn_readlane((int)x, 31));
    ev = exp_above((uint32_t)__builtin_amdgcn_readlane((int)x, 63));
    const int lk = exp_above(TOP - (uint32_t)__builtin_amdgcn_readlane((int)y, 31));
    const int lv = exp_above(TOP - (uint32_t)__builtin_amdgcn_readlane((int)y, 63));
    wide = (ek - lk > MANY_RANGE ? 1u : 0u) | (ev - lv > MANY_RANGE ? 2u : 0u);
}

// bytes of lo and hi (sel: a byte of each over zeros), each minus 128, times the halves of f
__device__ __forceinline__ uint32_t scaled2(uint32_t hi, uint32_t lo, uint32_t sel, uint32_t f) {
    const uint32_t u = __builtin_amdgcn_perm(hi, lo, sel) | 0x64006400u;     // as fp16: 1024 + u
    f16x2 x, y;
    __builtin_memcpy(&x, &u, 4);
    __builtin_memcpy(&y, &f, 4);
    x = (x - (f16x2){(_Float16)1152.0f, (_Float16)1152.0f}) * y;
    uint32_t r;
    __builtin_memcpy(&r, &x, 4);
    return r;
}

// 16-byte chunk c of row r (of CH chunks) in LDS: rows of less than 256 bytes
// share the banks, so the permutation changes with every 256 bytes
template <int CH>
__device__ __forceinline__ int chunk_at(int r, int c) {
    return r * CH + (c ^ (CH >= 16 ? r & 15 : (r / (16 / CH)) & (CH - 1)));
}

// What the second launch needs of a tile beside its numbers.
struct ManyHead {
    int ek, ev;                                              // 2^these > every K and V scale of it
    uint32_t bad[2];                                         // keys whose V is not finite (it is zeros in the tile)
    uint32_t hole;                                           // as ManyPages'
    uint32_t wide, unused[2];                                // many_exps'
};

// The tile to k and v, and its keys whose V is not finite to bad (in LDS): a
// key that some row may not attend must not reach it as 0 * NaN.
template <int D, bool Q8, int NT>
__device__ __forceinline__ void many_store(Stage<D, Q8, NT> &S, uint16_t *kt, uint16_t *vt, uint32_t *bads, uint32_t holes,
                                           int key, int len, int ek, int ev) {
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
                const float x = __builtin_amdgcn_ldexpf(S.ks[u][i], 8 - ek);
                const uint32_t f = pack2<_Float16>(x, x);
                u32x4 o;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    o[2 * w] = scaled2(0, S.k[u][2 * i + w], 0x0c010c00u, f);
                    o[2 * w + 1] = scaled2(0, S.k[u][2 * i + w], 0x0c030c02u, f);
                }
                *(u32x4 *)&kt[chunk_at<D / 8>(k, 2 * c + i) * 8] = o;
            }
        } else {
            *(u32x4 *)&kt[chunk_at<D / 8>(k, c) * 8] = S.k[u];
        }
    }
#pragma unroll
    for (int u = 0; u < T::VU; u++) {
        const int x = u * NT + tid;
        if (T::VT % NT && x >= T::VT) break;
        const int k = x / T::VROW * 4, c = x % T::VROW;
        {
            const bool hole = holes >> (k >> 4) & 1;
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
                if (bad && !gone) atomicOr(&bads[(k + i) >> 5], 1u << ((k + i) & 31));
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
                    f[g][w] = ev == MANY_NONE ? 0u
                                              : pack2<_Float16>(__builtin_amdgcn_ldexpf(S.vs[u][g][2 * w], 8 - ev),
                                                                __builtin_amdgcn_ldexpf(S.vs[u][g][2 * w + 1], 8 - ev));
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
                o.x = scaled2(S.v[u][1][0], S.v[u][0][0], sel, f[g][0]);
                o.y = scaled2(S.v[u][3][0], S.v[u][2][0], sel, f[g][1]);
            } else {
                dim = pos;
                const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                constexpr int H = T::ES - 1;
                o.x = __builtin_amdgcn_perm(S.v[u][1][e >> 1 ? H : 0], S.v[u][0][e >> 1 ? H : 0], sel);
                o.y = __builtin_amdgcn_perm(S.v[u][3][e >> 1 ? H : 0], S.v[u][2][e >> 1 ? H : 0], sel);
            }
            *(uint2 *)&vt[chunk_at<8>(dim, slot >> 3) * 8 + (slot & 7)] = o;
        }
    }
}

#define TILE_THREADS 256
// Tile blockIdx.x / hk of sequence blockIdx.y, head blockIdx.x % hk: its place
// in the workspace is (sequence * hk + head) * n + tile.
template <int D>
__device__ __forceinline__ unsigned char *tile_at(unsigned char *ws, int hk, int seq, int head, int n, int tile) {
    return ws + (((long long)seq * hk + head) * n + tile) * (4 * MANY_KEYS * D);
}
template <int D, bool Q8>
__global__ __launch_bounds__(TILE_THREADS) void k_kv_tiles(KvPages p, KvSeqs b, int n, unsigned char *ws, ManyHead *heads) {
    __shared__ uint32_t bad[2];
    __shared__ __align__(16) uint16_t made[2 * MANY_KEYS * D];
    const int seq = blockIdx.y, kh = blockIdx.x % p.hk, tile = blockIdx.x / p.hk, key = tile * MANY_KEYS;
    const KvSeq s = kv_seq(b, seq, p.shift);
    if (key >= s.len || s.n <= 0) return;
    if (threadIdx.x < 2) bad[threadIdx.x] = 0;
    __syncthreads();
    Stage<D, Q8, TILE_THREADS> S;
    const ManyPages pg = many_pages(p, b.table + seq * b.stride, b.pages, key);
    many_load<D, Q8, TILE_THREADS>(S, p, pg, kh, key);
    many_scales<D, Q8, TILE_THREADS>(S, p, pg, kh, key);
    int ek = 0, ev = 0;
    uint32_t wide = 0;
    if (Q8) many_exps<D, Q8, TILE_THREADS>(S, pg.hole, key, s.len, ek, ev, wide);
    many_store<D, Q8, TILE_THREADS>(S, made, made + MANY_KEYS * D, bad, pg.hole, key, s.len, ek, ev);
    __syncthreads();
    u32x4 *out = (u32x4 *)tile_at<D>(ws, p.hk, seq, kh, n, tile);
#pragma unroll
    for (int i = 0; i < 4 * MANY_KEYS * D / 16 / TILE_THREADS; i++)
        out[i * TILE_THREADS + threadIdx.x] = ((const u32x4 *)made)[i * TILE_THREADS + threadIdx.x];
    if (threadIdx.x == 0) {
        ManyHead h = {ek, ev, {bad[0], bad[1]}, pg.hole, wide, {0, 0}};
        heads[((long long)seq * p.hk + kh) * n + tile] = h;
    }
}

typedef const __attribute__((address_space(1))) void *many_gptr;
typedef __attribute__((address_space(3))) void *many_lptr;
// All but the last N of the wave's own loads into LDS have arrived, and every
// wave is here.
template <int N> __device__ __forceinline__ void many_arrive() {
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

// One row's keys k0 .. k1 - 1 by one wave, from the pages, in fp32: 64 keys at a
// time, first a key to a lane for the scores, then D / 64 of V's bytes to a lane.
// mem: D + 64 floats of the wave's own.  at: the row's part where the keys are split.
template <int D>
__device__ __noinline__ void many_slowly(KvPages p, const int *table, int pages, KvRows q, KvRows out, int r, int kh, int head,
                                         float scale2, int k0, int k1, float *mem, KvParts w, long long at) {
    constexpr int B = D >= 64 ? D / 64 : 1, G = D / 32;
    const int lane = threadIdx.x & 63, b0 = lane * B < D ? lane * B : 0;
    const uint32_t rows = 1u << p.shift;
    const long long head0 = (long long)kh * rows * D, v0 = (long long)p.hk * rows * D, scales = 2 * v0;
    auto dim_of = [](int byte) { return byte % (D / 16) * 16 + byte / (D / 16); };       // of V
    float *const qs = mem, *const ps = mem + D;
    const __bf16 *src = (const __bf16 *)q.p + r * q.row + head * q.head;
    auto lanes = []() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    lanes();
    for (int d = lane; d < D; d += 64) qs[d] = (float)src[d];
    float m = ninf(), l = 0.0f, acc[B] = {};
    for (int key = k0; key < k1; key += 64) {
        const int k = key + lane, page = k >> p.shift;
        const int id = k < k1 && page < pages ? table[page] : -1;
        const bool in = (unsigned)id < (unsigned)p.n_pages;
        const unsigned char *base = p.data + (in ? id : 0) * p.page_bytes;
        const uint32_t off = (uint32_t)k & (rows - 1);
        lanes();
        float x = 0.0f;
        for (int g = 0; g < G; g++) {
            float part = 0.0f;
            for (int h = 0; h < 4; h++) {
                const uint2 u = *(const uint2 *)(base + head0 + (long long)off * D + h * (D / 4) + g * 8);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    part = __builtin_fmaf((float)(int)(((i < 4 ? u.x : u.y) >> (8 * (i & 3))) & 255u) - 128.0f, qs[g * 32 + h * 8 + i], part);
            }
            x = __builtin_fmaf(part, *(const float *)(base + scales + (((long long)kh * G + g) * rows + off) * 4), x);
        }
        x = in ? x * scale2 : ninf();
        float mx = x;
        for (int i = 1; i < 64; i <<= 1) mx = fmaxf(mx, __shfl_xor(mx, i));
        mx = fmaxf(mx, m);
        const float f = m == ninf() ? 0.0f : kv_exp2(m - mx), pr = in ? kv_exp2(x - (mx == ninf() ? 0.0f : mx)) : 0.0f;
        float sum = pr;
        for (int i = 1; i < 64; i <<= 1) sum += __shfl_xor(sum, i);
        l = l * f + sum;
        m = mx;
        ps[lane] = pr;
        lanes();
#pragma unroll
        for (int i = 0; i < B; i++) acc[i] *= f;
        for (int i = 0; i < 64; i++) {
            const int vid = __shfl(id, i);
            if ((unsigned)vid >= (unsigned)p.n_pages) continue;
            const unsigned char *vb = p.data + vid * p.page_bytes;
            const long long vo = (uint32_t)(key + i) & (rows - 1);
            const float pi = ps[i];
#pragma unroll
            for (int e = 0; e < B; e++) {
                const float c = (float)(int)vb[v0 + head0 + vo * D + b0 + e] - 128.0f;
                const float sc = *(const float *)(vb + scales + (((long long)(p.hk + kh) * G + dim_of(b0 + e) / 32) * rows + vo) * 4);
                acc[e] = __builtin_fmaf(pi, c * sc, acc[e]);
            }
        }
    }
    if (w.splits > 1 && lane == 0) *(float2 *)(w.ml + 2 * at) = make_float2(l == l ? m : fmaxf(m, -3.0e38f), l);
    if (lane * B >= D) return;
#pragma unroll
    for (int e = 0; e < B; e++) {
        const int d = dim_of(b0 + e);
        if (w.splits > 1) w.o[at * D + d] = acc[e];
        else ((__bf16 *)out.p)[r * out.row + head * out.head + d] = (__bf16)(l == 0.0f ? 0.0f : acc[e] / l);
    }
}

template <int D, bool Q8, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 && NW == 4 ? 1 : 2) void k_kv_many(KvPages p, KvSeqs b, KvRows q, KvRows out,
                                                                                  int heads, int group, float scale2,
                                                                                  int chunk, int tiles, int vec, int per_seq,
                                                                                  unsigned char *ws, const ManyHead *hd,
                                                                                  KvParts w) {
    using E = typename std::conditional<Q8, _Float16, __bf16>::type;
    using V8 = typename std::conditional<Q8, f16x8, bf16x8>::type;
    constexpr int ROWS = NW * 32, KK = D / 16, DT = D / 32;
    constexpr int TILE = MANY_KEYS * D;                      // numbers of K, of V
    __shared__ __align__(16) uint16_t lk[3 * TILE], lv[4 * TILE];      // of tile % 3, % 4
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    // the sequences of a tile and head next to each other, the tiles with the most keys first
    const int split = blockIdx.x % w.splits, y = blockIdx.x / w.splits, seq = y % b.n_seq, z = y / b.n_seq;
    const int kh = z % p.hk, tile = tiles - 1 - z / p.hk;
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
    int k1 = k0 + chunk;
    const int end = end_of(tile * ROWS + ROWS - 1), all = end_of(tile * ROWS);
    k1 = k1 < end ? k1 : end;

    // The first tiles' loads go ahead of everything else.
    const int n_tiles = (k1 - k0 + MANY_KEYS - 1) / MANY_KEYS, t0 = k0 / MANY_KEYS;
    constexpr int LOADS = TILE * 2 / 1024, PER = 2 * LOADS / NW;         // of 1 KB, of K; a wave's
    const unsigned char *src = tile_at<D>(ws, p.hk, seq, kh, per_seq, t0) + wave * PER * 1024;
    auto load = [&](int i) {                             // tile i (the last one again behind the end)
        const unsigned char *a = src + (long long)(i < n_tiles ? i : n_tiles - 1) * (4 * TILE) + lane * 16;
        char *k = (char *)(lk + i % 3 * TILE), *v = (char *)(lv + (i & 3) * TILE);
#pragma unroll
        for (int e = 0; e < PER; e++) {
            const int x = wave * PER + e;
            __builtin_amdgcn_global_load_lds((many_gptr)(a + e * 1024),
                                             (many_lptr)(x < LOADS ? k + x * 1024 : v + (x - LOADS) * 1024), 16, 0, 0);
        }
    };
    if (k0 < k1) {
        load(0);
        load(1);
    }

    const int row = tile * ROWS + wave * 32 + n, j = row / group, head = kh * group + row % group, r = s.r0 + j;
    const bool on = j < nr && (unsigned)r < (unsigned)b.n_rows;
    const int lim = on ? end_of(row) : 0;
    // a negative scale turns q around, so that the factor of the scores is not negative
    float cq = fabsf(scale2);
    V8 qf[KK];
    {
        // (a row that is not reads another's: a guard around each load would make them wait for each other)
        const __bf16 *src = (const __bf16 *)q.p + (on ? r * q.row + head * q.head : 0);
        float x[KK][8];
        uint32_t big = 0;
#pragma unroll
        for (int c = 0; c < KK; c++) {
            const int at = 2 * c + h;                        // chunk of 8 in the order of K's rows
            const int d0 = Q8 ? (at % (D / 32)) * 32 + at / (D / 32) * 8 : at * 8;
            bf16x8 t;
            if (vec) {
                t = *(const bf16x8 *)(src + d0);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) t[i] = src[d0 + i];
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
            cq = __builtin_amdgcn_ldexpf(cq, e - 8);         // K comes with 2^(8 - ek)
        }
#pragma unroll
        for (int c = 0; c < KK; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) qf[c][i] = (E)(Q8 ? __builtin_amdgcn_ldexpf(x[c][i], -e) : x[c][i]);
    }
    f32x16 o[DT] = {}, st[2];
    u32x4 pw[2][2] = {};                                     // weights of the tile before
    float m = ninf(), l = 0.0f;
    int ev = -1000, ev_least = 1000, ev_most = -1000;        // the unit's exponent of the sums; of all tiles
    bool wide = false, huge = false;

    if (k0 < k1) {
        // Two halves of the block's waves, one of each on every SIMD, take turns:
        // while one has the matrix cores (the values of tile i - 1, the scores of
        // tile i), the other does tile i's softmax, a barrier between the turns.
        // With slots of time counted from 0, half g has the matrix cores for tile
        // i in slot 2 i + g, reads K of tile i and V of tile i - 1 there, and
        // starts its share of tile i + 2's loads, which has arrived by the end of
        // its next turn, slot 2 i + 2 + g.  So tile j's loads run in slots 2 j - 4 to
        // 2 j - 1, K's readers are in slots 2 j and 2 j + 1, V's in 2 j + 2 and
        // 2 j + 3: three buffers for K and four for V.
        // (Four waves, of small calls, have a SIMD each: they are all half 0.)
        const int g = NW == 8 ? wave / 4 : 0;
        // (constant memory to this launch: scalar loads, a tile ahead)
        typedef const __attribute__((address_space(4))) ManyHead *head_ptr;
        const head_ptr hds = (head_ptr)(uintptr_t)(hd + (((long long)seq * p.hk + kh) * per_seq + t0));
        auto head_of = [&](int i) {
            const head_ptr a = hds + (i < n_tiles ? i : n_tiles - 1);
            ManyHead x;
            x.ek = a->ek;
            x.ev = a->ev;
            x.bad[0] = a->bad[0];
            x.bad[1] = a->bad[1];
            x.hole = a->hole;
            x.wide = a->wide;
            return x;
        };
        ManyHead head = head_of(0);
        // the first turn's values are of a tile that is not: no weights, and numbers to take them times
        for (int x = threadIdx.x; x < TILE / 8; x += NW * 64) ((u32x4 *)(lv + 3 * TILE))[x] = u32x4{0, 0, 0, 0};
        __syncthreads();
        many_arrive<0>();
        if (g) many_arrive<0>();
        // The fragments of a turn: 4 DT of V for the values of tile i - 1, then 2 KK
        // of K for the scores of tile i, read in fours one four ahead of the
        // instructions that take them.  The scheduling barriers keep it so: left
        // to itself the compiler reads each where it is used, and waits for it.
        constexpr int NV = 4 * DT, NF = NV + 2 * KK;
        // byte addresses of the lane's row and first chunk; a fragment's own chunk
        // is an exclusive or away (chunk_at), its row a multiple of 32
        const uint32_t lane_v = chunk_at<8>(n, h) * 16, lane_k = chunk_at<D / 8>(n, h) * 16;
        uint32_t row_v = 0, row_k = 0;
        auto fragment = [&](int x) {
            if (x < NV) return *(const u32x4 *)((const char *)lv + (row_v ^ (uint32_t)(x / DT << 5)) + x % DT * (32 * 128));
            x -= NV;
            return *(const u32x4 *)((const char *)lk + (row_k ^ (uint32_t)(x / 2 << 5)) + x % 2 * (32 * 2 * D));
        };
        auto product = [&](int x, const u32x4 &f) {
            if (x < NV) {
                o[x % DT] = mfma32(as<V8>(f), as<V8>(pw[x / DT / 2][x / DT % 2]), o[x % DT]);
            } else {
                x -= NV;
                st[x % 2] = mfma32(as<V8>(f), qf[x / 2], st[x % 2]);
            }
        };
        // The first four, of V, are read before the turn's barrier (their tile is
        // there for two turns already); `beside` is done while the matrix cores
        // have them.
        u32x4 f0[4] = {};
        auto first_four = [&](int i) {                       // of turn i
            row_v = lane_v + ((i + 3) & 3) * (2 * TILE);
#pragma unroll
            for (int e = 0; e < 4; e++) f0[e] = fragment(e);
        };
        auto turn = [&](auto first, auto behind, int i, auto beside) {
            constexpr int A = decltype(first)::value, B = decltype(behind)::value;
            u32x4 f[2][4];
            row_k = lane_k + i % 3 * (2 * TILE);
            if (B == NF) {
                st[0] = f32x16{};
                st[1] = f32x16{};
            }
#pragma unroll
            for (int e = 0; e < 4; e++) f[0][e] = f0[e];
#pragma unroll
            for (int x = A; x < B; x += 4) {
                if (x + 4 < B)
#pragma unroll
                    for (int e = 0; e < 4; e++) f[(x - A) / 4 + 1 & 1][e] = fragment(x + 4 + e);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int e = 0; e < 4; e++) product(x + e, f[(x - A) / 4 & 1][e]);
                if (x == A) beside();
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        typedef std::integral_constant<int, 0> c0;
        typedef std::integral_constant<int, NV> cv;
        typedef std::integral_constant<int, NF> cf;
        first_four(0);
        for (int i = 0; i < n_tiles; i++) {
            const int key = k0 + i * MANY_KEYS;
            turn(c0(), cf(), i, [&]() { load(i + 2); });
            many_arrive<PER>();
            {
                const ManyHead hi = head;
                head = head_of(i + 1);
                const bool masked = key + MANY_KEYS > all || hi.hole || hi.bad[0] || hi.bad[1];
                if (Q8 && hi.ev != MANY_NONE) {
                    if (hi.ev > ev || hi.ev < ev - 4) {      // the sums' unit changes
                        const float f = __builtin_amdgcn_ldexpf(1.0f, ev - hi.ev);
#pragma unroll
                        for (int d = 0; d < DT; d++) o[d] *= f;
                        ev = hi.ev;
                    }
                    ev_least = hi.ev < ev_least ? hi.ev : ev_least;
                    ev_most = hi.ev > ev_most ? hi.ev : ev_most;
                }
                if (Q8) wide = wide || ((hi.wide & 2) && masked);
                float c = Q8 ? __builtin_amdgcn_ldexpf(cq, hi.ek) : cq;
                c = fmaxf(c, 1e-37f);                        // -inf * c stays -inf at a scale of zero
                // (a step of K's numbers, times D of q's, is below c / 8)
                if (Q8 && (hi.wide & 1)) wide = wide || __any(c > 0x1p-8f);
                float mx = ninf();
                if (masked) {
                    // (the lane's half taken out first, so that what is compared with is constant:
                    // it would be kept in 64 registers through the whole loop)
                    const uint32_t bad0 = hi.bad[0] >> (h * 4), bad1 = hi.bad[1] >> (h * 4);
                    const int left = lim - key - h * 4;
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int k = (e >> 2) * 8 + (e & 3);
                            const bool in = t * 32 + k < left && !(hi.hole >> (2 * t + (e >> 3)) & 1);
                            if (in && ((t ? bad1 : bad0) >> k & 1)) l = __builtin_nanf("");
                            st[t][e] = in ? st[t][e] : ninf();
                        }
                }
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) mx = fmaxf(mx, st[t][e]);
                mx = fmaxf(mx, __shfl_xor(mx, 32)) * c;
                // each row by itself: its bits must not depend on the wave's other rows
                const bool up = mx > m + 8.0f;
                if (__any(up)) {
                    const float mn = up ? mx : m, f = up ? kv_exp2(m - mn) : 1.0f;
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[d] *= f;
                    m = mn;
                    huge = __any(fabsf(m) > 0x1p20f && m != ninf());
                }
                // weights in the sums' unit: V's tile has its own
                const float less = Q8 && hi.ev != MANY_NONE ? (float)(ev - hi.ev) : 0.0f;
                float mu = (m == ninf() ? 0.0f : m) + less;
                // Of scores so large that the maximum's rounding is no small
                // difference the products are rounded like it.
                if (huge) {
                    const bool mine = fabsf(m) > 0x1p20f && m != ninf();
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int e = 0; e < 16; e++) st[t][e] = mine ? st[t][e] * c - m : st[t][e];
                    c = mine ? 1.0f : c;
                    mu = mine ? less : mu;
                }
                float sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float a = kv_exp2(__builtin_fmaf(st[t][u * 8 + 2 * e], c, -mu));
                            const float d = kv_exp2(__builtin_fmaf(st[t][u * 8 + 2 * e + 1], c, -mu));
                            pw[t][u][e] = pack2<E>(a, d);
                            sum = add2<E>(pw[t][u][e], sum);
                        }
                l = Q8 ? __builtin_fmaf(sum, kv_exp2(less), l) : l + sum;
            }
            first_four(i + 1);
            asm volatile("s_barrier" ::: "memory");
        }
        if (!g) asm volatile("s_barrier" ::: "memory");
        turn(c0(), cv(), n_tiles, []() {});
        if (Q8 && __syncthreads_or(wide || ev_most - ev_least > 60)) {
            for (int i = 0; i < 32; i++) {
                const int row = tile * ROWS + wave * 32 + i, j = row / group, r = s.r0 + j;
                if (j >= nr || (unsigned)r >= (unsigned)b.n_rows) continue;
                const int most = end_of(row);
                many_slowly<D>(p, b.table + seq * b.stride, b.pages, q, out, r, kh, kh * group + row % group, scale2, k0,
                               most < k1 ? most : k1, (float *)lk + wave * (D + 64), w,
                               ((long long)r * heads + kh * group + row % group) * w.splits + split);
            }
            return;
        }
    }
    l += __shfl_xor(l, 32);
    if (Q8) {
        const float f = __builtin_amdgcn_ldexpf(1.0f, ev == -1000 ? 0 : ev - 8);
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= f;
    }
    if (w.splits == 1) {
        // Through LDS, so that a wave's stores are of whole rows (as the lanes have
        // them, 8 bytes of each of 32 rows: nine packed prompts 419 us, so 411).
        constexpr int CH = D / 8;                            // 16-byte chunks of a row
        __syncthreads();                                     // the other waves' last turn
        uint16_t *const mine = lv + wave * (32 * D);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int c = d * 4 + (i >> 2);
                uint2 t;
                t.x = pack2<__bf16>(o[d][i] * inv, o[d][i + 1] * inv);
                t.y = pack2<__bf16>(o[d][i + 2] * inv, o[d][i + 3] * inv);
                *(uint2 *)(mine + n * D + (c ^ (n & (CH - 1))) * 8 + h * 4) = t;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const long long at = on ? r * out.row + head * out.head : -1;
#pragma unroll
        for (int i = 0; i < CH / 2; i++) {
            const int x = i * 64 + lane, m = x / CH, c = x % CH;
            const u32x4 t = *(const u32x4 *)(mine + m * D + (c ^ (m & (CH - 1))) * 8);
            const long long to = __shfl(at, m);
            if (to < 0) continue;
            uint16_t *dst = (uint16_t *)out.p + to + c * 8;
            if (vec) {
                *(u32x4 *)dst = t;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) dst[e] = (uint16_t)(t[e / 2] >> (16 * (e & 1)));
            }
        }
        return;
    }
    if (!on) return;
    const long long at = ((long long)r * heads + head) * w.splits + split;
    if (h == 0) {
        w.ml[2 * at] = l == l ? m : fmaxf(m, -3.0e38f);     // (scores that are all NaN leave m, and are not no keys)
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

// The tiles of one sequence, and how many sequences' tiles are made at a time:
// as many as take 1 GiB (the workspace grows no further with the batch).
static long long seq_tiles(const KvPages &p, const KvSeqs &b) {
    const long long cap = (long long)b.pages << p.shift, most = b.max_len < cap ? b.max_len : cap;
    return (most + MANY_KEYS - 1) / MANY_KEYS;
}
static int seqs_at_once(const KvPages &p, const KvSeqs &b) {
    const long long one = seq_tiles(p, b) * p.hk * (4 * MANY_KEYS * p.d), k = one ? (1LL << 30) / one : b.n_seq;
    return (int)(k < 1 ? 1 : k < b.n_seq ? k : b.n_seq);
}
extern "C" long long l98k_kv_many_ws(const KvPages &p, const KvSeqs &b) {
    return seqs_at_once(p, b) * seq_tiles(p, b) * p.hk * (4LL * MANY_KEYS * p.d + (long long)sizeof(ManyHead));
}

template <int D, bool Q8>
static int many(const KvPages &p, const KvSeqs &all, const KvRows &q, const KvRows &o, int heads, float scale2,
                const KvPlan &x, const KvParts &w, unsigned char *ws, hipStream_t st) {
    const int vec = aligned16(q) && aligned16(o), step = seqs_at_once(p, all);
    const long long n = seq_tiles(p, all), blocks = (long long)x.splits * p.hk * x.tiles * step;
    if (n * p.hk > INT_MAX || blocks > INT_MAX) return -1;
    ManyHead *hd = (ManyHead *)(ws + step * n * p.hk * (4LL * MANY_KEYS * D));
    for (int i = 0; i < all.n_seq; i += step) {
        KvSeqs b = all;
        b.table += i * b.stride;
        b.kv_len += i;
        b.row0 += i;
        b.n_seq = all.n_seq - i < step ? all.n_seq - i : step;
        if (n) {
            hipLaunchKernelGGL((k_kv_tiles<D, Q8>), dim3((unsigned)(n * p.hk), b.n_seq), dim3(TILE_THREADS), 0, st, p, b,
                               (int)n, ws, hd);
            const int rc = (int)hipGetLastError();
            if (rc) return rc;
        }
        const dim3 grid((unsigned)((long long)x.splits * p.hk * x.tiles * b.n_seq));
        if (x.rows == 128)
            hipLaunchKernelGGL((k_kv_many<D, Q8, 4>), grid, dim3(256), 0, st, p, b, q, o, heads, heads / p.hk, scale2,
                               x.chunk, x.tiles, vec, (int)n, ws, hd, w);
        else
            hipLaunchKernelGGL((k_kv_many<D, Q8, 8>), grid, dim3(512), 0, st, p, b, q, o, heads, heads / p.hk, scale2,
                               x.chunk, x.tiles, vec, (int)n, ws, hd, w);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    return 0;
}

extern "C" int l98k_kv_many(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads,
                            float scale2, const KvPlan &x, const KvParts &w, void *ws, hipStream_t st) {
#define MANY_D(DD)                                                                                         \
    if (p.d == DD)                                                                                         \
        return q8 ? many<DD, true>(p, b, q, o, heads, scale2, x, w, (unsigned char *)ws, st)               \
                  : many<DD, false>(p, b, q, o, heads, scale2, x, w, (unsigned char *)ws, st)
    MANY_D(32);
    MANY_D(64);
    MANY_D(128);
    return -1;
}
