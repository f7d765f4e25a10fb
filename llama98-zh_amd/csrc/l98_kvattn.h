// What the two attention kernels over the paged cache share.
#ifndef L98_KVATTN_H
#define L98_KVATTN_H
#include "l98_kv.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float kv_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float ninf() { return -__builtin_inff(); }

// bytes `b0` of lo and `b1` of hi, each minus 128, times 2^-9, as two fp16
__device__ __forceinline__ uint32_t codes2(uint32_t hi, uint32_t lo, uint32_t sel) {
    const uint32_t u = __builtin_amdgcn_perm(hi, lo, sel);
    f16x2 x;
    __builtin_memcpy(&x, &u, 4);
    const f16x2 a = {(_Float16)32768.0f, (_Float16)32768.0f}, c = {(_Float16)-0.25f, (_Float16)-0.25f};
    x = __builtin_elementwise_fma(x, a, c);
    uint32_t r;
    __builtin_memcpy(&r, &x, 4);
    return r;
}
template <class V> __device__ __forceinline__ V as(u32x4 x) {
    V v;
    __builtin_memcpy(&v, &x, 16);
    return v;
}
template <class E> struct Pair;
template <> struct Pair<_Float16> { typedef f16x2 type; };
template <> struct Pair<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(2))); };
// two floats rounded to E, half to even, as one instruction
template <class E> __device__ __forceinline__ typename Pair<E>::type round2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_convertvector((f32x2){a, b}, typename Pair<E>::type);
}
template <class E> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    const typename Pair<E>::type x = round2<E>(a, b);
    uint32_t r;
    __builtin_memcpy(&r, &x, 4);
    return r;
}
// N words whose halves' sums are a and b to N times E's bits
template <class E, int N> __device__ __forceinline__ void parts2(float a, float b, uint32_t *o) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        const typename Pair<E>::type x = round2<E>(a, b);
        __builtin_memcpy(&o[i], &x, 4);
        if (i + 1 < N) {
            a -= (float)x[0];
            b -= (float)x[1];
        }
    }
}

// Partial results in the workspace: of (row, head, split) D floats, then the
// pairs (M, sum): the sums are in units of 2^M.
struct KvParts {
    float *o, *ml;
    int splits;
};

struct KvPlan {
    bool many;
    int rows, tiles, chunk, splits;
};

extern "C" int l98k_kv_many(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads,
                            float scale2, const KvPlan &x, const KvParts &w, void *ws, hipStream_t st);
// bytes of its workspace, a multiple of 16
extern "C" long long l98k_kv_many_ws(const KvPages &p, const KvSeqs &b);
#endif
