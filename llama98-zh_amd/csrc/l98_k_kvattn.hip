// Causal attention over the paged key-value cache.
#include "l98_devmath.h"
#include "l98_kv.h"

// One wave per (row, query head): a lane holds D / 64 dimensions (of the first
// D lanes for D < 64), keys in turn, the running maximum and sum of the softmax.
template <class T, int D, bool Q8>
__global__ __launch_bounds__(64) void k_kv_attend_rows(KvPages p, KvSeqs b, KvRows q, KvRows o, int group, float scale) {
    constexpr int E = D > 64 ? D / 64 : 1;
    const int i = blockIdx.z, j = blockIdx.x, head = blockIdx.y, kh = head / group, lane = threadIdx.x;
    const KvSeq s = kv_seq(b, i, p.shift);
    const int r = s.r0 + j;
    if (j >= s.n || (unsigned)r >= (unsigned)b.n_rows) return;
    const bool on = lane < D;
    float qv[E], acc[E], m = -__builtin_inff(), l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        acc[e] = 0.0f;
        qv[e] = on ? (float)((const T *)q.p + r * q.row + head * q.head)[lane + 64 * e] * scale : 0.0f;
    }
    const int pos = s.pos0 + j, end = pos + 1 < s.len ? pos + 1 : s.len;
    for (int key = 0; key < end; key++) {
        const int id = b.table[i * b.stride + (key >> p.shift)];
        if ((unsigned)id >= (unsigned)p.n_pages) continue;
        const unsigned char *pg = kv_page(p, id);
        const int off = key & ((1 << p.shift) - 1);
        float kx[E], vx[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = on ? lane + 64 * e : 0;
            const long long row = ((long long)kh << p.shift) + off, vrow = ((long long)(p.hk + kh) << p.shift) + off;
            if (Q8) {
                const long long sc = ((long long)2 * p.hk << p.shift) * D;
                const float ks = *(const float *)(pg + sc + ((((long long)kh * (D / 32) + d / 32) << p.shift) + off) * 4);
                const float vs =
                    *(const float *)(pg + sc + ((((long long)(p.hk + kh) * (D / 32) + d / 32) << p.shift) + off) * 4);
                kx[e] = ((float)pg[row * D + ((d & 31) >> 3) * (D / 4) + (d >> 5) * 8 + (d & 7)] - 128.0f) * ks;
                vx[e] = ((float)pg[vrow * D + (d & 15) * (D / 16) + (d >> 4)] - 128.0f) * vs;
            } else {
                kx[e] = (float)((const __bf16 *)pg)[row * D + d];
                vx[e] = (float)((const __bf16 *)pg)[vrow * D + d];
            }
        }
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) dot = on ? __builtin_fmaf(qv[e], kx[e], dot) : 0.0f;
        for (int x = 32; x > 0; x >>= 1) dot += __shfl_xor(dot, x);
        const float mn = dot > m ? dot : m;
        const float a = m == mn ? 1.0f : expf(m - mn), w = expf(dot - mn);
        m = mn;
        l = l * a + w;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = __builtin_fmaf(w, vx[e], acc[e] * a);
    }
    if (on)
#pragma unroll
        for (int e = 0; e < E; e++)
            ((T *)o.p + r * o.row + head * o.head)[lane + 64 * e] = (T)(l == 0.0f ? 0.0f : acc[e] / l);
}

extern "C" long long l98k_kv_attend_ws(const KvPages &, int, const KvSeqs &, int, int) { return 0; }

template <class T, int D>
static void launch(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads, float scale,
                   hipStream_t st) {
    const dim3 grid(b.max_rows, heads, b.n_seq);
    if (q8) hipLaunchKernelGGL((k_kv_attend_rows<T, D, true>), grid, dim3(64), 0, st, p, b, q, o, heads / p.hk, scale);
    else hipLaunchKernelGGL((k_kv_attend_rows<T, D, false>), grid, dim3(64), 0, st, p, b, q, o, heads / p.hk, scale);
}

extern "C" int l98k_kv_attend(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &o, int heads,
                              int bf16, float scale, void *, hipStream_t st) {
    if (p.d == 32) bf16 ? launch<__bf16, 32>(p, q8, b, q, o, heads, scale, st) : launch<float, 32>(p, q8, b, q, o, heads, scale, st);
    else if (p.d == 64) bf16 ? launch<__bf16, 64>(p, q8, b, q, o, heads, scale, st) : launch<float, 64>(p, q8, b, q, o, heads, scale, st);
    else if (p.d == 128) bf16 ? launch<__bf16, 128>(p, q8, b, q, o, heads, scale, st) : launch<float, 128>(p, q8, b, q, o, heads, scale, st);
    else return -1;
    return (int)hipGetLastError();
}
