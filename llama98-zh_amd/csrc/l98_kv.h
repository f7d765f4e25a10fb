// The paged key-value cache: what its kernels (l98_k_kv.hip, l98_k_kvattn.hip)
// take, and their launchers.  The layout and the batch's meaning are those of
// include/llama98_hip.h; every launcher's arguments were checked by l98_kv.cpp.
#ifndef L98_KV_H
#define L98_KV_H
#include <hip/hip_runtime.h>
#include <stdint.h>

// A layer of a pool.  Page p's block of this layer starts at
// data + p * page_bytes; inside it lie K, V, and for Q8 the K scales and the
// V scales, each [n_kv_heads][page_rows][head_dim] numbers or
// [n_kv_heads][head_dim / 32][page_rows] scales.
struct KvPages {
    unsigned char *data;          // the pool + the layer's offset
    long long page_bytes;
    int n_pages, shift, hk, d;    // page_rows = 1 << shift
};

struct KvSeqs {
    const int *table, *kv_len, *row0;
    long long stride;             // table entries from one sequence to the next
    int pages, n_seq, n_rows, max_rows, max_len;   // pages: table entries of a sequence
};

// Rows [n][heads][d] at strides in elements.
struct KvRows {
    void *p;
    long long row, head;
};

// page pairs of one launch, in its arguments
template <int N>
struct KvMoves {
    int src[N], dst[N];
};

// One sequence of a batch as a kernel sees it: its first row, its number of
// new rows, the position of the first of them, and the keys that exist (the
// length within the table's and the caller's bounds).
struct KvSeq {
    int r0, n, pos0, len;
};
__device__ __forceinline__ KvSeq kv_seq(const KvSeqs &b, int i, int shift) {
    KvSeq s;
    s.r0 = b.row0[i];
    s.n = b.row0[i + 1] - s.r0;
    const int len = b.kv_len[i];
    s.pos0 = len - s.n;
    // the table's end, in 64 bits: 2^27 pages of 16 rows pass an int
    const long long cap = (long long)b.pages << shift;
    const int most = b.max_len < cap ? b.max_len : (int)cap;
    s.len = len < most ? len : most;
    return s;
}
__device__ __forceinline__ const unsigned char *kv_page(const KvPages &p, int id) {
    return p.data + (long long)id * p.page_bytes;
}

extern "C" {
int l98k_kv_append(const KvPages &p, int q8, const KvSeqs &b, const KvRows &k, const KvRows &v, int bf16,
                   hipStream_t st);
int l98k_kv_read(const KvPages &p, int q8, const KvSeqs &b, const KvRows &k, const KvRows &v, int bf16, hipStream_t st);
int l98k_kv_copy(unsigned char *data, long long page_bytes, const int *src, const int *dst, int n, hipStream_t st);
// Device scratch of l98k_kv_attend (0: none) for these shapes.
long long l98k_kv_attend_ws(const KvPages &p, int q8, const KvSeqs &b, int heads, int bf16);
int l98k_kv_attend(const KvPages &p, int q8, const KvSeqs &b, const KvRows &q, const KvRows &out, int heads, int bf16,
                   float scale, void *ws, hipStream_t st);
}
#endif
