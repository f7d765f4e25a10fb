// The paged key-value cache behind the C ABI: argument checks, launches, and
// the pages' book-keeping (include/llama98_hip.h).
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <functional>
#include <limits.h>
#include <math.h>
#include <queue>
#include <vector>

#include "../../include/llama98_hip.h"
#include "l98_kv.h"

namespace {

int fail(char *errbuf, int errlen, int code, const char *fmt, ...) {
    if (errbuf && errlen > 0) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(errbuf, (size_t)errlen, fmt, ap);
        va_end(ap);
    }
    return -code;
}
#define BAD(...) return fail(errbuf, errlen, LZ_ERR_NULL_ARG, __VA_ARGS__)

bool pool_in_limits(const L98KvPool *p) {
    return p && (p->format == L98_KV_Q8 || p->format == L98_KV_BF16) && p->n_layers >= 1 && p->n_layers <= 1024 &&
           p->n_pages >= 1 && p->page_rows >= 16 && p->page_rows <= 1024 && !(p->page_rows & (p->page_rows - 1)) &&
           p->n_kv_heads >= 1 && p->n_kv_heads <= 1024 &&
           (p->head_dim == 32 || p->head_dim == 64 || p->head_dim == 128);
}
long long layer_bytes(const L98KvPool *p);
// the kernels count a page in 16-byte units of 32 bits
bool pool_ok(const L98KvPool *p) { return pool_in_limits(p) && layer_bytes(p) * p->n_layers < (1LL << 36); }
long long layer_bytes(const L98KvPool *p) {
    const long long n = (long long)p->n_kv_heads * p->page_rows * p->head_dim;
    return p->format == L98_KV_Q8 ? 2 * (n + n / 32 * 4) : 4 * n;
}

// Null, or why the kernels cannot use the pointer on the current device.
const char *dev_ptr(const void *p, int dev, int align) {
    if (!p) return "is null";
    if ((uintptr_t)p % (uintptr_t)align) return "is not aligned to its elements";
    hipPointerAttribute_t a;
    if (hipPointerGetAttributes(&a, p) != hipSuccess) {
        (void)hipGetLastError();
        return "is not device memory";
    }
    if (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged) return "is not device memory";
    if (a.device != dev) return "is on another device than the current one";
    return nullptr;
}
#define DEV_PTR(ptr, align, name)                                                 \
    do {                                                                          \
        if (const char *why = dev_ptr(ptr, dev, align)) BAD("%s %s", name, why);  \
    } while (0)

// What a call's arguments say, checked without a device (the order of the
// checks: everything that needs none first).
int host_pool(const L98KvPool *p, int layer, KvPages *out, char *errbuf, int errlen) {
    if (!pool_ok(p)) BAD("the pool is null or outside the limits");
    if (layer < 0 || layer >= p->n_layers) BAD("layer %d of %d", layer, p->n_layers);
    out->data = (unsigned char *)p->data + layer * layer_bytes(p);
    out->page_bytes = layer_bytes(p) * p->n_layers;
    out->n_pages = p->n_pages;
    out->shift = __builtin_ctz((unsigned)p->page_rows);
    out->hk = p->n_kv_heads;
    out->d = p->head_dim;
    return 0;
}
int host_batch(const L98KvPool *p, const L98KvBatch *b, KvSeqs *s, char *errbuf, int errlen) {
    if (!b || b->n_seq < 0 || b->n_seq > 65535 || b->n_rows < 0 || b->max_rows < 0 || b->max_len < 0 ||
        b->table_pages < 0 || b->table_stride < 0)
        BAD("the batch is null or outside the limits");
    s->table = b->table;
    s->kv_len = b->kv_len;
    s->row0 = b->row0;
    s->stride = b->table_stride;
    s->pages = b->table_pages;
    s->n_seq = b->n_seq;
    s->n_rows = b->n_rows;
    s->max_rows = std::min(b->max_rows, b->n_rows);
    // what a table can hold is a bound too; the kernels count keys, a chunk ahead, in 31 bits
    s->max_len = (int)std::min<long long>(b->max_len, (long long)b->table_pages * p->page_rows);
    if (s->max_len > 1 << 30) BAD("sequences of %d positions", s->max_len);
    return 0;
}
bool no_rows(const KvSeqs &s) { return s.n_seq == 0 || s.max_rows == 0; }
// written: two places or heads that fall together would be written by several lanes
int host_rows(const L98KvRows *r, int dtype, int n_rows, int heads, int dim, bool written, const char *name, KvRows *out,
              char *errbuf, int errlen) {
    if (!r) BAD("%s is null", name);
    if (dtype != L98_F32 && dtype != L98_BF16) BAD("dtype %d", dtype);
    if (r->row_stride < 0 || r->head_stride < 0) BAD("%s has a negative stride", name);
    // one row's heads before the next, or one head's rows
    const __int128 row = r->row_stride, head = r->head_stride;
    if (written && !(n_rows <= 1 && (heads == 1 || head >= dim)) &&
        !(row >= (heads - 1) * head + dim && (heads == 1 || head >= dim)) &&
        !(head >= (n_rows - 1) * row + dim && row >= dim))
        BAD("%s has rows or heads that overlap, or lie in each other", name);
    out->p = r->p;
    out->row = r->row_stride;
    out->head = r->head_stride;
    return 0;
}
int host_heads(const L98KvPool *p, int n_heads, char *errbuf, int errlen) {
    if (n_heads < 1 || n_heads % p->n_kv_heads || n_heads / p->n_kv_heads > 16)
        BAD("n_heads %d is no multiple of n_kv_heads %d, or over 16 times it", n_heads, p->n_kv_heads);
    return 0;
}

int current(hipStream_t st, int *dev, char *errbuf, int errlen) {
    hipDevice_t sd = 0;
    if (hipGetDevice(dev) != hipSuccess) {
        (void)hipGetLastError();
        return fail(errbuf, errlen, LZ_ERR_FORWARD, "no current device");
    }
    if (st && hipStreamGetDevice(st, &sd) != hipSuccess) {
        (void)hipGetLastError();
        BAD("the stream is not one");
    }
    if (st && sd != *dev) BAD("the stream is on another device than the current one");
    return 0;
}
int dev_batch(const L98KvPool *p, const KvSeqs &s, int dev, char *errbuf, int errlen) {
    DEV_PTR(p->data, 16, "the pool's data");
    DEV_PTR(s.kv_len, 4, "kv_len");
    DEV_PTR(s.row0, 4, "row0");
    if (s.pages) DEV_PTR(s.table, 4, "the table");
    return 0;
}
int launched(int rc, char *errbuf, int errlen) {
    if (rc == 0) return 0;
    return fail(errbuf, errlen, LZ_ERR_FORWARD, "%s",
                rc < 0 ? "the kernels do not take these sizes" : hipGetErrorString((hipError_t)rc));
}
#define CHECK(x)                 \
    do {                         \
        const int rc_ = (x);     \
        if (rc_) return rc_;     \
    } while (0)

typedef int (*RowsFn)(const KvPages &, int, const KvSeqs &, const KvRows &, const KvRows &, int, hipStream_t);
int rows_call(RowsFn fn, bool written, const L98KvPool *pool, int layer, const L98KvBatch *b, const L98KvRows *k,
              const L98KvRows *v, int dtype, void *stream, char *errbuf, int errlen) {
    const hipStream_t st = (hipStream_t)stream;
    int dev = 0;
    KvPages p;
    KvSeqs s;
    KvRows rk, rv;
    CHECK(host_pool(pool, layer, &p, errbuf, errlen));
    CHECK(host_batch(pool, b, &s, errbuf, errlen));
    CHECK(host_rows(k, dtype, s.n_rows, p.hk, p.d, written, "k", &rk, errbuf, errlen));
    CHECK(host_rows(v, dtype, s.n_rows, p.hk, p.d, written, "v", &rv, errbuf, errlen));
    if (no_rows(s)) return 0;
    CHECK(current(st, &dev, errbuf, errlen));
    CHECK(dev_batch(pool, s, dev, errbuf, errlen));
    DEV_PTR(rk.p, dtype == L98_F32 ? 4 : 2, "k");
    DEV_PTR(rv.p, dtype == L98_F32 ? 4 : 2, "v");
    return launched(fn(p, pool->format == L98_KV_Q8, s, rk, rv, dtype == L98_BF16, st), errbuf, errlen);
}

}  // namespace

extern "C" long long l98_kv_page_bytes(const L98KvPool *p) {
    return pool_ok(p) ? layer_bytes(p) * p->n_layers : -LZ_ERR_NULL_ARG;
}

extern "C" int l98_kv_append(const L98KvPool *pool, int layer, const L98KvBatch *b, const L98KvRows *k,
                             const L98KvRows *v, int dtype, void *stream, char *errbuf, int errlen) {
    return rows_call(l98k_kv_append, false, pool, layer, b, k, v, dtype, stream, errbuf, errlen);
}

extern "C" int l98_kv_read(const L98KvPool *pool, int layer, const L98KvBatch *b, const L98KvRows *k,
                           const L98KvRows *v, int dtype, void *stream, char *errbuf, int errlen) {
    return rows_call(l98k_kv_read, true, pool, layer, b, k, v, dtype, stream, errbuf, errlen);
}

extern "C" long long l98_kv_attend_ws_bytes(const L98KvPool *pool, const L98KvBatch *b, int n_heads, int dtype) {
    KvPages p = {};
    KvSeqs s;
    if (host_pool(pool, 0, &p, nullptr, 0) || host_batch(pool, b, &s, nullptr, 0) || host_heads(pool, n_heads, nullptr, 0) ||
        (dtype != L98_F32 && dtype != L98_BF16))
        return -LZ_ERR_NULL_ARG;
    return no_rows(s) ? 0 : l98k_kv_attend_ws(p, pool->format == L98_KV_Q8, s, n_heads, dtype == L98_BF16);
}

extern "C" int l98_kv_attend(const L98KvPool *pool, int layer, const L98KvBatch *b, const L98KvRows *q,
                             const L98KvRows *out, int n_heads, int dtype, float scale, void *ws, long long ws_bytes,
                             void *stream, char *errbuf, int errlen) {
    const hipStream_t st = (hipStream_t)stream;
    int dev = 0;
    KvPages p;
    KvSeqs s;
    KvRows rq, ro;
    CHECK(host_pool(pool, layer, &p, errbuf, errlen));
    CHECK(host_batch(pool, b, &s, errbuf, errlen));
    CHECK(host_heads(pool, n_heads, errbuf, errlen));
    CHECK(host_rows(q, dtype, s.n_rows, n_heads, p.d, false, "q", &rq, errbuf, errlen));
    CHECK(host_rows(out, dtype, s.n_rows, n_heads, p.d, true, "out", &ro, errbuf, errlen));
    if (!(fabsf(scale) < 1e38f)) BAD("scale is not finite, or above 1e38");
    if (no_rows(s)) return 0;
    const int q8 = pool->format == L98_KV_Q8, bf16 = dtype == L98_BF16;
    const long long need = l98k_kv_attend_ws(p, q8, s, n_heads, bf16);
    if (ws_bytes < need) BAD("the workspace has %lld bytes, %lld are needed", ws_bytes, need);
    CHECK(current(st, &dev, errbuf, errlen));
    CHECK(dev_batch(pool, s, dev, errbuf, errlen));
    DEV_PTR(rq.p, bf16 ? 2 : 4, "q");
    DEV_PTR(ro.p, bf16 ? 2 : 4, "out");
    if (need) DEV_PTR(ws, 16, "the workspace");
    return launched(l98k_kv_attend(p, q8, s, rq, ro, n_heads, bf16, scale, ws, st), errbuf, errlen);
}

extern "C" int l98_kv_copy_pages(const L98KvPool *pool, const int *src, const int *dst, int n, void *stream,
                                 char *errbuf, int errlen) {
    const hipStream_t st = (hipStream_t)stream;
    int dev = 0;
    KvPages p;
    CHECK(host_pool(pool, 0, &p, errbuf, errlen));
    if (n < 0 || n > pool->n_pages || (n && (!src || !dst))) BAD("%d copies, or a null list", n);
    if (n == 0) return 0;
    try {
        std::vector<int> w(dst, dst + n);
        for (int i = 0; i < n; i++)
            if (src[i] < 0 || src[i] >= pool->n_pages || dst[i] < 0 || dst[i] >= pool->n_pages)
                BAD("copy %d: page %d to %d of %d", i, src[i], dst[i], pool->n_pages);
        std::sort(w.begin(), w.end());
        for (int i = 1; i < n; i++)
            if (w[(size_t)i] == w[(size_t)i - 1]) BAD("page %d is written twice", w[(size_t)i]);
        for (int i = 0; i < n; i++)
            if (std::binary_search(w.begin(), w.end(), src[i])) BAD("page %d is read and written", src[i]);
    } catch (...) {
        return fail(errbuf, errlen, LZ_ERR_STATE_ALLOC, "no host memory");
    }
    CHECK(current(st, &dev, errbuf, errlen));
    DEV_PTR(p.data, 16, "the pool's data");
    return launched(l98k_kv_copy(p.data, p.page_bytes, src, dst, n, st), errbuf, errlen);
}

// ---------------------------------------------------------- book-keeping ---

struct L98KvPages {
    int rows;                                 // of a page
    std::vector<int> refs;                    // of each page
    std::priority_queue<int, std::vector<int>, std::greater<int>> unused;
    struct Seq {
        bool live = false;
        int len = 0;
        std::vector<int> pages;
    };
    std::vector<Seq> seqs;

    Seq *get(int i) { return i >= 0 && (size_t)i < seqs.size() && seqs[(size_t)i].live ? &seqs[(size_t)i] : nullptr; }
    const Seq *get(int i) const { return const_cast<L98KvPages *>(this)->get(i); }
    int pages_of(int n) const { return (int)(((long long)n + rows - 1) / rows); }
    int place() {                             // a dead entry's index, or a new one's
        for (size_t i = 0; i < seqs.size(); i++)
            if (!seqs[i].live) return (int)i;
        seqs.emplace_back();
        return (int)seqs.size() - 1;
    }
    // `unused` holds room for every page from the start, so giving one back allocates nothing
    void drop(int page) {
        if (--refs[(size_t)page] == 0) unused.push(page);
    }
    int take() {
        const int page = unused.top();
        unused.pop();
        refs[(size_t)page] = 1;
        return page;
    }
};

#define GUARD(...)                       \
    try {                                \
        __VA_ARGS__                      \
    } catch (...) {                      \
        return -LZ_ERR_STATE_ALLOC;      \
    }

extern "C" L98KvPages *l98_kv_pages_open(int n_pages, int page_rows) {
    if (n_pages < 1 || page_rows < 16 || page_rows > 1024 || (page_rows & (page_rows - 1))) return nullptr;
    L98KvPages *h = nullptr;
    try {
        h = new L98KvPages;
        h->rows = page_rows;
        h->refs.assign((size_t)n_pages, 0);
        std::vector<int> ids((size_t)n_pages);
        for (int i = 0; i < n_pages; i++) ids[(size_t)i] = i;
        h->unused = std::priority_queue<int, std::vector<int>, std::greater<int>>(std::greater<int>(), std::move(ids));
        return h;
    } catch (...) {
        delete h;
        return nullptr;
    }
}

extern "C" void l98_kv_pages_close(L98KvPages *h) { delete h; }

extern "C" int l98_kv_pages_new(L98KvPages *h) {
    if (!h) return -LZ_ERR_NULL_ARG;
    GUARD({
        const int i = h->place();
        L98KvPages::Seq &s = h->seqs[(size_t)i];
        s.live = true;
        s.len = 0;
        s.pages.clear();
        return i;
    })
}

extern "C" int l98_kv_pages_fork(L98KvPages *h, int seq, int n_rows) {
    if (!h || !h->get(seq) || n_rows < 0 || n_rows > h->get(seq)->len) return -LZ_ERR_NULL_ARG;
    GUARD({
        const int i = h->place();             // may move seqs
        const L98KvPages::Seq &from = h->seqs[(size_t)seq];
        L98KvPages::Seq &to = h->seqs[(size_t)i];
        to.pages.assign(from.pages.begin(), from.pages.begin() + h->pages_of(n_rows));
        to.len = n_rows;
        to.live = true;
        for (int p : to.pages) h->refs[(size_t)p]++;
        return i;
    })
}

extern "C" int l98_kv_pages_extend(L98KvPages *h, int seq, int n, int *src, int *dst) {
    L98KvPages::Seq *s = h ? h->get(seq) : nullptr;
    if (!s || n < 0 || n > INT_MAX - s->len || !src || !dst) return -LZ_ERR_NULL_ARG;
    if (n == 0) return 0;
    const bool copy = s->len % h->rows && h->refs[(size_t)s->pages.back()] > 1;
    const int more = h->pages_of(s->len + n) - (int)s->pages.size();
    if ((size_t)more + (copy ? 1 : 0) > h->unused.size()) return -LZ_ERR_STATE_ALLOC;
    GUARD({
        s->pages.reserve(s->pages.size() + (size_t)more);
        if (copy) {
            *src = s->pages.back();
            *dst = h->take();
            h->drop(*src);
            s->pages.back() = *dst;
        }
        for (int k = 0; k < more; k++) s->pages.push_back(h->take());
        s->len += n;
        return copy ? 1 : 0;
    })
}

extern "C" int l98_kv_pages_trim(L98KvPages *h, int seq, int n_rows) {
    L98KvPages::Seq *s = h ? h->get(seq) : nullptr;
    if (!s || n_rows < 0 || n_rows > s->len) return -LZ_ERR_NULL_ARG;
    GUARD({
        const size_t keep = (size_t)h->pages_of(n_rows);
        while (s->pages.size() > keep) {
            h->drop(s->pages.back());
            s->pages.pop_back();
        }
        s->len = n_rows;
        return 0;
    })
}

extern "C" int l98_kv_pages_free(L98KvPages *h, int seq) {
    const int rc = l98_kv_pages_trim(h, seq, 0);
    if (rc == 0) h->seqs[(size_t)seq].live = false;
    return rc;
}

extern "C" int l98_kv_pages_len(const L98KvPages *h, int seq) {
    const L98KvPages::Seq *s = h ? h->get(seq) : nullptr;
    return s ? s->len : -LZ_ERR_NULL_ARG;
}

extern "C" int l98_kv_pages_table(const L98KvPages *h, int seq, int *out, int cap) {
    const L98KvPages::Seq *s = h ? h->get(seq) : nullptr;
    if (!s || cap < 0 || (cap && !out)) return -LZ_ERR_NULL_ARG;
    const int n = (int)s->pages.size();
    for (int i = 0; i < n && i < cap; i++) out[i] = s->pages[(size_t)i];
    return n;
}

extern "C" int l98_kv_pages_unused(const L98KvPages *h) { return h ? (int)h->unused.size() : -LZ_ERR_NULL_ARG; }

extern "C" int l98_kv_pages_compact(L98KvPages *h, int *src, int *dst, int cap) {
    if (!h || cap < 0 || (cap && (!src || !dst))) return -LZ_ERR_NULL_ARG;
    const int n = (int)h->refs.size(), used = n - (int)h->unused.size();
    GUARD({
        std::vector<int> to((size_t)n, -1), holes;
        std::vector<int> left;                // the unused pages afterwards
        int moves = 0;
        for (int i = 0; i < used; i++)
            if (h->refs[(size_t)i] == 0) holes.push_back(i);
        if ((int)holes.size() > cap) return -LZ_ERR_NULL_ARG;
        left.reserve((size_t)n);
        for (int i = used; i < n; i++) left.push_back(i);
        std::priority_queue<int, std::vector<int>, std::greater<int>> q(std::greater<int>(), std::move(left));
        // from here nothing allocates
        for (int i = used; i < n; i++) {
            if (h->refs[(size_t)i] == 0) continue;
            src[moves] = i;
            dst[moves] = holes[(size_t)moves];
            to[(size_t)i] = dst[moves];
            h->refs[(size_t)dst[moves]] = h->refs[(size_t)i];
            h->refs[(size_t)i] = 0;
            moves++;
        }
        for (auto &s : h->seqs)
            for (int &p : s.pages)
                if (to[(size_t)p] >= 0) p = to[(size_t)p];
        h->unused.swap(q);
        return moves;
    })
}
