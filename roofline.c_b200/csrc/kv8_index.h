/* kv8_index.h -- the index arithmetic of the 8-bit key/value cache, apart
 * from any device code so that a host program can check it: which rows and
 * positions a sequence has, which pages they lie in, and which keys and
 * tiles a block of query rows reads. Everything a kernel dereferences is
 * bounded here. */
#ifndef TCG_KV8_INDEX_H
#define TCG_KV8_INDEX_H

#include <stdbool.h>
#include <stdint.h>

#ifdef __CUDACC__
#define KV8_FN __host__ __device__ __forceinline__ static
#else
#define KV8_FN static inline
#endif

#define KV8_PAGE_TOKENS 64

typedef struct {
    int row0, n, kv;      /* first row, new rows, cached tokens with them */
} kv8_seq_t;

/* False when a sequence's numbers cannot be: rows outside the call's n_tok,
 * more rows than max_new or than cached tokens, or more tokens than the
 * table's row has pages for. */
KV8_FN bool kv8_seq_ok(int start, int end, int kv, int n_tok, int max_new, int table_ld, kv8_seq_t *q)
{
    q->row0 = start;
    q->n = 0;
    q->kv = kv;
    if (start < 0 || end < start || end > n_tok || end - start > max_new || kv < end - start ||
        (long long)kv > (long long)table_ld * KV8_PAGE_TOKENS)
        return false;
    q->n = end - start;
    return true;
}

KV8_FN bool kv8_page_ok(int page, int n_pages) { return page >= 0 && page < n_pages; }

/* Pages that `longest` consecutive tokens can touch. */
KV8_FN int kv8_reach(int longest) { return longest < 1 ? 1 : (longest + KV8_PAGE_TOKENS - 2) / KV8_PAGE_TOKENS + 1; }

/* The j-th page that a sequence's new rows touch: its index in the table's
 * row, the slots lo .. hi - 1 of the new tokens and the row of slot lo.
 * False when there are fewer such pages. */
typedef struct {
    int index, lo, hi, row;
} kv8_place_t;
KV8_FN bool kv8_place(const kv8_seq_t *q, int j, kv8_place_t *at)
{
    const int first = q->kv - q->n, index = first / KV8_PAGE_TOKENS + j;
    const long long begin = (long long)index * KV8_PAGE_TOKENS;
    if (q->n == 0 || begin >= q->kv) return false;
    at->index = index;
    at->lo = first > begin ? (int)(first - begin) : 0;
    at->hi = q->kv - begin < KV8_PAGE_TOKENS ? (int)(q->kv - begin) : KV8_PAGE_TOKENS;
    at->row = q->row0 + (int)(begin + at->lo - first);
    return true;
}

/* Keys lo .. hi that token `tok` (0 .. n - 1) of a sequence sees; hi >= 0. */
KV8_FN int kv8_hi(const kv8_seq_t *q, int tok, int causal) { return causal ? q->kv - q->n + tok : q->kv - 1; }
KV8_FN int kv8_lo(const kv8_seq_t *q, int tok, int window)
{
    const int pos = q->kv - q->n + tok;
    return window && pos >= window ? pos - window + 1 : 0;
}

/* The tiles t0 + part, t0 + part + parts, ... < t1 of 64 keys that a part of
 * CTA `rank` of `ranks` reads for tokens tok_a .. tok_z; their count. */
KV8_FN int kv8_tiles(const kv8_seq_t *q, int tok_a, int tok_z, int causal, int window, int rank, int ranks, int part,
                     int parts, int *t0)
{
    const int first = kv8_lo(q, tok_a, window) / KV8_PAGE_TOKENS;
    const int tiles = kv8_hi(q, tok_z, causal) / KV8_PAGE_TOKENS + 1 - first, share = (tiles + ranks - 1) / ranks;
    const int a = first + rank * share, end = first + tiles;     /* below 2^26: a cache has at most 2^25 tiles */
    const int z = a + share < end ? a + share : end;
    *t0 = a + part;
    return z > a + part ? (z - a - part + parts - 1) / parts : 0;
}

#endif /* TCG_KV8_INDEX_H */
