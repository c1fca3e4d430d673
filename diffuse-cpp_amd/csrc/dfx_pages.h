// dfx_pages.h — where the rows, keys and cells of a paged batch are: index arithmetic shared by
// the kernels and the host.  Every index that comes from device memory (row offsets, key counts,
// page ids) is bounded here, so that no content of those arrays reaches outside a buffer.
#pragma once
#include <stdint.h>

#include "dfx.h"

#define PG_BLOCK 16   // tokens per block: one scale, one transposed tile of values

// Kernel-side form of dfx_paged_cache and dfx_paged_batch.
struct paged_t {
    void * k;
    void * v;
    float * scale;
    const int32_t * rows;
    const int32_t * n_keys;
    const int32_t * pages;
    int64_t ld_pages;
    int32_t n_pages;
    int32_t page_shift;          // page_size = 1 << page_shift
    int32_t cap;                 // positions that a sequence's row of page ids covers
    int32_t Hkv;
    int32_t n_seqs, n_rows;
};

struct seq_t { int r0, n, keys; };   // first row, rows, keys

__host__ __device__ inline int pg_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

__host__ __device__ inline seq_t pg_seq(const paged_t & p, int s) {
    const int r0 = pg_clamp(p.rows[s], 0, p.n_rows), r1 = pg_clamp(p.rows[s + 1], 0, p.n_rows);
    return {r0, r1 > r0 ? r1 - r0 : 0, pg_clamp(p.n_keys[s], 0, p.cap)};
}

// Block (of the whole cache, head kvh) that holds position pos of sequence s, or -1: position
// outside the row of page ids, or no page.
__host__ __device__ inline int64_t pg_block(const paged_t & p, int s, int kvh, int pos) {
    if (pos < 0 || pos >= p.cap) return -1;
    const int page = p.pages[(int64_t)s * p.ld_pages + (pos >> p.page_shift)];
    if (page < 0 || page >= p.n_pages) return -1;
    const int bs = p.page_shift - 4;                     // log2 of a page's blocks
    return (((int64_t)page * p.Hkv + kvh) << bs) + ((pos >> 4) & ((1 << bs) - 1));
}

// Keys lo..hi (hi < lo: none) that the row at position pos sees.
struct seen_t { int lo, hi; };
__host__ __device__ inline seen_t pg_seen(int pos, int keys, int causal, int window) {
    if (!causal) return {0, keys - 1};
    const int hi = pos < keys ? pos : keys - 1;
    return {window > 0 && pos >= window ? pos - window + 1 : 0, hi};
}

// Tiles of 64 keys t0..t1-1 that the query tile of flat queries f0..f1 (G per row) sees.
struct tiles_t { int t0, t1; };
__host__ __device__ inline tiles_t pg_tiles(const seq_t & q, int f0, int f1, int G, int causal, int window) {
    const int p0 = q.keys - q.n;
    const int lo = pg_seen(p0 + f0 / G, q.keys, causal, window).lo;
    const int hi = pg_seen(p0 + f1 / G, q.keys, causal, window).hi;
    if (hi < lo) return {0, 0};
    return {lo >> 6, (hi >> 6) + 1};
}

// Key tiles of split `part` of n_parts at most, `chunk` tiles each (the last takes the rest, so that
// every key is covered whatever max_keys said).
struct part_at { int t0, t1, parts; };
__host__ __device__ inline part_at part_of(tiles_t r, int part, int chunk, int max_parts) {
    const int n = r.t1 - r.t0;
    const int parts = n <= 0 ? 1 : (n + chunk - 1) / chunk < max_parts ? (n + chunk - 1) / chunk : max_parts;
    if (part >= parts) return {0, 0, parts};
    const int a = r.t0 + part * chunk;
    return {a, part == parts - 1 ? r.t1 : a + chunk, parts};
}

// The kernel form of a cache and a batch (k_paged.hip); a status and its message where they are not
// sound.
int paged_of(const char * who, const dfx_paged_cache * c, const dfx_paged_batch * b, int n_head, paged_t * out);
