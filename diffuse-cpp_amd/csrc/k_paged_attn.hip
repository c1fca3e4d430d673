// k_paged_attn.hip — attention of ragged batches over a paged cache.
//
// One pass over the keys with a running maximum m and sum l per query (scores in log2 units,
// s = q.k log2(e) / sqrt(hd)):
//   m' = max(m, s),  p = 2^(s - m'),  l' = l 2^(m - m') + sum p,  o' = o 2^(m - m') + p V,
// out = o / l.  Products on the f16 matrix cores with f32 sums: E4M3 cells times their block's
// power of two are f16 values exactly, so both cache types give exact operands.
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that a query is a column: it
// stays in one lane column of every accumulator, its maximum, sum and rescaling factor are one
// value per lane, and NaN of a query stays in its column.  The rows of the S^T tiles are numbered
// so that the scores a lane holds are 16 consecutive tokens of ONE block: that is the order in which
// the P^T operand wants them, so P never leaves the lane, V^T's operand is 16 consecutive cells of
// one value column, and the block's scale is one value per lane.
#include "dfx_device.h"
#include "dfx_pages.h"

#include <algorithm>
#include <atomic>

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

#define LOG2E_F 1.44269504088896341f

// eight cells as f16
__device__ __forceinline__ half8 f8_half8(uint32_t w0, uint32_t w1, float scale) {
    const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, false);
    const half2v b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, true);
    const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, false);
    const half2v d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, true);
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ float16v mfma32(half8 a, half8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float4v mfma16(half8 a, half8 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quad_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float quad_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// maximum / sum over the two lanes l, l ^ 32
__device__ __forceinline__ float half_max(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// An f32 value as two f16 terms (the second rounded: 2^-23 of the value where it is f16-normal).
__device__ __forceinline__ void split16(float x, half_t & hi, half_t & lo) {
    hi = (half_t)x;
    lo = (half_t)(x - (float)hi);
}

// Power of two by which an f32 query row is divided, so that its largest magnitude is in 2^8 .. 2^9
// and the second terms keep their bits (rows of zeros and of no finite magnitude are left).
__device__ __forceinline__ int q_exponent(float amax) {
    if (!(amax > 0.0f && amax <= 3.402823466e38f)) return 0;
    int ex;
    (void)frexpf(amax, &ex);
    return max(ex - 9, -100);
}

// NaN and infinities among the values.  A query that does not see a key has probability 0 for it, and
// 0 times such a value is NaN; a probability that is 0 in f16, or the second term of a split one (0 or
// negative), makes NaN of an infinite value that is seen.  So they are taken out of the products (0 in
// their place) and the key tiles that have them are noted, in a map of MAP_BITS tiles (tile modulo
// that: a tile noted for another costs time, not a result); at the end the cells of those tiles are
// looked through again, and what a query sees of them is added to its sums.
//
// The word's cells that are NaN or infinite (exponent, in E4M3 all bits, of ones): their top bits.
template <bool F8> __device__ __forceinline__ uint32_t special_bits(uint32_t w) {
    return F8 ? ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
template <bool F8> __device__ __forceinline__ uint32_t without_special(uint32_t w) {
    const uint32_t b = special_bits<F8>(w);
    return w & ~(F8 ? (b >> 7) * 0xffu : (b >> 15) * 0xffffu);
}
#define MAP_BITS 512
struct special_map {
    uint32_t w[MAP_BITS / 32];
    __device__ __forceinline__ void note(int t) { atomicOr(&w[(t & (MAP_BITS - 1)) >> 5], 1u << (t & 31)); }
    __device__ __forceinline__ bool has(int t) const { return w[(t & (MAP_BITS - 1)) >> 5] >> (t & 31) & 1u; }
    __device__ __forceinline__ bool any() const {
        uint32_t a = 0;
        for (int i = 0; i < MAP_BITS / 32; i++) a |= w[i];
        return a != 0;
    }
};

// ---------------------------------------------------------------------------
// Work: query tiles of ragged sequences
// ---------------------------------------------------------------------------
// A sequence's rows times the G heads of a KV head are its flat queries f = row * G + g, cut into
// tiles of T.  Tile t of the batch: found by a prefix sum over the sequences' tile counts, 64 at a
// time (one load each of row offsets and key counts for up to 64 sequences).
struct tile_at { int s, tile; seq_t q; };   // s < 0: no such tile
template <int T> __device__ __forceinline__ tile_at wave_tile(const paged_t & p, int G, int t) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < p.n_seqs; base += 64) {
        seq_t q = {0, 0, 0};
        if (base + lane < p.n_seqs) q = pg_seq(p, base + lane);
        const int cnt = (q.n * G + T - 1) / T;
        int sum = cnt;
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o, WAVE);
            if (lane >= o) sum += v;
        }
        const int total = __builtin_amdgcn_readlane(sum, 63);
        if (t < total) {
            const int from = __ffsll((unsigned long long)__ballot(sum > t)) - 1;
            return {base + from, t - __builtin_amdgcn_readlane(sum - cnt, from),
                    {__builtin_amdgcn_readlane(q.r0, from), __builtin_amdgcn_readlane(q.n, from),
                     __builtin_amdgcn_readlane(q.keys, from)}};
        }
        t -= total;
    }
    return {-1, 0, {0, 0, 0}};
}

// Sum over the wave, the same in every lane (and known to be: a scalar).
__device__ __forceinline__ int wave_sum_i(int v) {
    v += __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);        // within rows of 16 lanes
    v += __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true);
    v += __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true);
    return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) +
           (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}

template <int T> __device__ __forceinline__ tile_at one_tile(const paged_t & p, int G, int t) {
    const seq_t q = pg_seq(p, 0);
    return t < (q.n * G + T - 1) / T ? tile_at{0, t, q} : tile_at{-1, 0, {0, 0, 0}};
}

// The tiles of the batch in the order of their work, the ones with the most key tiles first (what runs
// last is short, and neighbours are alike: workgroups go to the parts of the chip in turn).  The weight
// k of tile t: the largest with more than t tiles of at least that weight, found bit by bit.  Up to 64
// sequences (a lane each); more: sequence by sequence, each from its end.  (4 causal prompts of 1600 to
// 3700 tokens: 261 us in the batch's order, 250 in this; interleaved by distance from the end 325.)
template <int T>
__device__ __forceinline__ tile_at wave_tile_by_work(const paged_t & p, int G, int causal, int window, int t) {
    const int lane = threadIdx.x & 63;
    if (p.n_seqs > 64 || p.n_seqs == 1) {
        tile_at at = p.n_seqs == 1 ? one_tile<T>(p, G, t) : wave_tile<T>(p, G, t);
        if (at.s >= 0) at.tile = (at.q.n * G + T - 1) / T - 1 - at.tile;
        return at;
    }
    seq_t q = {0, 0, 0};
    if (lane < p.n_seqs) q = pg_seq(p, lane);
    const int nq = q.n * G, cnt = (nq + T - 1) / T, p0 = q.keys - q.n;
    const int heaviest = window > 0 ? (window + 63) / 64 + 1 : 1 << 26;
    // the sequence's first tile of weight k or more: its last row sees position 64 (k - 1)
    auto first_of = [&](int k) {
        if (k <= 0) return 0;
        if (k > heaviest) return cnt;
        if (!causal) return 64 * (int64_t)(k - 1) < q.keys ? 0 : cnt;
        const int64_t f = ((int64_t)64 * (k - 1) - p0) * G;
        return f <= 0 ? 0 : f > nq - 1 ? cnt : (int)f / T;
    };
    const int most = cnt ? min(max(q.keys - 1, 0) / 64 + 1, heaviest) : 0;
    int k = 0;
    for (int bit = 1 << 25; bit > 0; bit >>= 1) {
        const int c = k | bit;
        if (!__any(most >= c)) continue;                           // no tile is that heavy
        if (wave_sum_i(cnt - first_of(c)) > t) k = c;
    }
    const int above = wave_sum_i(cnt - first_of(k + 1));           // tiles heavier than k
    const int from_k = first_of(k), mine = first_of(k + 1) - from_k;
    int sum = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(sum, o, WAVE);
        if (lane >= o) sum += v;
    }
    const uint64_t has = __ballot(above + sum > t);
    if (!has) return {-1, 0, {0, 0, 0}};
    const int from = __ffsll((unsigned long long)has) - 1;
    return {from, __builtin_amdgcn_readlane(from_k, from) + t - above - __builtin_amdgcn_readlane(sum - mine, from),
            {__builtin_amdgcn_readlane(q.r0, from), __builtin_amdgcn_readlane(q.n, from),
             __builtin_amdgcn_readlane(q.keys, from)}};
}

// Workgroup number -> (KV head, tile of the batch).  Workgroups go round the 8 XCDs, so head kvh's
// tiles are put on XCD kvh % 8 (with fewer heads, which divide 8, on 8 / Hkv XCDs each): an L2 holds the
// keys of its heads only.  Other head counts: heads in turn.
struct unit_at { int kvh, tile; };
__device__ __forceinline__ unit_at unit_of(int L, int Hkv, int tiles) {
    const int xcd = L & 7, j = L >> 3;
    if (Hkv >= 8) return {8 * (j / tiles) + xcd, j % tiles};
    if (8 % Hkv == 0) return {xcd % Hkv, j * (8 / Hkv) + xcd / Hkv};
    return {L % Hkv, L / Hkv};
}
static unsigned unit_grid(int Hkv, int tiles) {
    if (Hkv >= 8) return 8u * (unsigned)((Hkv + 7) / 8) * (unsigned)tiles;
    if (8 % Hkv == 0) return 8u * (unsigned)((tiles + 8 / Hkv - 1) / (8 / Hkv));
    return (unsigned)Hkv * (unsigned)tiles;
}

// Sum of the NaN and infinite values of column `dim` that a query sees among the noted tiles.
template <int HD, bool F8>
__device__ __forceinline__ float special_sum(const paged_t & p, const special_map & map, int s, int kvh, int dim,
                                                       int t0, int t1, seen_t see, int keys) {
    float sum = 0.0f;
#pragma unroll 1
    for (int t = t0; t < t1; t++) {
        if (!map.has(t - t0)) continue;
#pragma unroll 1
        for (int b = 0; b < 4; b++) {
            const int k0 = 64 * t + 16 * b;
            const int lo = pg_clamp(see.lo - k0, 0, 16), hi = pg_clamp(min(see.hi + 1, keys) - k0, 0, 16);
            if (hi <= lo) continue;
            const int64_t blk = pg_block(p, s, kvh, k0);
            if (blk < 0) continue;
#pragma unroll 1
            for (int j = lo; j < hi; j++) {
                if constexpr (F8) {
                    const uint8_t c = ((const uint8_t *)p.v)[(blk * HD + dim) * 16 + j];
                    if ((c & 0x7f) == 0x7f) sum += __builtin_nanf("");
                } else {
                    const uint16_t c = ((const uint16_t *)p.v)[(blk * HD + dim) * 16 + j];
                    if ((c & 0x7c00) == 0x7c00) sum += h2f(c);
                }
            }
        }
    }
    return sum;
}

struct attn_t {
    const void * q;
    void * out;
    float * part_o;      // [parts][n_rows * H][hd] unscaled sums
    float * part_ml;     // [parts][n_rows * H][2] maximum, sum
    int32_t * n_parts;   // [n_rows * H]
    int H, G, causal, window, chunk, parts, tiles;
};

// The four waves' maxima, sums and outputs ([4][T], [4][T], [4][T][HD + 4] in LDS) of a query tile as
// one: results, or a part of them.
template <int HD, bool F8, bool F32, int T>
__device__ __forceinline__ void join_waves(const paged_t & p, const attn_t & a, const tile_at & at, const part_at & pt,
                                           int kvh, int f0, int f1, const float * so, const float * sm,
                                           const float * sl, const special_map & map) {
    constexpr int OS = HD + 4;
    const int keys = at.q.keys, p0 = keys - at.q.n;
    const bool special = map.any();
    for (int e = threadIdx.x; e < T * (HD / 4); e += 256) {
        const int c = e / (HD / 4), d = 4 * (e % (HD / 4)), fc = f0 + c;
        if (fc > f1) continue;
        const float mx = fmaxf(fmaxf(sm[c], sm[T + c]), fmaxf(sm[2 * T + c], sm[3 * T + c]));
        float sum = 0.0f;
        float4v v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float mw = sm[w * T + c], lw = sl[w * T + c];
            const float r = mw == -INFINITY ? (lw == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(mw - mx);
            sum += r * lw;
            const float4v x = *(const float4v *)(so + (w * T + c) * OS + d);
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = fmaf(r, x[k], v[k]);
        }
        if (special)
#pragma unroll 1
            for (int k = 0; k < 4; k++) {
                const float add = special_sum<HD, F8>(p, map, at.s, kvh, d + k, pt.t0, pt.t1,
                                                      pg_seen(p0 + fc / a.G, keys, a.causal, a.window), keys);
                v.x += k == 0 ? add : 0.0f;
                v.y += k == 1 ? add : 0.0f;
                v.z += k == 2 ? add : 0.0f;
                v.w += k == 3 ? add : 0.0f;
            }
        const int64_t rh = (int64_t)(at.q.r0 + fc / a.G) * a.H + kvh * a.G + fc % a.G;
        if (F32) v *= 1.0f / 16384.0f;
        if (pt.parts == 1) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            v *= inv;
            if constexpr (F32) *(float4v *)((float *)a.out + rh * HD + d) = v;
            else *(half4 *)((half_t *)a.out + rh * HD + d) =
                    half4{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
        } else {
            const int64_t at_part = (int64_t)blockIdx.y * p.n_rows * a.H + rh;
            *(float4v *)(a.part_o + at_part * HD + d) = v;
        }
        if (d == 0 && a.parts > 1) {
            const int64_t at_part = (int64_t)blockIdx.y * p.n_rows * a.H + rh;
            if (blockIdx.y == 0) a.n_parts[rh] = pt.parts;
            if (pt.parts > 1) {
                a.part_ml[2 * at_part] = mx;
                a.part_ml[2 * at_part + 1] = sum;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Few rows: 16 queries per workgroup, keys straight from memory
// ---------------------------------------------------------------------------
// Bound by the cells' bytes, and where a workgroup has few tiles by its chain of loads (offsets, page,
// cells).  Four waves take the 64-key tiles of the workgroup's range in turn and join through LDS at
// the end.  Lane (i, g) = (lane % 16, lane / 16): query column i; S^T tile u (16 of the 64 keys): row
// 4b + r is token 4u + r of block b, so the lane's D values (rows 4g + r) over the four tiles are the 16
// tokens of block g.
// Measured: 64 sequences of one row, 32 heads of 128, 32469 E4M3 keys in all (266 MB) 70.5 us, 3.8 TB/s
// (5.1 in a copy); one row of 28 heads over 32701 keys of 4 KV heads (33.5 MB), in 64 parts, 13.5 us and
// 3.9 of the join.  64 equal ranges of 1001 keys: 97 us from E4M3 cells (5.4 TB/s), 179 from f16 (5.9).
// f32 queries of E4M3 caches are kept in LDS: in registers the third workgroup per CU spilled, and those 64
// ranges took 128 us, 102 so.  (f16 cells leave room for two workgroups either way: no difference.)
#define FEW_T 16
template <int HD, bool F8, bool F32>
__global__ void __launch_bounds__(256, !F8 ? (HD == 64 ? 3 : 2) : HD == 64 ? 4 : 3) k_paged_few(paged_t p, attn_t a) {
    constexpr int KS = HD / 32;                 // 32-dim steps of S
    constexpr int DT = HD / 16;                 // 16-dim tiles of O
    constexpr int KW = F8 ? HD / 64 : HD / 32;  // 16-byte loads of a lane per S tile
    constexpr int VW = F8 ? 1 : 2;              // 16-byte loads of a lane per O tile
    constexpr int OS = HD + 4;                  // LDS floats per query
    constexpr bool QL = F32 && F8;              // Q's terms in LDS, read in every turn
    __shared__ __attribute__((aligned(16))) float so[4][FEW_T][OS];         // Q's terms, then the waves' sums
    static_assert(sizeof(so) >= KS * 2 * 64 * sizeof(half8), "room for Q's terms");
    __shared__ float sm[4][FEW_T], sl[4][FEW_T];
    __shared__ special_map map;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const unit_at un = unit_of(blockIdx.x, p.Hkv, a.tiles);
    if (un.kvh >= p.Hkv) return;
    const tile_at at = wave_tile_by_work<FEW_T>(p, a.G, a.causal, a.window, un.tile);
    if (at.s < 0) return;
    const int nq = at.q.n * a.G, f0 = at.tile * FEW_T, f1 = min(f0 + FEW_T, nq) - 1;
    const part_at pt = part_of(pg_tiles(at.q, f0, f1, a.G, a.causal, a.window), blockIdx.y, a.chunk, a.parts);
    if ((int)blockIdx.y >= pt.parts) return;
    const int p0 = at.q.keys - at.q.n, keys = at.q.keys;
    // keys that every query of the tile sees, and this lane's
    const int all_lo = pg_seen(p0 + f1 / a.G, keys, a.causal, a.window).lo;
    const int all_hi = pg_seen(p0 + f0 / a.G, keys, a.causal, a.window).hi;
    const int f = min(f0 + i, f1), row = at.q.r0 + f / a.G, head = un.kvh * a.G + f % a.G;
    const seen_t me = pg_seen(p0 + f / a.G, keys, a.causal, a.window);

    // ---- Q: step s holds dims in the order in which the lane's key loads bring them
    half8 qh[QL ? 1 : KS], ql[QL ? 1 : KS];
    half8 * const qs = (half8 *)&so[0][0][0] + lane;    // step s: the terms at 128 s and 128 s + 64
    float sc = LOG2E_F / sqrtf((float)HD);
    {
        const int64_t qo = ((int64_t)row * a.H + head) * HD;
        auto dim = [&](int s) { return F8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };
        if constexpr (F32) {
            float x[KS][8];
            float amax = 0.0f;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const float * src = (const float *)a.q + qo + dim(s);
                const float4 u = *(const float4 *)src, v = *(const float4 *)(src + 4);
                const float e[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    x[s][k] = e[k];
                    amax = fmaxf(amax, fabsf(e[k]));
                }
            }
            const int ex = q_exponent(quad_max(amax));
            sc = ldexpf(sc, ex);
#pragma unroll
            for (int s = 0; s < KS; s++) {
                half8 th, tl;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    half_t hi, lo;
                    split16(ldexpf(x[s][k], -ex), hi, lo);
                    th[k] = hi;
                    tl[k] = lo;
                }
                if constexpr (!QL) {
                    qh[s] = th;
                    ql[s] = tl;
                } else if (s % 4 == wv) {                           // the four waves' queries are the same
                    qs[128 * s] = th;
                    qs[128 * s + 64] = tl;
                }
            }
        } else {
#pragma unroll
            for (int s = 0; s < KS; s++) qh[s] = *(const half8 *)((const half_t *)a.q + qo + dim(s));
        }
    }

    if (threadIdx.x < MAP_BITS / 32) map.w[threadIdx.x] = 0;
    __syncthreads();
    float m, l;
    float4v o[DT];

    // Q is waited for here, not inside the loop (where the wait would be for the next tile's loads)
    if constexpr (!QL)
#pragma unroll
        for (int c = 0; c < KS; c++) {
            asm volatile("" : "+v"(qh[c]));
            if constexpr (F32) asm volatile("" : "+v"(ql[c]));
        }

    // Keys and values take turns in the same registers: the tile's values are loaded when its scores are
    // taken, the next tile's keys when the values are added.  That leaves room for three workgroups per CU
    // (E4M3, 128 dims: 168 registers), whose waves hide each other's loads (the 64 sequences above: 70.5 us;
    // 78 with keys and values in registers of their own, 141 with both of the next tile on their way); the
    // next tile's pages are looked up a tile earlier.
    constexpr int CB = F8 ? 1 : 2;
    const int bs = p.page_shift - 4;                                // log2 of a page's blocks
    int page_k = -1, page_v = -1, have = 0;
    float ks = 1.0f, vs = 1.0f;
    static_assert(4 * KW == DT * VW, "keys and values of a tile");
    u32x4 cells[4 * KW];
    auto page_of = [&](int pos) __attribute__((always_inline)) {
        const int pg = pos < p.cap ? p.pages[(int64_t)at.s * p.ld_pages + (pos >> p.page_shift)] : -1;
        return pg < p.n_pages ? pg : -1;
    };
    // block of the cache; where there is no page, block 0: read and not used
    auto block_of = [&](int pg, int blk) __attribute__((always_inline)) {
        return pg < 0 ? (int64_t)0 : (((int64_t)pg * p.Hkv + un.kvh) << bs) + (blk & ((1 << bs) - 1));
    };
    auto look_up = [&](int t) __attribute__((always_inline)) {
        if (t >= pt.t1) return;
        page_k = page_of(64 * t + 16 * (i >> 2));
        page_v = page_of(64 * t + 16 * g);
    };
    auto load_k = [&](int t) __attribute__((always_inline)) {
        const int64_t blk = block_of(page_k, 4 * t + (i >> 2));
        const uint8_t * kp = (const uint8_t *)p.k + (blk * (16 * HD) + (i & 3) * HD + (F8 ? 16 : 8) * g) * CB;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int w = 0; w < KW; w++) cells[u * KW + w] = *(const u32x4 *)(kp + 4 * u * HD * CB + 64 * w);
        if constexpr (F8) ks = p.scale[2 * blk];
    };
    auto load_v = [&](int t) __attribute__((always_inline)) {
        const int64_t blk = block_of(page_v, 4 * t + g);
        const uint8_t * vp = (const uint8_t *)p.v + (blk * (16 * HD) + i * 16) * CB;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int w = 0; w < VW; w++) cells[d * VW + w] = *(const u32x4 *)(vp + (d * 16 * 16) * CB + 16 * w);
        have = page_v < 0 ? 0 : pg_clamp(keys - (64 * t + 16 * g), 0, 16);   // tokens of the lane's block that exist
        if constexpr (F8) {
            vs = p.scale[2 * blk + 1];
            if (have == 0) vs = 1.0f;                               // no page, or not written: anything, NaN too
        }
    };
    bool careful = false;                                           // this wave alone: nothing is shared here
    while (true) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = float4v{0.f, 0.f, 0.f, 0.f};
        {
            const int t = pt.t0 + wv;
            if (t < pt.t1) {
                look_up(t);
                load_k(t);
            }
        }
        for (int t = pt.t0 + wv; t < pt.t1; t += 4) {
            if constexpr (QL) asm volatile("" ::: "memory");       // not kept in registers from turn to turn
            half8 qa[KS], qb[KS];
#pragma unroll
            for (int c = 0; c < KS; c++) {
                qa[c] = QL ? qs[128 * c] : qh[QL ? 0 : c];
                if constexpr (F32) qb[c] = QL ? qs[128 * c + 64] : ql[QL ? 0 : c];
            }
            float s[16];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < KW; w++) {
                    if constexpr (F8) {
                        const u32x4 c = cells[u * KW + w];
                        const half8 k0 = f8_half8(c.x, c.y, ks), k1 = f8_half8(c.z, c.w, ks);
                        acc = mfma16(k0, qa[2 * w], acc);
                        acc = mfma16(k1, qa[2 * w + 1], acc);
                        if constexpr (F32) {
                            acc = mfma16(k0, qb[2 * w], acc);
                            acc = mfma16(k1, qb[2 * w + 1], acc);
                        }
                    } else {
                        const half8 k0 = __builtin_bit_cast(half8, cells[u * KW + w]);
                        acc = mfma16(k0, qa[w], acc);
                        if constexpr (F32) acc = mfma16(k0, qb[w], acc);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) s[4 * u + r] = acc[r] * sc;
            }
            load_v(t);
            look_up(t + 4);
            // every key of the tile is there and every query sees it
            const bool full = __all(have == 16) && 64 * t >= all_lo && 64 * t + 63 <= all_hi;
            if (!full) {
                const int k0 = 64 * t + 16 * g;
                const int lo = pg_clamp(me.lo - k0, 0, 16), hi = pg_clamp(min(me.hi + 1 - k0, have), 0, 16);
#pragma unroll
                for (int k = 0; k < 16; k++) s[k] = k >= lo && k < hi ? s[k] : -INFINITY;
            }
            float tm = s[0];
#pragma unroll
            for (int k = 1; k < 16; k++) tm = fmaxf(tm, s[k]);
            tm = fmaxf(quad_max(tm), m);
            if (__any(tm > m)) {
                const float r = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - tm);
                l *= r;
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] *= r;
                m = tm;
            }
            // 2^14 p goes into the products, in f16: small probabilities keep their bits.  With f16 results
            // the exponent carries the factor (l has it too); for f32 results it is applied after, as the
            // exponent's rounding would show.  Nothing seen yet: every p is 0.
            const float mm = (m == -INFINITY ? 0.0f : m) - (F32 ? 0.0f : 14.0f);
            half8 ph[2], pl[2];
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const float e = __builtin_amdgcn_exp2f(s[k] - mm);
                l += e;
                if constexpr (F32) {
                    half_t hi, lo;
                    split16(e * 16384.0f, hi, lo);
                    ph[k >> 3][k & 7] = hi;
                    pl[k >> 3][k & 7] = lo;
                } else {
                    ph[k >> 3][k & 7] = (half_t)e;
                }
            }
            if (!full) {
                // cells of tokens that do not exist are taken as 0
                if (__any(have < 16)) {
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int w = 0; w < VW; w++)
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                constexpr int PER = F8 ? 4 : 2;          // tokens per word
                                const int n = have - PER * (4 * w + c);  // of which exist
                                const uint32_t keep = n >= PER ? 0xffffffffu : n <= 0 ? 0u : (1u << (n * (32 / PER))) - 1u;
                                cells[d * VW + w][c] &= keep;
                            }
                }
            }
            if (careful) {
                uint32_t sp = 0;
#pragma unroll
                for (int c = 0; c < DT * VW; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        sp |= special_bits<F8>(cells[c][e]);
                        cells[c][e] = without_special<F8>(cells[c][e]);
                    }
                if (sp) map.note(t - pt.t0);
            }
#pragma unroll
            for (int d = 0; d < DT; d++) {
                half8 v0, v1;
                if constexpr (F8) {
                    v0 = f8_half8(cells[d * VW].x, cells[d * VW].y, vs);
                    v1 = f8_half8(cells[d * VW].z, cells[d * VW].w, vs);
                } else {
                    v0 = __builtin_bit_cast(half8, cells[d * VW]);
                    v1 = __builtin_bit_cast(half8, cells[d * VW + VW - 1]);
                }
                o[d] = mfma16(v0, ph[0], o[d]);
                o[d] = mfma16(v1, ph[1], o[d]);
                if constexpr (F32) {
                    o[d] = mfma16(v0, pl[0], o[d]);
                    o[d] = mfma16(v1, pl[1], o[d]);
                }
            }
            if (t + 4 < pt.t1) load_k(t + 4);
        }
        if (careful) break;
        bool odd = false;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 4; r++) odd |= !(fabsf(o[d][r]) <= 3.402823466e38f);
        if (!__any(odd)) break;
        careful = true;
    }

    // ---- the four waves' results
    l = quad_sum(l);
    if constexpr (QL) __syncthreads();                              // Q has been read
    if (g == 0) {
        sm[wv][i] = m;
        sl[wv][i] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; d++) *(float4v *)&so[wv][i][16 * d + 4 * g] = o[d];
    __syncthreads();
    join_waves<HD, F8, F32, FEW_T>(p, a, at, pt, un.kvh, f0, f1, &so[0][0][0], &sm[0][0], &sl[0][0], map);
}

// ---------------------------------------------------------------------------
// Some rows: 32 queries per workgroup, keys straight from memory
// ---------------------------------------------------------------------------
// k_paged_few with the wider product (32 x 32), which takes half the key reads and matrix operands per
// query: four waves take the key steps of the workgroup's range in turn and join through LDS.  A step is KT
// keys, 64 in 8 bits, 32 in f16 (registers).  Lane (i, h) = (lane % 32, lane / 32), rows of the S^T tiles
// as in k_paged_many: a lane's 16 D values of tile u are the tokens of block 2u + h in order.
// Bound by latency: two or three workgroups' work per CU.  f32 queries of E4M3 caches are in LDS: registers
// for two workgroups per CU instead of one (4 x 128 rows of 32 heads over 828 keys 44.3 us, 30.3 so; with
// f16 cells two fit either way, and three, with Q in LDS, spill: 29.3 us to 36.5).  Measured: 429 f32 rows of 8 sequences, 32 heads of
// 128, 4525 f16 keys (88 MB) 29.3 us, 3.0 TB/s, the matrix cores busy 13 % of the time; 1414 rows of 6
// sequences, 8 heads of 64 on 2 KV heads, a window of 512: 11.8 us.
#define MID_T 32
template <int HD, bool F8, bool F32>
__global__ void __launch_bounds__(256, 2) k_paged_mid(paged_t p, attn_t a) {
    constexpr int U = F8 ? 2 : 1, KT = 32 * U;
    constexpr int QS = HD / 16, DT = HD / 32;
    constexpr int KW = F8 ? HD / 32 : HD / 16;  // 16-byte loads of a lane per S tile
    constexpr int VW = F8 ? 1 : 2;              // 16-byte loads of a lane per O tile and S tile
    constexpr int CB = F8 ? 1 : 2;
    constexpr int OS = HD + 4;                  // LDS floats per query
    constexpr bool QL = F32 && F8;              // Q's terms in LDS, read in every turn
    extern __shared__ __attribute__((aligned(16))) float so[];              // Q's terms, then [4][MID_T][OS]
    __shared__ float sm[4][MID_T], sl[4][MID_T];
    __shared__ special_map map;
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unit_at un = unit_of(blockIdx.x, p.Hkv, a.tiles);
    if (un.kvh >= p.Hkv) return;
    const tile_at at = wave_tile_by_work<MID_T>(p, a.G, a.causal, a.window, un.tile);
    if (at.s < 0) return;
    const int nq = at.q.n * a.G, f0 = at.tile * MID_T, f1 = min(f0 + MID_T, nq) - 1;
    const tiles_t all = pg_tiles(at.q, f0, f1, a.G, a.causal, a.window);
    const part_at pt = {all.t0, all.t1, 1};
    const int keys = at.q.keys, p0 = keys - at.q.n;
    const int all_lo = pg_seen(p0 + f1 / a.G, keys, a.causal, a.window).lo;
    const int all_hi = pg_seen(p0 + f0 / a.G, keys, a.causal, a.window).hi;
    const int f = min(f0 + i, f1), row = at.q.r0 + f / a.G, head = un.kvh * a.G + f % a.G;
    const seen_t me = pg_seen(p0 + f / a.G, keys, a.causal, a.window);

    // ---- Q: step c holds dims in the order in which the lane's key loads bring them
    half8 qh[QL ? 1 : QS], ql[F32 && !QL ? QS : 1];
    half8 * const qs = (half8 *)so + lane;      // step c: the terms at 128 c and 128 c + 64
    float sc = LOG2E_F / sqrtf((float)HD);
    {
        const int64_t qo = ((int64_t)row * a.H + head) * HD;
        auto dim = [&](int c) { return F8 ? 32 * (c >> 1) + 16 * h + 8 * (c & 1) : 16 * c + 8 * h; };
        if constexpr (F32) {
            float x[QS][8];
            float amax = 0.0f;
#pragma unroll
            for (int c = 0; c < QS; c++) {
                const float * src = (const float *)a.q + qo + dim(c);
                const float4 u = *(const float4 *)src, v = *(const float4 *)(src + 4);
                const float e[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    x[c][k] = e[k];
                    amax = fmaxf(amax, fabsf(e[k]));
                }
            }
            const int ex = q_exponent(half_max(amax));
            sc = ldexpf(sc, ex);
#pragma unroll
            for (int c = 0; c < QS; c++) {
                half8 th, tl;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    half_t hi, lo;
                    split16(ldexpf(x[c][k], -ex), hi, lo);
                    th[k] = hi;
                    tl[k] = lo;
                }
                if constexpr (!QL) {
                    qh[c] = th;
                    ql[c] = tl;
                } else if (c % 4 == wv) {                           // the four waves' queries are the same
                    qs[128 * c] = th;
                    qs[128 * c + 64] = tl;
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < QS; c++) qh[c] = *(const half8 *)((const half_t *)a.q + qo + dim(c));
        }
    }
    if (threadIdx.x < MAP_BITS / 32) map.w[threadIdx.x] = 0;
    __syncthreads();
    if constexpr (!QL)
#pragma unroll
        for (int c = 0; c < QS; c++) {                              // waited for here, as in k_paged_few
            asm volatile("" : "+v"(qh[c]));
            if constexpr (F32) asm volatile("" : "+v"(ql[c]));
        }

    const int bs = p.page_shift - 4;
    const int s0 = pt.t0 * (64 / KT), s1 = pt.t1 * (64 / KT);       // key steps
    int page_k[U], page_v[U], have[U];
    float ks[U], vs[U];
    static_assert(KW == DT * VW, "keys and values of a step");
    u32x4 cells[U][KW];                                             // keys, then values, as in k_paged_few
    auto page_of = [&](int pos) __attribute__((always_inline)) {
        const int pg = pos < p.cap ? p.pages[(int64_t)at.s * p.ld_pages + (pos >> p.page_shift)] : -1;
        return pg < p.n_pages ? pg : -1;
    };
    auto block_of = [&](int pg, int blk) __attribute__((always_inline)) {
        return pg < 0 ? (int64_t)0 : (((int64_t)pg * p.Hkv + un.kvh) << bs) + (blk & ((1 << bs) - 1));
    };
    // blocks (counted over the sequence) of the lane's key row and of its values in tile u of step s
    auto blk_k = [&](int s, int u) { return s * (KT / 16) + 2 * u + ((i >> 2) & 1); };
    auto blk_v = [&](int s, int u) { return s * (KT / 16) + 2 * u + h; };
    auto look_up = [&](int s) __attribute__((always_inline)) {
        if (s >= s1) return;
#pragma unroll
        for (int u = 0; u < U; u++) {
            page_k[u] = page_of(16 * blk_k(s, u));
            page_v[u] = page_of(16 * blk_v(s, u));
        }
    };
    auto load_k = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t blk = block_of(page_k[u], blk_k(s, u));
            const uint8_t * kp = (const uint8_t *)p.k + (blk * 16 + 4 * (i >> 3) + (i & 3)) * (HD * CB) + 16 * h;
#pragma unroll
            for (int w = 0; w < KW; w++) cells[u][w] = *(const u32x4 *)(kp + 32 * w);
            ks[u] = 1.0f;
            if constexpr (F8) ks[u] = p.scale[2 * blk];
        }
    };
    auto load_v = [&](int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t blk = block_of(page_v[u], blk_v(s, u));
            const uint8_t * vp = (const uint8_t *)p.v + (blk * HD + i) * (16 * CB);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int w = 0; w < VW; w++) cells[u][d * VW + w] = *(const u32x4 *)(vp + 32 * d * 16 * CB + 16 * w);
            have[u] = page_v[u] < 0 ? 0 : pg_clamp(keys - 16 * blk_v(s, u), 0, 16);
            vs[u] = 1.0f;
            if constexpr (F8) {
                vs[u] = p.scale[2 * blk + 1];
                if (have[u] == 0) vs[u] = 1.0f;
            }
        }
    };

    float m, l;
    float16v o[DT];
    bool careful = false;                                           // this wave alone: nothing is shared here
    while (true) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
        if (s0 + wv < s1) {
            look_up(s0 + wv);
            load_k(s0 + wv);
        }
        for (int st = s0 + wv; st < s1; st += 4) {
            if constexpr (QL) asm volatile("" ::: "memory");       // not kept in registers from turn to turn
            float16v s[U];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[u][r] = 0.0f;
#pragma unroll
            for (int c = 0; c < QS; c++) {
                half8 qa, qb;
                if constexpr (QL) {
                    qa = qs[128 * c];
                    qb = qs[128 * c + 64];
                } else {
                    qa = qh[c];
                    if constexpr (F32) qb = ql[c];
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    half8 k;
                    if constexpr (F8) {
                        const u32x4 w = cells[u][c / 2];
                        k = c % 2 ? f8_half8(w.z, w.w, ks[u]) : f8_half8(w.x, w.y, ks[u]);
                    } else {
                        k = __builtin_bit_cast(half8, cells[u][c]);
                    }
                    s[u] = mfma32(k, qa, s[u]);
                    if constexpr (F32) s[u] = mfma32(k, qb, s[u]);
                }
            }
            load_v(st);
            look_up(st + 4);
            bool there = true;
#pragma unroll
            for (int u = 0; u < U; u++) there &= have[u] == 16;
            const bool full = __all(there) && KT * st >= all_lo && KT * st + KT - 1 <= all_hi;
            if (!full) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int k0 = 16 * blk_v(st, u);
                    const int lo = pg_clamp(me.lo - k0, 0, 16), hi = pg_clamp(min(me.hi + 1 - k0, have[u]), 0, 16);
#pragma unroll
                    for (int r = 0; r < 16; r++) s[u][r] = r >= lo && r < hi ? s[u][r] : -INFINITY;
                }
            }
            float tm = s[0][0];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) tm = fmaxf(tm, s[u][r]);
            tm = fmaxf(half_max(tm) * sc, m);
            if (__any(tm > m)) {
                const float r = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - tm);
                l *= r;
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] *= r;
                m = tm;
            }
            // 2^14 p goes into the products, as in k_paged_few
            const float mm = (F32 ? 0.0f : 14.0f) - (m == -INFINITY ? 0.0f : m);
            half8 ph[2 * U], pl[F32 ? 2 * U : 1];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[u][r], sc, mm));
                    l += e;
                    if constexpr (F32) {
                        half_t hi, lo;
                        split16(e * 16384.0f, hi, lo);
                        ph[2 * u + (r >> 3)][r & 7] = hi;
                        pl[2 * u + (r >> 3)][r & 7] = lo;
                    } else {
                        ph[2 * u + (r >> 3)][r & 7] = (half_t)e;
                    }
                }
            if (!full) {
                // cells of tokens that do not exist are taken as 0
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int w = 0; w < VW; w++)
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                constexpr int PER = F8 ? 4 : 2;
                                const int n = have[u] - PER * (4 * w + c);
                                cells[u][d * VW + w][c] &= n >= PER ? 0xffffffffu : n <= 0 ? 0u : (1u << (n * (32 / PER))) - 1u;
                            }
            }
            if (careful) {
                uint32_t sp = 0;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int c = 0; c < KW; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            sp |= special_bits<F8>(cells[u][c][e]);
                            cells[u][c][e] = without_special<F8>(cells[u][c][e]);
                        }
                if (sp) map.note(st / (64 / KT) - pt.t0);
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        half8 v;
                        if constexpr (F8)
                            v = j ? f8_half8(cells[u][d * VW].z, cells[u][d * VW].w, vs[u])
                                  : f8_half8(cells[u][d * VW].x, cells[u][d * VW].y, vs[u]);
                        else
                            v = __builtin_bit_cast(half8, cells[u][d * VW + j]);
                        o[d] = mfma32(v, ph[2 * u + j], o[d]);
                        if constexpr (F32) o[d] = mfma32(v, pl[2 * u + j], o[d]);
                    }
            if (st + 4 < s1) load_k(st + 4);
        }
        if (careful) break;
        bool odd = false;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) odd |= !(fabsf(o[d][r]) <= 3.402823466e38f);
        if (!__any(odd)) break;
        careful = true;
    }

    // ---- the four waves' results
    l = half_sum(l);
    if constexpr (QL) __syncthreads();                              // Q has been read
    if (h == 0) {
        sm[wv][i] = m;
        sl[wv][i] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int b = 0; b < 4; b++)
            *(float4v *)&so[(wv * MID_T + i) * OS + 32 * d + 8 * b + 4 * h] =
                float4v{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
    __syncthreads();
    join_waves<HD, F8, F32, MID_T>(p, a, at, pt, un.kvh, f0, f1, so, &sm[0][0], &sl[0][0], map);
}

// ---------------------------------------------------------------------------
// Many rows: 32 queries per wave, keys through LDS
// ---------------------------------------------------------------------------
// Bound by issue: the matrix instructions, the exponentials and the loader's conversions of two waves per
// SIMD do not overlap fully.  Four waves share tiles of 64 keys in LDS, in f16 (so an E4M3 cell is
// converted once for all of them), two buffers: while a tile is multiplied, the next one goes from
// registers to LDS and the one after it is on its way to registers; one barrier per tile.  Lane (i, h) = (lane % 32,
// lane / 32): query column i; S^T tile u (32 of the 64 keys): row 8a + 4b + r is token 4a + r of block
// 2u + b, so the lane's 16 D values are the 16 tokens of block 2u + h in order.
// LDS: K by 8-dim chunks, [HD / 8][64 tokens in S^T row order][16 B]; V by halves of blocks,
// [4 blocks][2][HD][16 B]: every operand read is 64 lanes of consecutive 16 bytes per half wave.
// The running maximum is let lag (by up to 2^8): sums are rescaled only where it moves further.
// Measured: 4 causal prompts, 9716 rows of 28 heads on 4 E4M3 KV heads of 128, 188.6 GFLOP: 239 us, 789
// TFLOP/s (a library's square f16 product of 8192: 1212), the matrix cores busy 37 % of the time.  Of 250 us
// in an earlier state the loads took 28, the stores to LDS and their conversions 33, the exponentials 11
// (each left out in turn).  Other forms, beside 250: 64 queries a wave (two columns of tiles) 405, as the
// accumulators no longer fit the vector registers; 256 queries a workgroup 254; scores of the next tile
// taken before this one's values are added 258-275.
template <int HD> struct many_lds {
    static constexpr int KS = 64 * 16 + 16;             // bytes per key chunk (the rest of a bank row: writes spread)
    static constexpr int VS = HD * 16 + 64;             // bytes per half block of values
    static constexpr int K = (HD / 8) * KS, V = 8 * VS;
    static constexpr int FLAGS = 12 * 4 + (int)sizeof(special_map);      // per buffer: 4 counts of tokens; one mark
    static constexpr int BYTES = 2 * (K + V) + FLAGS;
};

#define MANY_WAVES 4
#define MANY_T (32 * MANY_WAVES)
template <int HD, bool F8, bool F32>
__global__ void __launch_bounds__(64 * MANY_WAVES, 2) k_paged_many(paged_t p, attn_t a) {
    constexpr int NT = 64 * MANY_WAVES, T = 32 * MANY_WAVES;
    constexpr int CB = F8 ? 1 : 2;
    constexpr int QS = HD / 16;                         // 16-dim steps of S
    constexpr int DT = HD / 32;                         // 32-dim tiles of O
    constexpr int UNITS = 64 * HD * CB / 16;            // 16-byte units of a tile of K (as many of V)
    constexpr int LU = UNITS / NT;                      // of them per thread
    constexpr int PER_BLOCK = UNITS / 4;
    using lds_t = many_lds<HD>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int * flags = (int *)(lds + 2 * (lds_t::K + lds_t::V));      // [2][4], the mark of a careful pass
    special_map & map = *(special_map *)(flags + 12);
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unit_at un = unit_of(blockIdx.x, p.Hkv, a.tiles);
    if (un.kvh >= p.Hkv) return;
    const tile_at at = wave_tile_by_work<T>(p, a.G, a.causal, a.window, un.tile);
    if (at.s < 0) return;
    const int nq = at.q.n * a.G;
    const int f0 = at.tile * T, f1 = min(f0 + T, nq) - 1;
    const tiles_t pt = pg_tiles(at.q, f0, f1, a.G, a.causal, a.window);
    const int keys = at.q.keys, p0 = keys - at.q.n;
    // this wave's queries, the keys that all and that any of them see
    const int w0 = f0 + 32 * wv, w1 = min(w0 + 31, f1);
    const bool idle = w0 > f1;
    const seen_t first = pg_seen(p0 + min(w0, f1) / a.G, keys, a.causal, a.window);
    const seen_t last = pg_seen(p0 + max(w1, 0) / a.G, keys, a.causal, a.window);
    const int f = min(w0 + i, f1), row = at.q.r0 + f / a.G, head = un.kvh * a.G + f % a.G;
    const seen_t me = pg_seen(p0 + f / a.G, keys, a.causal, a.window);

    // ---- loader: this thread's 16-byte units of a tile.  A unit's block is the same for its whole wave, but
    // its page and scales are held per lane (loads through the vector cache, counted with the cells', not
    // scalar ones, which would be waited for with the LDS reads).
    u32x4 kr[LU], vr[LU];
    f32x2 scale[LU];
    int page[LU], have[LU];
    int zero;
    asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
    const int32_t * const pages = p.pages + (int64_t)at.s * p.ld_pages + zero;
    const int bs = p.page_shift - 4;                    // log2 of a page's blocks
    const uint32_t page_units = (uint32_t)p.Hkv << bs;  // blocks of a page
    // unit w: number `in` of block b0 + BW w
    constexpr int BW = NT / PER_BLOCK;
    static_assert(NT % PER_BLOCK == 0 && BW * LU == 4, "whole blocks");
    const int b0 = __builtin_amdgcn_readfirstlane(tid / PER_BLOCK), in = tid % PER_BLOCK;
    uint32_t lk, lv;                                    // where unit 0 goes in LDS; the others at k_step, v_step
    {
        constexpr int ROW = HD * CB / 16;               // units per token
        const int tok = in / ROW, c = in % ROW;
        const int slot = 32 * (b0 >> 1) + 8 * (tok >> 2) + 4 * (b0 & 1) + (tok & 3);
        lk = (F8 ? 2 * c : c) * lds_t::KS + slot * 16;
        lv = lds_t::K + (F8 ? 2 * b0 * lds_t::VS + in * 16 : (2 * b0 + (in & 1)) * lds_t::VS + (in >> 1) * 16);
    }
    auto k_step = [](int w) { return BW == 1 ? (32 * (w >> 1) + 4 * (w & 1)) * 16 : 32 * (BW / 2) * w * 16; };
    auto v_step = [](int w) { return 2 * BW * w * lds_t::VS; };
    auto look_up = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < LU; w++) {
            const int pos = 64 * t + 16 * (b0 + BW * w);
            page[w] = -1;
            if (t < pt.t1 && pos < p.cap) page[w] = pages[pos >> p.page_shift];
        }
    };
    auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int w = 0; w < LU; w++) {
            const int b = b0 + BW * w;
            const bool is = (uint32_t)page[w] < (uint32_t)p.n_pages;
            // no page: page 0, not used
            const uint64_t blk = (uint64_t)(is ? (uint32_t)page[w] : 0u) * page_units +
                                 (uint32_t)((un.kvh << bs) + ((4 * t + b) & ((1 << bs) - 1)));
            const uint64_t unit = blk * PER_BLOCK + in;
            kr[w] = ((const u32x4 *)p.k)[unit];
            vr[w] = ((const u32x4 *)p.v)[unit];
            have[w] = is ? pg_clamp(keys - 64 * t - 16 * b, 0, 16) : 0;
            if constexpr (F8) {
                scale[w] = *(const f32x2 *)(p.scale + 2 * blk);
                if (have[w] == 0) scale[w] = f32x2{1.0f, 1.0f};         // no page, or not written: anything, NaN too
            }
        }
        look_up(t + 1);
    };
    bool careful = false;
    auto store = [&](int buf, int t) __attribute__((always_inline)) {
        uint8_t * to = lds + buf * (lds_t::K + lds_t::V);
#pragma unroll
        for (int w = 0; w < LU; w++) {
            if constexpr (F8) {
                *(half8 *)(to + lk + k_step(w)) = f8_half8(kr[w].x, kr[w].y, scale[w].x);
                *(half8 *)(to + lk + k_step(w) + lds_t::KS) = f8_half8(kr[w].z, kr[w].w, scale[w].x);
            } else {
                *(u32x4 *)(to + lk + k_step(w)) = kr[w];
            }
            // cells of tokens that do not exist are taken as 0
            if (__any(have[w] < 16)) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    constexpr int PER = F8 ? 4 : 2;                          // tokens per word
                    const int n = have[w] - PER * (4 * (F8 ? 0 : in & 1) + k);
                    vr[w][k] &= n >= PER ? 0xffffffffu : n <= 0 ? 0u : (1u << (n * (32 / PER))) - 1u;
                }
            }
            if (careful) {
                uint32_t sp = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    sp |= special_bits<F8>(vr[w][k]);
                    vr[w][k] = without_special<F8>(vr[w][k]);
                }
                if (sp) map.note(t - pt.t0);
            }
            if constexpr (F8) {
                *(half8 *)(to + lv + v_step(w)) = f8_half8(vr[w].x, vr[w].y, scale[w].y);
                *(half8 *)(to + lv + v_step(w) + lds_t::VS) = f8_half8(vr[w].z, vr[w].w, scale[w].y);
            } else {
                *(u32x4 *)(to + lv + v_step(w)) = vr[w];
            }
            if (in == 0) flags[4 * buf + b0 + BW * w] = have[w];
        }
    };

    look_up(pt.t0);                                     // on its way with Q

    half8 qh[QS], ql[F32 ? QS : 1];
    float sc = LOG2E_F / sqrtf((float)HD);
    {
        const int64_t qo = ((int64_t)row * a.H + head) * HD + 8 * h;
        if constexpr (F32) {
            float x[QS][8];
            float amax = 0.0f;
#pragma unroll
            for (int s = 0; s < QS; s++) {
                const float * src = (const float *)a.q + qo + 16 * s;
                const float4 u = *(const float4 *)src, v = *(const float4 *)(src + 4);
                const float e[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    x[s][k] = e[k];
                    amax = fmaxf(amax, fabsf(e[k]));
                }
            }
            const int ex = q_exponent(half_max(amax));
            sc = ldexpf(sc, ex);
#pragma unroll
            for (int s = 0; s < QS; s++)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    half_t hi, lo;
                    split16(ldexpf(x[s][k], -ex), hi, lo);
                    qh[s][k] = hi;
                    ql[s][k] = lo;
                }
        } else {
#pragma unroll
            for (int s = 0; s < QS; s++) qh[s] = *(const half8 *)((const half_t *)a.q + qo + 16 * s);
        }
    }

    // ---- one tile's steps
    auto read_k = [&](int buf, int c, int u) __attribute__((always_inline)) {
        return *(const half8 *)(lds + buf * (lds_t::K + lds_t::V) + (2 * c + h) * lds_t::KS + (32 * u + i) * 16);
    };
    auto read_v = [&](int buf, int d, int g) __attribute__((always_inline)) {   // (u, half of the block) = (g / 2, g % 2)
        return *(const half8 *)(lds + buf * (lds_t::K + lds_t::V) + lds_t::K +
                                (2 * (2 * (g >> 1) + h) + (g & 1)) * lds_t::VS + (32 * d + i) * 16);
    };
    // operands read ahead of their products: fewer where f32 results and f16 cells need the registers
    constexpr int KH = QS / (F32 && !F8 ? 4 : 2), VH = DT / (F32 && !F8 && DT == 4 ? 4 : 2);
    float m, l;
    float16v o[DT];
    half8 ph[4], pl[F32 ? 4 : 1];
    auto mask = [&](float16v (&s)[2], int buf, int t) __attribute__((always_inline)) {
        const int4 there = *(const int4 *)(flags + 4 * buf);
        const bool whole = min(min(there.x, there.y), min(there.z, there.w)) == 16;
        if (whole && 64 * t >= last.lo && 64 * t + 63 <= first.hi) return;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int k0 = 64 * t + 32 * u + 16 * h;
            const int n = u == 0 ? (h ? there.y : there.x) : (h ? there.w : there.z);
            const int lo = pg_clamp(me.lo - k0, 0, 16), hi = pg_clamp(min(me.hi + 1 - k0, n), 0, 16);
#pragma unroll
            for (int r = 0; r < 16; r++) s[u][r] = r >= lo && r < hi ? s[u][r] : -INFINITY;
        }
    };
    // Probabilities against the running maximum as it is (weigh); where a lane's sum of them says that one
    // may leave f16's range, or a query has no maximum yet, the maximum is taken anew and the sums are
    // brought to it (settle).  2^6 p (f32 results: 2^7 p, applied after the exponential) goes into the
    // products: small probabilities keep their bits.
    auto weigh = [&](const float16v (&s)[2], int u, int r, float mm) __attribute__((always_inline)) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[u][r], sc, mm));
        if constexpr (F32) {
            half_t hi, lo;
            split16(e * 128.0f, hi, lo);
            ph[2 * u + (r >> 3)][r & 7] = hi;
            pl[2 * u + (r >> 3)][r & 7] = lo;
        } else {
            ph[2 * u + (r >> 3)][r & 7] = (half_t)e;
        }
        return e;
    };
    auto reference = [&]() __attribute__((always_inline)) { return (F32 ? 0.0f : 6.0f) - (m == -INFINITY ? 0.0f : m); };
    auto settle = [&](const float16v (&s)[2], float sum) __attribute__((always_inline)) {
        if (__any(m == -INFINITY || sum > (F32 ? 256.0f : 16384.0f))) {
            float tm = s[0][0];
#pragma unroll
            for (int r = 0; r < 16; r++) tm = fmaxf(tm, fmaxf(s[0][r], s[1][r]));
            tm = half_max(tm) * sc;
            const float to = fmaxf(m, tm), f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= f;
            m = to;
            sum = 0.0f;
            const float mm = reference();
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) sum += weigh(s, u, r, mm);
        }
        l += sum;
    };

    if (tid < MAP_BITS / 32) map.w[tid] = 0;
    if (tid == 0) flags[8] = 0;
    while (true) {
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
        __syncthreads();
        // In registers: tile t + 1, loaded in the turn before; it goes to LDS as turn t begins, and the next
        // one is loaded.  Tiles behind the last are read as no page and not used.
        load(pt.t0);
        store(0, pt.t0);
        load(pt.t0 + 1);
        // Q is waited for here, not by the loop's first products (whose wait would be for the loads of the
        // next tile in every later turn)
#pragma unroll
        for (int c = 0; c < QS; c++) {
            asm volatile("" : "+v"(qh[c]));
            if constexpr (F32) asm volatile("" : "+v"(ql[c]));
        }
        __syncthreads();
        for (int t = pt.t0; t < pt.t1; t++) {
            const int buf = (t - pt.t0) & 1;
            store(buf ^ 1, t + 1);
            load(t + 2);
            if (!idle && 64 * t <= last.hi && 64 * t + 63 >= first.lo) {
                float16v s[2];
#pragma unroll
                for (int r = 0; r < 16; r++) s[0][r] = s[1][r] = 0.0f;
#pragma unroll
                for (int c0 = 0; c0 < QS; c0 += KH) {
                    half8 kf[KH][2];
#pragma unroll
                    for (int c = 0; c < KH; c++)
#pragma unroll
                        for (int u = 0; u < 2; u++) kf[c][u] = read_k(buf, c0 + c, u);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < KH; c++)
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            s[u] = mfma32(kf[c][u], qh[c0 + c], s[u]);
                            if constexpr (F32) s[u] = mfma32(kf[c][u], ql[c0 + c], s[u]);
                        }
                }
                mask(s, buf, t);
                const float mm = reference();
                float sum = 0.0f;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 16; r++) sum += weigh(s, u, r, mm);
                settle(s, sum);
#pragma unroll
                for (int d0 = 0; d0 < DT; d0 += VH) {
                    half8 vf[VH][4];
#pragma unroll
                    for (int d = 0; d < VH; d++)
#pragma unroll
                        for (int g = 0; g < 4; g++) vf[d][g] = read_v(buf, d0 + d, g);
#pragma unroll
                    for (int g = 0; g < 4; g++)
#pragma unroll
                        for (int d = 0; d < VH; d++) {
                            o[d0 + d] = mfma32(vf[d][g], ph[g], o[d0 + d]);
                            if constexpr (F32) o[d0 + d] = mfma32(vf[d][g], pl[g], o[d0 + d]);
                        }
                }
            }
            __syncthreads();
        }
        if (careful) break;
        // a sum that is not finite: there is such a value among the cells, or such a score
        bool odd = false;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) odd |= !(fabsf(o[d][r]) <= 3.402823466e38f);
        if (!idle && __any(odd) && lane == 0) flags[8] = 1;
        __syncthreads();
        if (!flags[8]) break;
        careful = true;
        look_up(pt.t0);
    }

    if (careful && map.any()) {
        // every wave is past the tiles (the barriers above): their room takes the sums, 32 dims at a time
        constexpr int OS = 34;
        static_assert(T * OS * 4 <= 2 * (lds_t::K + lds_t::V), "room for the sums");
        float * so = (float *)lds + (32 * wv + i) * OS;
#pragma unroll
        for (int d = 0; d < DT; d++) {
#pragma unroll
            for (int r = 0; r < 16; r++) so[8 * (r >> 2) + 4 * h + (r & 3)] = o[d][r];
#pragma unroll 1
            for (int e = 0; e < 16; e++) {
                const int dim = 8 * (e >> 2) + 4 * h + (e & 3);
                so[dim] += special_sum<HD, F8>(p, map, at.s, un.kvh, 32 * d + dim, pt.t0, pt.t1, me, keys);
            }
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] = so[8 * (r >> 2) + 4 * h + (r & 3)];
        }
    }

    // ---- results: lane's query, dims 32 d + 8 b + 4 h + 0..3 of o[d][4 b ..]
    if (idle || w0 + i > f1) return;
    l = half_sum(l);
    const int64_t rh = (int64_t)row * a.H + head;
    const float mul = l == 0.0f ? 0.0f : (F32 ? 1.0f / 128.0f : 1.0f) / l;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
            const int dim = 32 * d + 8 * b + 4 * h;
            const float4v v = {o[d][4 * b] * mul, o[d][4 * b + 1] * mul, o[d][4 * b + 2] * mul, o[d][4 * b + 3] * mul};
            if constexpr (F32) *(float4v *)((float *)a.out + rh * HD + dim) = v;
            else *(half4 *)((half_t *)a.out + rh * HD + dim) =
                    half4{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
        }
}

// ---------------------------------------------------------------------------
// Joining the parts of a split range
// ---------------------------------------------------------------------------
// o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  W waves per (row, head): half a wave reads a part's
// sums, HD / 32 dims a lane, so W waves take 2 W parts at a time, all that there may be (ALL of them per
// half wave) before any is known to be needed: one round of loads.  The sums are added in a fixed
// order: the same bits on every run.  28 rows and heads of 64 parts (0.9 MB): 3.9 us, a launch and two
// dependent loads.
template <int HD, bool F32, int W, int ALL>
__global__ void __launch_bounds__(256) k_paged_join(paged_t p, attn_t a) {
    constexpr int DL = HD / 32;                                 // dims per lane
    __shared__ float sv[4][HD];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, half = lane >> 5, w = wv % W;
    const int64_t rows = (int64_t)p.n_rows * a.H, rh = (int64_t)blockIdx.x * (4 / W) + wv / W;
    if (W < 4 && rh >= rows) return;                            // W = 4: the grid is the rows
    // rows of no sequence have no parts; the others' number was written with their first part
    const int row = (int)(rh / a.H);
    const bool in = row >= p.rows[0] && row < p.rows[p.n_seqs];
    const int n = a.n_parts[rh];
    float mi[ALL], v[ALL][DL];
    const float * src = a.part_o + rh * HD + DL * (lane & 31);
#pragma unroll
    for (int i = 0; i < ALL; i++) {
        const int64_t at = (int64_t)min(2 * (w + W * i) + half, a.parts - 1) * rows;
        mi[i] = a.part_ml[2 * (at + rh)];
#pragma unroll
        for (int k = 0; k < DL; k++) v[i][k] = src[at * HD + k];
    }
    float m_l = -INFINITY, l_l = 0.0f;                          // lane's part of the row's maximum and sum
    if (lane < a.parts) {
        m_l = a.part_ml[2 * (lane * rows + rh)];
        l_l = a.part_ml[2 * (lane * rows + rh) + 1];
    }
    const int parts = in ? min(n, a.parts) : 1;
    if (parts <= 1) return;                                     // the same for the output's W waves
    const float mx = wave_max(lane < parts ? m_l : -INFINITY);
    float sum = lane < parts ? (m_l == -INFINITY ? l_l : __builtin_amdgcn_exp2f(m_l - mx) * l_l) : 0.0f;
    sum = wave_sum(sum);
    float t[DL] = {};
#pragma unroll
    for (int i = 0; i < ALL; i++) {
        // held above 0: an infinite sum stays one; a part that saw nothing has zeros, or NaN
        const float r = mi[i] == -INFINITY ? 1.0f : fmaxf(__builtin_amdgcn_exp2f(mi[i] - mx), 0x1p-126f);
        const bool is = 2 * (w + W * i) + half < parts;
#pragma unroll
        for (int k = 0; k < DL; k++) t[k] = is ? fmaf(r, v[i][k], t[k]) : t[k];
    }
#pragma unroll
    for (int k = 0; k < DL; k++) t[k] += __shfl_xor(t[k], 32, WAVE);
    if constexpr (W > 1) {
        if (half == 0)
#pragma unroll
            for (int k = 0; k < DL; k++) sv[wv][DL * lane + k] = t[k];
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int k = 0; k < DL; k++) {
            t[k] = 0.0f;
#pragma unroll
            for (int j = 0; j < W; j++) t[k] += sv[wv + j][DL * (lane & 31) + k];
        }
    }
    if (half) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int k = 0; k < DL; k++) {
        const int64_t o = rh * HD + DL * lane + k;
        if constexpr (F32) ((float *)a.out)[o] = t[k] * inv;
        else ((half_t *)a.out)[o] = (half_t)(t[k] * inv);
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// T: queries per workgroup; 16 is k_paged_few, 32 k_paged_mid, 128 k_paged_many.
// most: parts that the workspace has room for, whatever the window (fewer key tiles, no more parts).
struct attn_plan { int T, tiles, chunk, parts, most; };
// A range is split where a query tile has more than WHOLE key tiles and the workgroups are few: the join
// costs a launch (12 tiles, 32 heads: 1 row in 8 sequences 16.1 us whole, 18.2 in two parts, 128 rows 15.1 /
// 19.7; 55 tiles, 4 KV heads, 2 rows: 14.9 in 4 parts, 10.0 in 14).
#define WHOLE 16
#define MIN_CHUNK 4    // key tiles of a part: one per wave
#define MAX_PARTS 64   // a lane each in the join
static attn_plan plan_of(const paged_t & p, int H, int64_t max_keys, int window, bool split) {
    const int G = H / p.Hkv;
    const int64_t queries = (int64_t)p.n_rows * G, seqs = std::min<int64_t>(p.n_seqs, p.n_rows), all = queries * p.Hkv;
    attn_plan r;
    // The narrow tiles read the keys more often but come in more workgroups, four waves to a range of keys:
    // they are taken up to two (16 queries) and four (32) workgroups per CU, or where no sequence fills more.
    // 16 / 32 / 128 queries, us: 4 x 64 rows of 32 heads over 764 f16 keys 26 / 31 / 41, 4 x 128 rows 52 / 35 /
    // 52, 4 x 512 rows 236 / 160 / 115; 32 rows of 28 heads over 3532 keys 16.3 / 15.6 / 26, 512 rows 85 / 57 / 58,
    // 1024 rows 144 / 109 / 100; 8 x 32 rows of 32 heads over 732 keys 17 / 27 / 31, 8 x 256 101 / 85 / 57.
    r.T = queries <= 16 * seqs || all <= 512 * 16 ? FEW_T : queries <= 32 * seqs || all <= 1024 * 32 ? MID_T : MANY_T;
    r.tiles = (int)(queries / r.T + seqs);
    const int64_t units = (int64_t)p.Hkv * std::max<int64_t>(seqs, queries / r.T);
    // Parts of kt key tiles: as many as make 512 workgroups, and where the parts still have 16 tiles up to 2048,
    // as a batch's ranges are seldom equal (32 sequences of 17 to 4000 keys, 32 heads: 64.5 us whole, 55 in two
    // parts; 96 such of 4 KV heads 33.6 / 27.6 in three; 16 of 2000 61.3 / 57.2; 96 equal ones of 2000, 4 KV
    // heads, lose: 42.2 / 45.8; 64 of 32 heads, 2048 workgroups, stay whole: 69.8 / 76.7).  32 and 128 queries
    // come in more than 256 workgroups (8192 / 32, 32768 / 128): their ranges stay whole.
    const auto want = [&](int64_t kt) {
        const int64_t n = std::max<int64_t>(512 / units, std::min<int64_t>(kt / WHOLE, 2048 / units));
        return r.T == FEW_T ? std::min<int64_t>(MAX_PARTS, std::max<int64_t>(1, n)) : 1;
    };
    // key tiles that a query tile can see
    int64_t kt = (std::min<int64_t>(std::max<int64_t>(max_keys, 1), p.cap) + 63) / 64;
    r.most = kt <= WHOLE ? 1 : (int)std::min<int64_t>(want(kt), (kt + MIN_CHUNK - 1) / MIN_CHUNK);
    if (window > 0) kt = std::min<int64_t>(kt, ((int64_t)window + r.T / G + 63) / 64 + 1);
    r.chunk = (int)std::max<int64_t>(MIN_CHUNK, (kt + want(kt) - 1) / want(kt));
    r.parts = split && kt > WHOLE ? (int)((kt + r.chunk - 1) / r.chunk) : 1;
    return r;
}

// More than 64 KB of LDS needs the kernel's limit raised, once per device (`set`: a bit per device).
static int many_lds_limit(const void * kernel, int bytes, std::atomic<uint64_t> & set) {
    if (bytes <= 64 * 1024) return DFX_OK;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    if (set.load(std::memory_order_acquire) >> dev & 1) return DFX_OK;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) {
        dfx_set_error("dfx_paged_attention: %d bytes of LDS: %s", bytes, hipGetErrorString(e));
        return DFX_ERR_HIP;
    }
    set.fetch_or(1ull << dev, std::memory_order_release);
    return DFX_OK;
}

template <int HD, bool F8, bool F32>
static int many_launch(const paged_t & p, const attn_t & a, dim3 grid, hipStream_t st) {
    static std::atomic<uint64_t> set;
    constexpr int bytes = many_lds<HD>::BYTES;
    const int rc = many_lds_limit((const void *)k_paged_many<HD, F8, F32>, bytes, set);
    if (rc != DFX_OK) return rc;
    hipLaunchKernelGGL((k_paged_many<HD, F8, F32>), grid, dim3(64 * MANY_WAVES), bytes, st, p, a);
    return DFX_OK;
}

template <int HD, bool F8, bool F32>
static int attn_launch(const paged_t & p, const attn_t & a, const attn_plan & pl, hipStream_t st) {
    const dim3 grid(unit_grid(p.Hkv, pl.tiles), (unsigned)pl.parts);
    int rc = DFX_OK;
    if (pl.T == FEW_T) hipLaunchKernelGGL((k_paged_few<HD, F8, F32>), grid, dim3(256), 0, st, p, a);
    else if (pl.T == MID_T) {
        static std::atomic<uint64_t> set;
        constexpr int bytes = 4 * MID_T * (HD + 4) * (int)sizeof(float);
        static_assert(bytes >= (HD / 16) * 2 * 64 * (int)sizeof(half8), "room for Q's terms");
        rc = many_lds_limit((const void *)k_paged_mid<HD, F8, F32>, bytes, set);
        if (rc == DFX_OK) hipLaunchKernelGGL((k_paged_mid<HD, F8, F32>), grid, dim3(256), bytes, st, p, a);
    }
    else rc = many_launch<HD, F8, F32>(p, a, grid, st);
    if (rc != DFX_OK) return rc;
    DFX_CHECK_LAUNCH("dfx_paged_attention");
    if (pl.parts > 1) {
        const int64_t rows = (int64_t)p.n_rows * a.H;
        if (pl.parts <= 8)
            hipLaunchKernelGGL((k_paged_join<HD, F32, 1, 4>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p, a);
        else if (pl.parts <= 32)
            hipLaunchKernelGGL((k_paged_join<HD, F32, 4, 4>), dim3((unsigned)rows), dim3(256), 0, st, p, a);
        else
            hipLaunchKernelGGL((k_paged_join<HD, F32, 4, MAX_PARTS / 8>), dim3((unsigned)rows), dim3(256), 0, st, p, a);
        DFX_CHECK_LAUNCH("dfx_paged_attention (join)");
    }
    return DFX_OK;
}

extern "C" size_t dfx_paged_attention_ws_bytes(const dfx_paged_cache * cache, const dfx_paged_batch * batch, int n_head,
                                               int type) {
    paged_t p;
    (void)type;
    if (paged_of("dfx_paged_attention_ws_bytes", cache, batch, n_head, &p) != DFX_OK) return 0;
    if (p.n_rows == 0 || p.n_seqs == 0) return 0;
    const attn_plan pl = plan_of(p, n_head, batch->max_keys, 0, true);
    return pl.most <= 1 ? 0 : ((size_t)pl.most * (cache->head_dim + 2) + 1) * p.n_rows * n_head * sizeof(float);
}

extern "C" int dfx_paged_attention(const dfx_paged_cache * cache, const dfx_paged_batch * batch, const void * q, int type,
                                   int n_head, int causal, int window, void * out, void * ws, void * stream) {
    paged_t p;
    const int rc = paged_of("dfx_paged_attention", cache, batch, n_head, &p);
    if (rc != DFX_OK) return rc;
    if (type != DFX_TYPE_F16 && type != DFX_TYPE_F32) {
        dfx_set_error("dfx_paged_attention: type %d (DFX_TYPE_F16 or DFX_TYPE_F32)", type);
        return DFX_ERR_UNSUPPORTED;
    }
    if (window < 0 || (window > 0 && !causal)) {
        dfx_set_error("dfx_paged_attention: window=%d causal=%d (a window needs the causal mask)", window, causal);
        return DFX_ERR_ARG;
    }
    if (p.n_rows == 0 || p.n_seqs == 0) return DFX_OK;
    auto a16 = [](const void * x) { return ((uintptr_t)x & 15) == 0; };
    if (!q || !out || !a16(q) || !a16(out) || !a16(ws)) {
        dfx_set_error("dfx_paged_attention: q or out missing, or q, out or ws not aligned to 16 bytes");
        return DFX_ERR_ARG;
    }
    const int hd = cache->head_dim;
    const attn_plan pl = plan_of(p, n_head, batch->max_keys, window, ws != nullptr);
    attn_t a = {q,      out,      (float *)ws, nullptr, nullptr, n_head, n_head / p.Hkv, causal ? 1 : 0, window, pl.chunk,
                pl.parts, pl.tiles};
    a.part_ml = a.part_o + (size_t)pl.parts * p.n_rows * n_head * hd;
    a.n_parts = (int32_t *)(a.part_ml + (size_t)pl.parts * p.n_rows * n_head * 2);
    hipStream_t st = (hipStream_t)stream;
    const bool f8 = cache->type == DFX_TYPE_F8, f32 = type == DFX_TYPE_F32;
    const auto launch = hd == 128 ? (f8 ? (f32 ? attn_launch<128, true, true> : attn_launch<128, true, false>)
                                        : (f32 ? attn_launch<128, false, true> : attn_launch<128, false, false>))
                                  : (f8 ? (f32 ? attn_launch<64, true, true> : attn_launch<64, true, false>)
                                        : (f32 ? attn_launch<64, false, true> : attn_launch<64, false, false>));
    return launch(p, a, pl, st);
}
