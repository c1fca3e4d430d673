// k_paged.hip — rotation and append to a paged key / value cache, for ragged batches.
//
// The unit of the cache is a block of 16 tokens of one KV head: keys [16][hd], values transposed
// [hd][16], so that a value column's 16 tokens are consecutive for the attention's P V products,
// and in 8 bits one power of two per side.  A wave owns a block of one head and side from the row
// that enters it (the sequence's first row of the call, or a position divisible by 16) to the last
// row that falls into it: one largest magnitude, one scale, no atomics.
#include "dfx_device.h"
#include "dfx_pages.h"

#include <algorithm>

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------------------
// Rows to sequences
// ---------------------------------------------------------------------------

// Last sequence s with rows[s] <= m (rows not decreasing: the one that holds row m, if any does),
// or -1.  The wave's lanes probe 64 sequences at a time: one load for up to 64 sequences.
__device__ __forceinline__ int wave_find_seq(const paged_t & p, int m) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = p.n_seqs;
    while (true) {
        const int step = (len + 63) >> 6;
        const int i = lane * step;
        const bool le = i < len && p.rows[lo + i] <= m;
        const int k = __popcll(__ballot(le));
        if (k == 0) return -1;
        lo += (k - 1) * step;
        if (step == 1) return lo;
        len = min(step, len - (k - 1) * step);
    }
}

struct row_place { int s, pos, r0, r1; };   // s < 0: the row belongs to no sequence

// Lane j < N (N a power of two) gets the place of row m0 + j; the lanes above repeat them.  Decoding
// batches have a sequence per row, prompts one for all rows.
template <int N> __device__ __forceinline__ row_place wave_places(const paged_t & p, int m0) {
    const int lane = threadIdx.x & 63;
    row_place mine = {-1, 0, 0, 0};
    for (int base = max(wave_find_seq(p, m0), 0); base < p.n_seqs; base += 64) {
        seq_t q = {0, 0, 0};
        if (base + lane < p.n_seqs) q = pg_seq(p, base + lane);
        const int r1 = q.r0 + q.n;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int m = m0 + j;
            const uint64_t has = __ballot(q.r0 <= m && m < r1);
            if (has) {
                const int from = __ffsll((unsigned long long)has) - 1;
                const int a = __builtin_amdgcn_readlane(q.r0, from), b = __builtin_amdgcn_readlane(r1, from);
                const int k = __builtin_amdgcn_readlane(q.keys, from);
                if ((lane & (N - 1)) == j && mine.s < 0) mine = {base + from, k - (b - m), a, b};
            }
        }
        // rows up to the last of these sequences are placed; the next ones may begin behind the tile
        if (__builtin_amdgcn_readlane(r1, 63) >= min(m0 + N, p.n_rows)) break;
        if (base + 64 < p.n_seqs && p.rows[base + 64] >= m0 + N) break;
    }
    return mine;
}

// ---------------------------------------------------------------------------
// E4M3 cells
// ---------------------------------------------------------------------------

// 2^k, the least power of two with a <= 448 * 2^k, k in -15..7 (448 = 1.75 * 2^8).
__device__ __forceinline__ float f8_scale(float a) {
    const uint32_t b = __float_as_uint(a);
    int k = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    k = min(max(k, -15), 7);
    return __uint_as_float((uint32_t)(k + 127) << 23);
}
// whether s is a scale that f8_scale gives
__device__ __forceinline__ bool f8_scale_ok(float s) {
    return s >= 0x1p-15f && s <= 0x1p7f && (__float_as_uint(s) & 0x7fffffu) == 0;
}
__device__ __forceinline__ float f8_finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}
// x * inv held within +-448; what is not finite becomes NaN.  Rounded to nearest even by the
// conversion, half a step (2^-4 of the value) at most.
__device__ __forceinline__ float f8_ready(float x, float inv) {
    const float y = fminf(fmaxf(x * inv, -448.0f), 448.0f);
    return fabsf(x) <= 3.402823466e38f ? y : __builtin_nanf("");
}
__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return (uint32_t)r;
}
// four cells brought to another scale: cell * ratio (ratio a power of two <= 1)
__device__ __forceinline__ uint32_t f8_rescale4(uint32_t w, float ratio) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return f8_pack4(a.x * ratio, a.y * ratio, b.x * ratio, b.y * ratio);
}

struct f8_choice { float scale, ratio; };   // ratio: what kept cells are multiplied by (1: left alone)
__device__ __forceinline__ f8_choice f8_choose(float amax, bool kept, float old) {
    const float s = f8_scale(amax);
    if (!kept || !f8_scale_ok(old) || old == s) return {s, 1.0f};
    return old > s ? f8_choice{old, 1.0f} : f8_choice{s, old / s};
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// Waves: first the cells, one wave per (RT rows, KV head, side), each taking the blocks whose first
// row of the call is among its RT rows; then Q, one wave per (rows of one pass, QHEADS heads), whose
// angles are read once (3539 rows of 28 heads: 34.6 us read for each, 26.9 so).  RT = 1 where the rows
// belong to many sequences (each row enters a block of its own, and one wave per row keeps its chain
// of dependent loads - places, page, scale, kept cells - alone on it), 16 otherwise.
// Bound by bytes for prompts, by that chain and the launch for steps.  Measured, heads of 128: 3539 rows of
// 28 + 4 + 4 heads with f32 Q into E4M3 (120 MB) 26.5 us, 4.5 TB/s (5.1 in a copy); 3583 rows of 32 + 32 +
// 32 heads into f16 (264 MB) 57.9 us, 4.6 TB/s; one row of 64 sequences of 32 + 32 + 32 heads (4.2 MB) 7.1
// us; one row 3.8 us.
#define APPEND_WAVES 4
#define QHEADS 4

// (cos, sin) and the two halves of four pairs of a row
struct rope4 {
    float4 a, b, c01, c23;
    __device__ __forceinline__ void load_x(const float * src, int half) {
        a = *(const float4 *)src;
        b = *(const float4 *)(src + half);
    }
    __device__ __forceinline__ void load_angles(const float * cs) {
        c01 = *(const float4 *)cs;
        c23 = *(const float4 *)(cs + 4);
    }
    __device__ __forceinline__ void load(const float * src, const float * cs, int half) {
        load_x(src, half);
        load_angles(cs);
    }
    // a, b = the rotated halves
    __device__ __forceinline__ void turn() {
#pragma clang fp contract(off)
        const float4 x = a, y = b;
        a = make_float4(x.x * c01.x - y.x * c01.y, x.y * c01.z - y.y * c01.w, x.z * c23.x - y.z * c23.y,
                        x.w * c23.z - y.w * c23.w);
        b = make_float4(x.x * c01.y + y.x * c01.x, x.y * c01.w + y.y * c01.z, x.z * c23.y + y.z * c23.x,
                        x.w * c23.w + y.w * c23.z);
    }
};
__device__ __forceinline__ half4 to_half4(float4 x) {
    return half4{(half_t)x.x, (half_t)x.y, (half_t)x.z, (half_t)x.w};
}
__device__ __forceinline__ float f8_max4(float m, float4 x) {
    return fmaxf(m, fmaxf(fmaxf(f8_finite_abs(x.x), f8_finite_abs(x.y)), fmaxf(f8_finite_abs(x.z), f8_finite_abs(x.w))));
}
__device__ __forceinline__ uint32_t f8_cells4(float4 x, float inv) {
    return f8_pack4(f8_ready(x.x, inv), f8_ready(x.y, inv), f8_ready(x.z, inv), f8_ready(x.w, inv));
}

template <int HD, bool F8, bool QF32>
__global__ void __launch_bounds__(64 * APPEND_WAVES, 3) k_paged_append(paged_t p, const float * __restrict__ qkv, int H,
                                                                    const float * __restrict__ tab, int n_pos,
                                                                    void * __restrict__ q_out, int RT, int n_cell_waves,
                                                                    int n_waves) {
    constexpr int HALF = HD / 2;
    constexpr int CELL = F8 ? 1 : 2;
    // one head's 16 values per dimension, transposed, per wave
    __shared__ __attribute__((aligned(16))) uint8_t vt_all[APPEND_WAVES][HD * 16 * CELL];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int w = blockIdx.x * APPEND_WAVES + wv;
    if (w >= n_waves) return;
    const int Hkv = p.Hkv;
    const int64_t ld = (int64_t)(H + 2 * Hkv) * HD;
    const int limit = min(p.cap, n_pos);                 // positions that can be written

    constexpr int LPR = HALF / 4;                        // lanes per rotated row, four pairs each
    constexpr int RPP = 64 / LPR;                        // rows per pass of the wave
    const int lr = lane / LPR, j4 = 4 * (lane % LPR);

    if (w >= n_cell_waves) {                             // ---- Q: RPP rows of QHEADS heads
        const int groups = (H + QHEADS - 1) / QHEADS;
        const int u = w - n_cell_waves, h0 = (u % groups) * QHEADS, m0 = (u / groups) * RPP, m = m0 + lr;
        rope4 x[QHEADS];
        const float * src = qkv + min(m, p.n_rows - 1) * ld + (int64_t)h0 * HD + j4;    // clamped: not stored
#pragma unroll
        for (int k = 0; k < QHEADS; k++) x[k].load_x(src + (int64_t)min(k, H - 1 - h0) * HD, HALF);
        const row_place at = wave_places<RPP>(p, m0);
        const int s = __shfl(at.s, lr, WAVE), pos = __shfl(at.pos, lr, WAVE);
        if (s < 0 || pos < 0 || pos >= n_pos) return;
        x[0].load_angles(tab + ((int64_t)pos * HALF + j4) * 2);
#pragma unroll
        for (int k = 0; k < QHEADS; k++) {
            if (h0 + k >= H) break;
            x[k].c01 = x[0].c01;
            x[k].c23 = x[0].c23;
            x[k].turn();
            const int64_t o = ((int64_t)m * H + h0 + k) * HD + j4;
            if constexpr (QF32) {
                float * dst = (float *)q_out + o;
                *(float4 *)dst = x[k].a;
                *(float4 *)(dst + HALF) = x[k].b;
            } else {
                half_t * dst = (half_t *)q_out + o;
                *(half4 *)dst = to_half4(x[k].a);
                *(half4 *)(dst + HALF) = to_half4(x[k].b);
            }
        }
        return;
    }

    // ---- cells: RT rows of one head and side
    const int unit = w % (2 * Hkv), kvh = unit >> 1, side = unit & 1, m0 = (w / (2 * Hkv)) * RT;
    // one row: its line is on its way while its place is looked up
    float warm = 0.0f;
    if (RT == 1 && lane < HD / 16) warm = qkv[m0 * ld + (int64_t)(H + side * Hkv + kvh) * HD + 16 * lane];
    const row_place at = RT == 1 ? wave_places<1>(p, m0) : wave_places<16>(p, m0);
    const bool enters = lane < RT && at.s >= 0 && at.pos >= 0 && at.pos < limit &&
                        ((at.pos & 15) == 0 || m0 + lane == at.r0);
    for (uint64_t todo = __ballot(enters); todo; todo &= todo - 1) {
        const int j = __ffsll((unsigned long long)todo) - 1, m = m0 + j;
        const int s = __shfl(at.s, j, WAVE), pos = __shfl(at.pos, j, WAVE), r1 = __shfl(at.r1, j, WAVE);
        const int t0 = pos & 15;                                            // first new token of the block
        const int cnt = min(min(r1 - m, 16 - t0), limit - pos);             // new tokens t0 .. t0 + cnt - 1
        const int64_t blk = pg_block(p, s, kvh, pos);
        if (blk < 0) continue;
        asm volatile("" : : "v"(warm));
        float old = 0.0f;
        if constexpr (F8) old = p.scale[2 * blk + side];
        if (side == 0) {
            // keys: rotated, cells [16][HD]
            constexpr int NP = 16 / RPP;
            float amax = 0.0f;
            const float * src = qkv + (int64_t)(H + kvh) * HD + j4;
            rope4 x[NP];
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (i * RPP >= cnt) break;
                const int r = min(i * RPP + lr, cnt - 1);                   // clamped: not stored
                x[i].load(src + (m + r) * ld, tab + ((int64_t)(pos + r) * HALF + j4) * 2, HALF);
            }
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (i * RPP >= cnt) break;
                x[i].turn();
                amax = f8_max4(f8_max4(amax, x[i].a), x[i].b);
            }
            if constexpr (F8) {
                const f8_choice c = f8_choose(wave_max(amax), t0 > 0, old);
                const float inv = 1.0f / c.scale;
                uint8_t * cell = (uint8_t *)p.k + blk * (16 * HD);
                if (c.ratio != 1.0f)
                    for (int o = 16 * lane; o < t0 * HD; o += 16 * 64) {
                        u32x4 v = *(const u32x4 *)(cell + o);
#pragma unroll
                        for (int k = 0; k < 4; k++) v[k] = f8_rescale4(v[k], c.ratio);
                        *(u32x4 *)(cell + o) = v;
                    }
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const int r = i * RPP + lr;
                    if (r >= cnt) break;
                    uint8_t * dst = cell + (t0 + r) * HD + j4;
                    *(uint32_t *)dst = f8_cells4(x[i].a, inv);
                    *(uint32_t *)(dst + HALF) = f8_cells4(x[i].b, inv);
                }
                if (lane == 0) p.scale[2 * blk] = c.scale;
            } else {
                half_t * cell = (half_t *)p.k + blk * (16 * HD);
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const int r = i * RPP + lr;
                    if (r >= cnt) break;
                    half_t * dst = cell + (t0 + r) * HD + j4;
                    *(half4 *)dst = to_half4(x[i].a);
                    *(half4 *)(dst + HALF) = to_half4(x[i].b);
                }
            }
        } else {
            // values: cells [HD][16], transposed through LDS
            constexpr int LV = HD / 4, RV = 64 / LV, NP = 16 / RV;
            const int vr = lane / LV, d4 = 4 * (lane % LV);
            const float * src = qkv + (int64_t)(H + Hkv + kvh) * HD + d4;
            float4 x[NP];
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (i * RV >= cnt) break;
                x[i] = *(const float4 *)(src + (m + min(i * RV + vr, cnt - 1)) * ld);
            }
#pragma unroll
            for (int i = 0; i < NP; i++) {
                if (i * RV >= cnt) break;
                amax = f8_max4(amax, x[i]);
            }
            f8_choice c = {1.0f, 1.0f};
            if constexpr (F8) c = f8_choose(wave_max(amax), t0 > 0, old);
            const float inv = 1.0f / c.scale;
            if (cnt == 1 && c.ratio == 1.0f) {
                // one token, the kept ones as they are: its cells alone are written, none read
                if (vr == 0) {
                    uint8_t * cell = (uint8_t *)p.v + (blk * (16 * HD) + d4 * 16 + t0) * CELL;
                    const float e[4] = {x[0].x, x[0].y, x[0].z, x[0].w};
                    if constexpr (F8) {
                        const uint32_t q = f8_cells4(x[0], inv);
#pragma unroll
                        for (int k = 0; k < 4; k++) cell[16 * k] = (uint8_t)(q >> (8 * k));
                        if (lane == 0) p.scale[2 * blk + 1] = c.scale;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; k++) ((uint16_t *)cell)[16 * k] = f2h(e[k]);
                    }
                }
                continue;
            }
            uint8_t * vt = vt_all[wv];
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int r = i * RV + vr;
                if (r >= cnt) break;
                const float e[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                if constexpr (F8) {
                    const uint32_t q = f8_cells4(x[i], inv);
#pragma unroll
                    for (int k = 0; k < 4; k++) vt[(d4 + k) * 16 + t0 + r] = (uint8_t)(q >> (8 * k));
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) ((uint16_t *)vt)[(d4 + k) * 16 + t0 + r] = f2h(e[k]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            // whole columns of 16 tokens are stored; a partly written block keeps its other tokens
            constexpr int WORDS = 4 * CELL, PER = 4 / CELL;                 // 32-bit words per column, tokens per word
            uint32_t * cell = (uint32_t *)((uint8_t *)p.v + blk * (16 * HD * CELL));
#pragma unroll
            for (int d0 = 0; d0 < HD; d0 += 64) {
                const int d = d0 + lane;
                u32x4 nw[CELL], ow[CELL];
#pragma unroll
                for (int k = 0; k < CELL; k++) nw[k] = *(const u32x4 *)(vt + d * 16 * CELL + 16 * k);
                if (cnt < 16) {
#pragma unroll
                    for (int k = 0; k < CELL; k++) ow[k] = *(const u32x4 *)(cell + d * WORDS + 4 * k);
#pragma unroll
                    for (int i = 0; i < WORDS; i++) {
                        uint32_t keep = 0, kept = 0;                        // bits of tokens not new, and before those
#pragma unroll
                        for (int e = 0; e < PER; e++) {
                            const int t = i * PER + e;
                            const uint32_t bits = (F8 ? 0xffu : 0xffffu) << (e * 8 * CELL);
                            if (t < t0) kept |= bits;
                            if (t < t0 || t >= t0 + cnt) keep |= bits;
                        }
                        uint32_t o = ow[i / 4][i % 4];
                        if constexpr (F8)
                            if (c.ratio != 1.0f) o = (f8_rescale4(o, c.ratio) & kept) | (o & ~kept);
                        nw[i / 4][i % 4] = (o & keep) | (nw[i / 4][i % 4] & ~keep);
                    }
                }
#pragma unroll
                for (int k = 0; k < CELL; k++) *(u32x4 *)(cell + d * WORDS + 4 * k) = nw[k];
            }
            if constexpr (F8)
                if (lane == 0) p.scale[2 * blk + 1] = c.scale;
            __builtin_amdgcn_wave_barrier();                                // vt is written again for the next block
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static bool aligned(const void * ptr, uintptr_t to) { return ((uintptr_t)ptr & (to - 1)) == 0; }

// Rows times heads of one call: what a grid of 256-thread workgroups holds in one dimension, halved.
#define MAX_ROW_HEADS (1 << 23)
#define MAX_POSITIONS (1 << 30)   // of a sequence: positions a few tiles further are 32-bit integers

// The kernel form of a cache and a batch; a status and message where they are not sound.
int paged_of(const char * who, const dfx_paged_cache * c, const dfx_paged_batch * b, int n_head, paged_t * out) {
    if (!c || !b) {
        dfx_set_error("%s: no cache or no batch", who);
        return DFX_ERR_ARG;
    }
    if (c->type != DFX_TYPE_F16 && c->type != DFX_TYPE_F8) {
        dfx_set_error("%s: cache type %d (DFX_TYPE_F16 or DFX_TYPE_F8)", who, c->type);
        return DFX_ERR_UNSUPPORTED;
    }
    if (c->head_dim != 64 && c->head_dim != 128) {
        dfx_set_error("%s: head size %d (64 or 128 supported)", who, c->head_dim);
        return DFX_ERR_UNSUPPORTED;
    }
    int shift = 4;
    while (shift < 8 && (1 << shift) < c->page_size) shift++;
    if ((1 << shift) != c->page_size) {
        dfx_set_error("%s: pages of %d tokens (16, 32, 64, 128 or 256)", who, c->page_size);
        return DFX_ERR_UNSUPPORTED;
    }
    if (c->n_head_kv <= 0 || n_head <= 0 || n_head % c->n_head_kv || n_head > 4096 || c->n_pages <= 0 ||
        c->n_pages > INT32_MAX) {
        dfx_set_error("%s: bad shape H=%d Hkv=%d pages=%lld", who, n_head, c->n_head_kv, (long long)c->n_pages);
        return DFX_ERR_ARG;
    }
    if (!c->k || !c->v || (c->type == DFX_TYPE_F8 && !c->scale) || !aligned(c->k, 16) || !aligned(c->v, 16) ||
        !aligned(c->scale, 8)) {
        dfx_set_error("%s: cache buffers missing or not aligned (k, v: 16 bytes; scale: 8)", who);
        return DFX_ERR_ARG;
    }
    if (b->n_seqs < 0 || b->n_rows < 0 || b->max_keys < 0 || (int64_t)b->n_rows * n_head > MAX_ROW_HEADS) {
        dfx_set_error("%s: bad batch seqs=%d rows=%d max_keys=%lld H=%d (rows times heads: at most %d)", who, b->n_seqs,
                      b->n_rows, (long long)b->max_keys, n_head, MAX_ROW_HEADS);
        return DFX_ERR_ARG;
    }
    if (b->n_seqs > 0 && b->n_rows > 0 && (!b->rows || !b->n_keys || !b->pages || b->ld_pages <= 0)) {
        dfx_set_error("%s: batch without row offsets, key counts or page ids", who);
        return DFX_ERR_ARG;
    }
    const int64_t cap = std::min<int64_t>(b->ld_pages, MAX_POSITIONS >> shift) << shift;
    *out = {c->k, c->v, c->scale, b->rows, b->n_keys, b->pages, b->ld_pages, (int32_t)c->n_pages, shift, (int32_t)cap,
            c->n_head_kv, b->n_seqs, b->n_rows};
    return DFX_OK;
}

extern "C" int dfx_paged_append(const dfx_paged_cache * cache, const dfx_paged_batch * batch, const float * qkv,
                                int n_head, const float * tab, int64_t n_pos, int q_type, void * q_out,
                                void * stream) {
    paged_t p;
    const int rc = paged_of("dfx_paged_append", cache, batch, n_head, &p);
    if (rc != DFX_OK) return rc;
    if (q_type != DFX_TYPE_F16 && q_type != DFX_TYPE_F32) {
        dfx_set_error("dfx_paged_append: query type %d (DFX_TYPE_F16 or DFX_TYPE_F32)", q_type);
        return DFX_ERR_UNSUPPORTED;
    }
    if (p.n_rows == 0 || p.n_seqs == 0) return DFX_OK;
    if (!qkv || !tab || !q_out || n_pos <= 0 || !aligned(qkv, 16) || !aligned(tab, 16) || !aligned(q_out, 16)) {
        dfx_set_error("dfx_paged_append: qkv, tab or q_out missing or not aligned to 16 bytes, or n_pos=%lld",
                      (long long)n_pos);
        return DFX_ERR_ARG;
    }
    const int RT = (int64_t)p.n_seqs * 8 > p.n_rows ? 1 : 16;
    const int64_t cell_waves = ((int64_t)(p.n_rows + RT - 1) / RT) * 2 * p.Hkv;
    const int q_rows = 64 / (cache->head_dim / 8);              // rows of a wave's pass
    const int64_t waves = cell_waves + (int64_t)((p.n_rows + q_rows - 1) / q_rows) * ((n_head + QHEADS - 1) / QHEADS);
    const int np = (int)(n_pos < INT32_MAX ? n_pos : INT32_MAX);
    const dim3 grid((unsigned)((waves + APPEND_WAVES - 1) / APPEND_WAVES)), wg(64 * APPEND_WAVES);
#define APPEND(HD, F8, QF32)                                                                                          \
    hipLaunchKernelGGL((k_paged_append<HD, F8, QF32>), grid, wg, 0, (hipStream_t)stream, p, qkv, n_head, tab, np,      \
                       q_out, RT, (int)cell_waves, (int)waves)
#define APPEND_T(HD)                                                                                                  \
    do {                                                                                                              \
        if (cache->type == DFX_TYPE_F8) {                                                                             \
            if (q_type == DFX_TYPE_F32) APPEND(HD, true, true);                                                       \
            else APPEND(HD, true, false);                                                                             \
        } else {                                                                                                      \
            if (q_type == DFX_TYPE_F32) APPEND(HD, false, true);                                                      \
            else APPEND(HD, false, false);                                                                            \
        }                                                                                                             \
    } while (0)
    if (cache->head_dim == 128) APPEND_T(128);
    else APPEND_T(64);
#undef APPEND_T
#undef APPEND
    DFX_CHECK_LAUNCH("dfx_paged_append");
    return DFX_OK;
}
