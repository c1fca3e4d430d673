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

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

#define LOG2E_F 1.44269504088896341f

// eight cells as f16
__device__ __forceinline__ half8 f8_half8(uint32_t w0, uint32_t w1, float scale) {
    const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, false);
    const half2v b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, scale, true);
    const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, false);
    const half2v d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, scale, true);
    return half8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
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

// An f32 value as two f16 terms (the second rounded: 2^-23 of the value where it is f16-normal).
__device__ __forceinline__ void split16(float x, half_t & hi, half_t & lo) {
    hi = (half_t)x;
    lo = (half_t)(x - (float)hi);
}

// NaN and infinities among the values.  A query that does not see a key has probability 0 for it, and
// 0 times such a value is NaN; a probability that is 0 in f16, or the second term of a split one (0 or
// negative), makes NaN of an infinite value that is seen.  So where a tile has such values and needs it
// (NaN alone, seen by all, is right as it is), they are taken out (0 in their place), and a second
// product of marks (NaN 2^14, -inf 2^7, +inf 1; a tile sums at most 64 of each) with visibility
// (0 or 1) says what each output gets.
//
// Nonzero if one of the word's cells is NaN or infinite (exponent, in E4M3 all bits, of ones).
template <bool F8> __device__ __forceinline__ uint32_t special_bits(uint32_t w) {
    return F8 ? ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
__device__ __forceinline__ void split_special(half8 v, half8 & fine, half8 & mark) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint16_t b = __builtin_bit_cast(uint16_t, (half_t)v[e]);
        const bool sp = (b & 0x7c00u) == 0x7c00u;
        fine[e] = sp ? (half_t)0.0f : (half_t)v[e];
        mark[e] = !sp ? (half_t)0.0f : (b & 0x3ffu) ? (half_t)16384.0f : (b & 0x8000u) ? (half_t)128.0f : (half_t)1.0f;
    }
}
__device__ __forceinline__ float special_of(float marks) {   // what is added to an output
    if (marks == 0.0f) return 0.0f;
    const int k = (int)marks;
    const bool neg = (k & 16383) >= 128, pos = (k & 127) != 0;
    return k >= 16384 || (neg && pos) ? __builtin_nanf("") : neg ? -INFINITY : INFINITY;
}

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

struct attn_t {
    const void * q;
    void * out;
    float * part_o;      // [parts][n_rows * H][hd] unscaled sums
    float * part_ml;     // [parts][n_rows * H][2] maximum, sum
    int H, G, causal, window, chunk, parts, tiles;
};

// ---------------------------------------------------------------------------
// Few rows: 16 queries per workgroup, keys straight from memory
// ---------------------------------------------------------------------------
// Bound by the cells' bytes.  Four waves take the 64-key tiles of the workgroup's range in turn and
// join through LDS at the end.  Lane (i, g) = (lane % 16, lane / 16): query column i; S^T tile u
// (16 of the 64 keys): row 4b + r is token 4u + r of block b, so the lane's D values (rows 4g + r)
// over the four tiles are the 16 tokens of block g.
#define FEW_T 16
template <int HD, bool F8, bool F32>
__global__ void __launch_bounds__(256, 2) k_paged_few(paged_t p, attn_t a) {
    constexpr int KS = HD / 32;                 // 32-dim steps of S
    constexpr int DT = HD / 16;                 // 16-dim tiles of O
    constexpr int KW = F8 ? HD / 64 : HD / 32;  // 16-byte loads of a lane per S tile
    constexpr int VW = F8 ? 1 : 2;              // 16-byte loads of a lane per O tile
    constexpr int OS = HD + 4;                  // LDS floats per query
    __shared__ float so[4][FEW_T][OS];
    __shared__ float sm[4][FEW_T], sl[4][FEW_T];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const unit_at un = unit_of(blockIdx.x, p.Hkv, a.tiles);
    if (un.kvh >= p.Hkv) return;
    const tile_at at = wave_tile<FEW_T>(p, a.G, un.tile);
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
    half8 qh[KS], ql[KS];
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
            // the row is brought to 2^8 .. 2^9 by a power of two, so that the second terms keep their bits
            amax = quad_max(amax);
            int ex = 0;
            if (amax > 0.0f && amax <= 3.402823466e38f) (void)frexpf(amax, &ex);
            ex = amax > 0.0f && amax <= 3.402823466e38f ? ex - 9 : 0;
            sc = ldexpf(sc, ex);
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    half_t hi, lo;
                    split16(ldexpf(x[s][k], -ex), hi, lo);
                    qh[s][k] = hi;
                    ql[s][k] = lo;
                }
        } else {
#pragma unroll
            for (int s = 0; s < KS; s++) qh[s] = *(const half8 *)((const half_t *)a.q + qo + dim(s));
        }
    }

    float m = -INFINITY, l = 0.0f;
    float4v o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = float4v{0.f, 0.f, 0.f, 0.f};

    for (int t = pt.t0 + wv; t < pt.t1; t += 4) {
        const int64_t kb = pg_block(p, at.s, un.kvh, 64 * t + 16 * (i >> 2));
        const int64_t vb = pg_block(p, at.s, un.kvh, 64 * t + 16 * g);
        // tokens of the lane's block that exist
        const int have = vb < 0 ? 0 : pg_clamp(keys - (64 * t + 16 * g), 0, 16);
        float ks = 1.0f, vs = 1.0f;
        if constexpr (F8) {
            if (kb >= 0) ks = p.scale[2 * kb];
            if (vb >= 0) vs = p.scale[2 * vb + 1];
        }
        constexpr int CB = F8 ? 1 : 2;
        // blocks that do not exist are read at block 0 and not used
        const uint8_t * kp = (const uint8_t *)p.k + ((kb < 0 ? 0 : kb) * (16 * HD) + (i & 3) * HD + (F8 ? 16 : 8) * g) * CB;
        const uint8_t * vp = (const uint8_t *)p.v + ((vb < 0 ? 0 : vb) * (16 * HD) + i * 16) * CB;
        u32x4 kr[4][KW], vr[DT][VW];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int w = 0; w < KW; w++) kr[u][w] = *(const u32x4 *)(kp + 4 * u * HD * CB + 64 * w);
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int w = 0; w < VW; w++) vr[d][w] = *(const u32x4 *)(vp + (d * 16 * 16) * CB + 16 * w);

        float s[16];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            float4v acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < KW; w++) {
                if constexpr (F8) {
                    const half8 k0 = f8_half8(kr[u][w].x, kr[u][w].y, ks), k1 = f8_half8(kr[u][w].z, kr[u][w].w, ks);
                    acc = mfma16(k0, qh[2 * w], acc);
                    acc = mfma16(k1, qh[2 * w + 1], acc);
                    if constexpr (F32) {
                        acc = mfma16(k0, ql[2 * w], acc);
                        acc = mfma16(k1, ql[2 * w + 1], acc);
                    }
                } else {
                    const half8 k0 = __builtin_bit_cast(half8, kr[u][w]);
                    acc = mfma16(k0, qh[w], acc);
                    if constexpr (F32) acc = mfma16(k0, ql[w], acc);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[4 * u + r] = acc[r] * sc;
        }
        // every key of the tile is there and every query sees it
        const bool full = __all(have == 16) && 64 * t >= all_lo && 64 * t + 63 <= all_hi;
        uint32_t vis = 0xffffu;                                     // of this lane's 16 tokens
        if (!full) {
            const int k0 = 64 * t + 16 * g;
            const int lo = pg_clamp(me.lo - k0, 0, 16), hi = pg_clamp(min(me.hi + 1 - k0, have), 0, 16);
            vis = hi > lo ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
#pragma unroll
            for (int k = 0; k < 16; k++) s[k] = (vis >> k) & 1u ? s[k] : -INFINITY;
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
                            vr[d][w][c] &= keep;
                        }
            }
        }
        bool special = false;
        if (!full || !F8) {
            uint32_t sp = 0;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int w = 0; w < VW; w++)
#pragma unroll
                    for (int c = 0; c < 4; c++) sp |= special_bits<F8>(vr[d][w][c]);
            special = __any(sp != 0);
        }
        half8 vis_h[2];
        if (special)
#pragma unroll
            for (int k = 0; k < 16; k++) vis_h[k >> 3][k & 7] = (half_t)(float)((vis >> k) & 1u);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            half8 v0, v1;
            if constexpr (F8) {
                v0 = f8_half8(vr[d][0].x, vr[d][0].y, vs);
                v1 = f8_half8(vr[d][0].z, vr[d][0].w, vs);
            } else {
                v0 = __builtin_bit_cast(half8, vr[d][0]);
                v1 = __builtin_bit_cast(half8, vr[d][1]);
            }
            float4v marks = {0.f, 0.f, 0.f, 0.f};
            if (special) {
                half8 m0, m1, n0, n1;
                split_special(v0, n0, m0);
                split_special(v1, n1, m1);
                v0 = n0;
                v1 = n1;
                marks = mfma16(m0, vis_h[0], marks);
                marks = mfma16(m1, vis_h[1], marks);
            }
            o[d] = mfma16(v0, ph[0], o[d]);
            o[d] = mfma16(v1, ph[1], o[d]);
            if constexpr (F32) {
                o[d] = mfma16(v0, pl[0], o[d]);
                o[d] = mfma16(v1, pl[1], o[d]);
            }
            if (special)
#pragma unroll
                for (int r = 0; r < 4; r++) o[d][r] += special_of(marks[r]);
        }
    }

    // ---- the four waves' results
    l = quad_sum(l);
    if (g == 0) {
        sm[wv][i] = m;
        sl[wv][i] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; d++) *(float4v *)&so[wv][i][16 * d + 4 * g] = o[d];
    __syncthreads();
    for (int e = threadIdx.x; e < FEW_T * (HD / 4); e += 256) {
        const int c = e / (HD / 4), d = 4 * (e % (HD / 4)), fc = f0 + c;
        if (fc > f1) continue;
        const float mx = fmaxf(fmaxf(sm[0][c], sm[1][c]), fmaxf(sm[2][c], sm[3][c]));
        float sum = 0.0f;
        float4v v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float r = sm[w][c] == -INFINITY ? (sl[w][c] == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(sm[w][c] - mx);
            sum += r * sl[w][c];
            const float4v x = *(const float4v *)&so[w][c][d];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = fmaf(r, x[k], v[k]);
        }
        const int64_t rh = (int64_t)(at.q.r0 + fc / a.G) * a.H + un.kvh * a.G + fc % a.G;
        if (F32) v *= 1.0f / 16384.0f;
        if (pt.parts == 1) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            v *= inv;
            if constexpr (F32) *(float4v *)((float *)a.out + rh * HD + d) = v;
            else *(half4 *)((half_t *)a.out + rh * HD + d) = half4{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
        } else {
            const int64_t at_part = (int64_t)blockIdx.y * p.n_rows * a.H + rh;
            *(float4v *)(a.part_o + at_part * HD + d) = v;
            if (d == 0) {
                a.part_ml[2 * at_part] = mx;
                a.part_ml[2 * at_part + 1] = sum;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Joining the parts of a split range
// ---------------------------------------------------------------------------
// One workgroup per (row, head): o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i; wave w takes the
// parts w, w + 4, .. in order, the waves are added in order: the same bits on every run.
template <int HD, bool F32, int T>
__global__ void __launch_bounds__(256) k_paged_join(paged_t p, attn_t a) {
    constexpr int DL = HD / 64;                 // dims per lane
    __shared__ float sv[4][HD], ss[4];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int kvh = blockIdx.y, G = a.G;
    const tile_at at = wave_tile<1>(p, G, blockIdx.x);          // tiles of one query: the flat query itself
    if (at.s < 0) return;
    const int nq = at.q.n * G, f0 = at.tile / T * T, f1 = min(f0 + T, nq) - 1;
    const int parts = part_of(pg_tiles(at.q, f0, f1, G, a.causal, a.window), 0, a.chunk, a.parts).parts;
    if (parts == 1) return;
    const int64_t rh = (int64_t)(at.q.r0 + at.tile / G) * a.H + kvh * G + at.tile % G;
    const int64_t step = (int64_t)p.n_rows * a.H;
    float mx = -INFINITY;
    for (int i = lane; i < parts; i += 64) mx = fmaxf(mx, a.part_ml[2 * (i * step + rh)]);
    mx = wave_max(mx);
    float sum = 0.0f, v[DL] = {};
#pragma unroll 4
    for (int i = wv; i < parts; i += 4) {
        const float mi = a.part_ml[2 * (i * step + rh)], li = a.part_ml[2 * (i * step + rh) + 1];
        const float r = mi == -INFINITY ? (li == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(mi - mx);
        sum += r * li;
#pragma unroll
        for (int k = 0; k < DL; k++) v[k] = fmaf(r, a.part_o[(i * step + rh) * HD + DL * lane + k], v[k]);
    }
#pragma unroll
    for (int k = 0; k < DL; k++) sv[wv][DL * lane + k] = v[k];
    if (lane == 0) ss[wv] = sum;
    __syncthreads();
    if (threadIdx.x < HD) {
        const int d = threadIdx.x;
        const float l = (ss[0] + ss[1]) + (ss[2] + ss[3]), x = (sv[0][d] + sv[1][d]) + (sv[2][d] + sv[3][d]);
        const float y = l == 0.0f ? 0.0f : x * (1.0f / l);
        if constexpr (F32) ((float *)a.out)[rh * HD + d] = y;
        else ((half_t *)a.out)[rh * HD + d] = (half_t)y;
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct attn_plan { int tiles, chunk, parts; };
static attn_plan plan_of(const paged_t & p, int H, int64_t max_keys, bool split) {
    const int G = H / p.Hkv;
    const int64_t queries = (int64_t)p.n_rows * G;
    attn_plan r;
    r.tiles = (int)(queries / FEW_T + std::min<int64_t>(p.n_seqs, p.n_rows));
    const int64_t kt = (std::min<int64_t>(std::max<int64_t>(max_keys, 1), p.cap) + 63) / 64;
    const int64_t units = (int64_t)p.Hkv * std::max<int64_t>(std::min<int64_t>(p.n_seqs, p.n_rows), queries / FEW_T);
    const int64_t want = std::max<int64_t>(1, 512 / units);
    r.chunk = (int)std::max<int64_t>(8, (kt + want - 1) / want);
    r.parts = split ? (int)((kt + r.chunk - 1) / r.chunk) : 1;
    return r;
}

extern "C" size_t dfx_paged_attention_ws_bytes(const dfx_paged_cache * cache, const dfx_paged_batch * batch, int n_head,
                                               int type) {
    paged_t p;
    (void)type;
    if (paged_of("dfx_paged_attention_ws_bytes", cache, batch, n_head, &p) != DFX_OK) return 0;
    if (p.n_rows == 0 || p.n_seqs == 0) return 0;
    const attn_plan pl = plan_of(p, n_head, batch->max_keys, true);
    return pl.parts <= 1 ? 0 : (size_t)pl.parts * p.n_rows * n_head * (cache->head_dim + 2) * sizeof(float);
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
    const attn_plan pl = plan_of(p, n_head, batch->max_keys, ws != nullptr);
    attn_t a = {q, out, (float *)ws, nullptr, n_head, n_head / p.Hkv, causal ? 1 : 0, window, pl.chunk, pl.parts, pl.tiles};
    a.part_ml = a.part_o + (size_t)pl.parts * p.n_rows * n_head * hd;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid(unit_grid(p.Hkv, pl.tiles), (unsigned)pl.parts);
#define FEW(HD, F8, F32) hipLaunchKernelGGL((k_paged_few<HD, F8, F32>), grid, dim3(256), 0, st, p, a)
#define FEW_TYPES(HD)                                                                                                 \
    do {                                                                                                              \
        if (cache->type == DFX_TYPE_F8) {                                                                             \
            if (type == DFX_TYPE_F32) FEW(HD, true, true);                                                            \
            else FEW(HD, true, false);                                                                                \
        } else {                                                                                                      \
            if (type == DFX_TYPE_F32) FEW(HD, false, true);                                                           \
            else FEW(HD, false, false);                                                                               \
        }                                                                                                             \
    } while (0)
    if (hd == 128) FEW_TYPES(128);
    else FEW_TYPES(64);
    DFX_CHECK_LAUNCH("dfx_paged_attention");
    if (pl.parts > 1) {
        const dim3 jg((unsigned)((int64_t)p.n_rows * a.G), (unsigned)p.Hkv);
#define JOIN(HD, F32) hipLaunchKernelGGL((k_paged_join<HD, F32, FEW_T>), jg, dim3(256), 0, st, p, a)
        if (hd == 128) {
            if (type == DFX_TYPE_F32) JOIN(128, true);
            else JOIN(128, false);
        } else {
            if (type == DFX_TYPE_F32) JOIN(64, true);
            else JOIN(64, false);
        }
        DFX_CHECK_LAUNCH("dfx_paged_attention (join)");
    }
    return DFX_OK;
}
