// k_logprobs.hip — log probabilities of given tokens, entropy and best alternatives of logits rows.
//
//   m = max x,  S = sum e,  T = sum e (x - m),  e = exp(x - m)
//   log p_t = (x_t - m) - log S,   entropy = log S - T / S
// A row is cut into pieces of 64 * 4 * U logits, one wave each, so that one row fills the chip as
// well as many do.  A wave keeps its piece in registers: one read gives m, S, T and the piece's
// candidates for the alternatives; no barrier, nothing shared.  A second kernel joins a row's pieces.
//
// Alternatives: of the 128 values that are the two largest of each lane, the n-th largest is a bound
// that at least n elements of the piece reach; few more do (n of 20 over 4096 normal values: about
// 22).  It is found to 16 bits by counting with ballots, and what reaches it is listed.  A piece
// where too many do (equal values) finds its n largest one after another instead.
#include "dfx_device.h"

#include <algorithm>

#define LP_MAX_TOP 64
#define LOG2E_F 1.44269504088896341f

// Order of values as unsigned integers: larger value, larger key; NaN and -inf lowest, -0 as +0.
__device__ __forceinline__ uint32_t lp_key(float x) {
    const float y = x > -INFINITY ? x + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(y);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
#define LP_NONE 0x007fffffu   // key of -inf: no candidate

// The largest 16-bit prefix P with at least n of the wave's 128 keys >= P << 16.
__device__ __forceinline__ uint32_t wave_bound(uint32_t a, uint32_t b, int n) {
    uint32_t t = 0;
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t c = t | (1u << bit);
        if (__popcll(__ballot(a >= c)) + __popcll(__ballot(b >= c)) >= n) t = c;
    }
    return t;
}

struct lp_cand { float x; int32_t i; };
struct lp_part { float m, S, T; int32_t n; };   // n: candidates listed

// candidate a before b: larger value, then lower index
__device__ __forceinline__ bool lp_before(uint32_t ka, int ia, uint32_t kb, int ib) {
    return ka != kb ? ka > kb : ia < ib;
}

// The wave's best (key, index) of each lane's: in every lane.
__device__ __forceinline__ void wave_best(uint32_t & k, int & i) {
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t ok = __shfl_xor(k, o, WAVE);
        const int oi = __shfl_xor(i, o, WAVE);
        if (lp_before(ok, oi, k, i)) {
            k = ok;
            i = oi;
        }
    }
}

template <int U, bool VEC>
__global__ void __launch_bounds__(256, 4) k_lp_pieces(const float * __restrict__ logits, int64_t ld, int64_t n_logits,
                                                   const int32_t * __restrict__ rows, int V, int pieces, int n_top,
                                                   int cap, lp_part * __restrict__ part,
                                                   lp_cand * __restrict__ cand) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int piece = blockIdx.x * 4 + wv;
    if (piece >= pieces) return;
    const int64_t row = rows ? (int64_t)rows[blockIdx.y] : (int64_t)blockIdx.y;
    if (row < 0 || row >= n_logits) return;
    const float * x = logits + row * ld;
    const int base = piece * (256 * U);
    // element c of lane's group u
    auto index = [&](int u, int c) { return VEC ? base + 256 * u + 4 * lane + c : base + 256 * u + 64 * c + lane; };
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if constexpr (VEC) {
            const int i = index(u, 0);
            const float4 w = *(const float4 *)(x + min(i, V - 4));
            v[u][0] = i < V ? w.x : -INFINITY;
            v[u][1] = i < V ? w.y : -INFINITY;
            v[u][2] = i < V ? w.z : -INFINITY;
            v[u][3] = i < V ? w.w : -INFINITY;
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int i = index(u, c);
                const float w = x[min(i, V - 1)];
                v[u][c] = i < V ? w : -INFINITY;
            }
        }
    }
    float m1 = -INFINITY, m2 = -INFINITY;             // the lane's two largest
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            m2 = __builtin_amdgcn_fmed3f(m1, m2, v[u][c]);   // with NaN the least of the others: m2
            m1 = fmaxf(m1, v[u][c]);
        }
    const float m = wave_max(m1);
    // -inf adds 0 (not 0 * -inf); NaN stays, and so does +inf - inf
    float S = 0.0f, T = 0.0f;
    const float mm = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const float d = v[u][c] - mm;
            const float e = __builtin_amdgcn_exp2f(d * LOG2E_F);
            S += e;
            T = fmaf(e, fmaxf(d, -256.0f), T);
        }
    const double Sd = wave_sum_d((double)S), Td = wave_sum_d((double)T);
    const int64_t slot = (int64_t)blockIdx.y * pieces + piece;
    int n = 0;
    if (n_top > 0) {
        lp_cand * out = cand + slot * cap;
        const uint32_t t = max(wave_bound(lp_key(m1), lp_key(m2), n_top), LP_NONE + 1);
        const float tf = lp_value(t);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float g = fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3]));
            if (!__any(g >= tf)) continue;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const bool is = v[u][c] >= tf;
                const uint64_t has = __ballot(is);
                const int at = n + __popcll(has & ((1ull << lane) - 1));
                if (is && at < cap) out[at] = {v[u][c], index(u, c)};
                n += __popcll(has);
            }
        }
        if (n > cap) {
            // too many equal values: the n_top best, each the best behind the one before
            uint32_t pk = 0xffffffffu;
            int pi = -1;
            for (n = 0; n < n_top; n++) {
                uint32_t bk = LP_NONE;
                int bi = 0x7fffffff;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const uint32_t k = lp_key(v[u][c]);
                        const int i = index(u, c);
                        if (lp_before(pk, pi, k, i) && lp_before(k, i, bk, bi)) {
                            bk = k;
                            bi = i;
                        }
                    }
                wave_best(bk, bi);
                if (bk <= LP_NONE) break;
                if (lane == 0) out[n] = {lp_value(bk), bi};
                pk = bk;
                pi = bi;
            }
        }
    }
    if (lane == 0) part[slot] = {m, (float)Sd, (float)Td, n};
}

// One workgroup per row: sums of the pieces in double, then the n_top best of the pieces' candidates
// the same way: a bound from each lane's two largest, what reaches it into LDS, places by counting.
#define LP_LIST 1024
__global__ void __launch_bounds__(256) k_lp_join(const float * __restrict__ logits, int64_t ld, int64_t n_logits,
                                                 const int32_t * __restrict__ rows, int V, int pieces, int n_top,
                                                 int cap, const lp_part * __restrict__ part,
                                                 const lp_cand * __restrict__ cand,
                                                 const int32_t * __restrict__ tokens, int n_tok,
                                                 float * __restrict__ logprob, float * __restrict__ entropy,
                                                 int32_t * __restrict__ top_id, float * __restrict__ top_logprob) {
    __shared__ float red_m[4];
    __shared__ double red_s[4], red_t[4];
    __shared__ uint32_t red_k[4];
    __shared__ int red_i[4];
    __shared__ uint32_t list_k[LP_LIST];
    __shared__ int list_i[LP_LIST];
    __shared__ int list_n;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int64_t r = blockIdx.x;
    const int64_t row = rows ? (int64_t)rows[r] : r;
    const float nan = __builtin_nanf("");
    if (row < 0 || row >= n_logits) {
        for (int j = tid; j < n_tok; j += 256) logprob[r * n_tok + j] = nan;
        for (int j = tid; j < n_top; j += 256) {
            top_id[r * n_top + j] = -1;
            top_logprob[r * n_top + j] = nan;
        }
        if (tid == 0 && entropy) entropy[r] = nan;
        return;
    }
    const float * x = logits + row * ld;
    const lp_part * pr = part + r * pieces;
    float m = -INFINITY;
    for (int i = tid; i < pieces; i += 256) m = fmaxf(m, pr[i].m);
    m = wave_max(m);
    if (lane == 0) red_m[wv] = m;
    if (tid == 0) list_n = 0;
    __syncthreads();
    m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    double S = 0.0, T = 0.0;
    for (int i = tid; i < pieces; i += 256) {
        const lp_part q = pr[i];
        if (q.m == -INFINITY) {
            S += (double)q.S;                          // 0, or NaN
        } else {
            const double d = (double)q.m - (double)m, w = exp(d);
            S += w * (double)q.S;
            if (w > 0.0) T += w * ((double)q.T + d * (double)q.S);
        }
    }
    S = wave_sum_d(S);
    T = wave_sum_d(T);
    if (lane == 0) {
        red_s[wv] = S;
        red_t[wv] = T;
    }
    __syncthreads();
    S = (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]);
    T = (red_t[0] + red_t[1]) + (red_t[2] + red_t[3]);
    // nothing above -inf: S is 0 and its logarithm no number
    const double log_s = S > 0.0 ? log(S) : (double)nan;
    if (tid == 0 && entropy) entropy[r] = (float)(log_s - T / S);
    for (int j = tid; j < n_tok; j += 256) {
        const int t = tokens[r * n_tok + j];
        logprob[r * n_tok + j] = t >= 0 && t < V ? (float)(((double)x[t] - (double)m) - log_s) : nan;
    }
    if (n_top == 0) return;

    const lp_cand * cr = cand + r * pieces * cap;
    // the candidates of this wave's pieces: wave wv takes the pieces wv, wv + 4, ..
    uint32_t k1 = 0, k2 = 0;
    for (int i = wv; i < pieces; i += 4) {
        const int n = pr[i].n;
        for (int j = lane; j < n; j += 64) {
            const uint32_t k = lp_key(cr[(int64_t)i * cap + j].x);
            k2 = max(k2, min(k1, k));
            k1 = max(k1, k);
        }
    }
    const uint32_t tw = wave_bound(k1, k2, n_top);
    if (lane == 0) red_k[wv] = tw;
    __syncthreads();
    const uint32_t t = max(max(red_k[0], red_k[1]), max(red_k[2], red_k[3]));
    for (int i = wv; i < pieces; i += 4) {
        const int n = pr[i].n;
        for (int j = lane; j < n; j += 64) {
            const lp_cand c = cr[(int64_t)i * cap + j];
            const uint32_t k = lp_key(c.x);
            if (k >= t) {
                const int at = atomicAdd(&list_n, 1);
                if (at < LP_LIST) {
                    list_k[at] = k;
                    list_i[at] = c.i;
                }
            }
        }
    }
    __syncthreads();
    int n = list_n;
    if (n <= LP_LIST) {
        for (int e = tid; e < n; e += 256) {
            const uint32_t k = list_k[e];
            const int i = list_i[e];
            int before = 0;
            for (int f = 0; f < n; f++) before += lp_before(list_k[f], list_i[f], k, i) ? 1 : 0;
            if (before < n_top) {
                top_id[r * n_top + before] = i;
                top_logprob[r * n_top + before] = (float)(((double)lp_value(k) - (double)m) - log_s);
            }
        }
    } else {
        // equal values throughout: one after another
        uint32_t pk = 0xffffffffu;
        int pi = -1;
        for (int e = 0; e < n_top; e++) {
            uint32_t bk = 0;
            int bi = 0x7fffffff;
            for (int i = wv; i < pieces; i += 4)
                for (int j = lane; j < pr[i].n; j += 64) {
                    const lp_cand c = cr[(int64_t)i * cap + j];
                    const uint32_t k = lp_key(c.x);
                    if (lp_before(pk, pi, k, c.i) && lp_before(k, c.i, bk, bi)) {
                        bk = k;
                        bi = c.i;
                    }
                }
            wave_best(bk, bi);
            __syncthreads();                           // the round before has been read
            if (lane == 0) {
                red_k[wv] = bk;
                red_i[wv] = bi;
            }
            __syncthreads();
            bk = red_k[0];
            bi = red_i[0];
            for (int w = 1; w < 4; w++)
                if (lp_before(red_k[w], red_i[w], bk, bi)) {
                    bk = red_k[w];
                    bi = red_i[w];
                }
            if (tid == 0) {
                top_id[r * n_top + e] = bi;
                top_logprob[r * n_top + e] = (float)(((double)lp_value(bk) - (double)m) - log_s);
            }
            pk = bk;
            pi = bi;
        }
        n = n_top;
    }
    // fewer than n_top above -inf: the rest in index order (-inf, NaN), then nothing
    if (n < n_top && wv == 0) {
        for (int i0 = 0; i0 < V && n < n_top; i0 += 64) {
            const int i = i0 + lane;
            const bool low = i < V && !(x[min(i, V - 1)] > -INFINITY);
            const uint64_t has = __ballot(low);
            const int at = n + __popcll(has & ((1ull << lane) - 1));
            if (low && at < n_top) {
                top_id[r * n_top + at] = i;
                top_logprob[r * n_top + at] = (float)(((double)x[i] - (double)m) - log_s);
            }
            n += __popcll(has);
        }
        for (int j = n + lane; j < n_top; j += 64) {
            top_id[r * n_top + j] = -1;
            top_logprob[r * n_top + j] = -INFINITY;
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct lp_plan { int u, pieces, cap; size_t part_bytes, bytes; };
static lp_plan lp_plan_of(int64_t n_rows, int64_t V, int n_top) {
    lp_plan p;
    p.u = n_rows * ((V + 4095) / 4096) >= 4096 ? 16 : 4;
    p.pieces = (int)((V + 256 * p.u - 1) / (256 * p.u));
    p.cap = n_top > 0 ? 2 * n_top + 32 : 0;
    p.part_bytes = align256((size_t)n_rows * p.pieces * sizeof(lp_part));
    p.bytes = p.part_bytes + (size_t)n_rows * p.pieces * p.cap * sizeof(lp_cand);
    return p;
}
static bool lp_shape_ok(int64_t n_rows, int64_t V, int n_top) {
    return n_rows >= 0 && n_rows <= (1 << 24) && V > 0 && V <= (1 << 30) && n_top >= 0 && n_top <= LP_MAX_TOP;
}

extern "C" size_t dfx_token_logprobs_ws_bytes(int64_t n_rows, int64_t V, int n_top) {
    if (!lp_shape_ok(n_rows, V, n_top)) return 0;
    return lp_plan_of(n_rows, V, n_top).bytes;
}

extern "C" int dfx_token_logprobs(const float * logits, int64_t ld, int64_t n_logits, const int32_t * rows,
                                  int64_t n_rows, int64_t V, const int32_t * tokens, int n_tok, float * logprob,
                                  float * entropy, int n_top, int32_t * top_id, float * top_logprob, void * ws,
                                  void * stream) {
    if (!lp_shape_ok(n_rows, V, n_top) || ld < V || n_logits < 0 || n_tok < 0) {
        dfx_set_error("dfx_token_logprobs: bad shape rows=%lld V=%lld ld=%lld logits=%lld tokens=%d top=%d (at most %d)",
                      (long long)n_rows, (long long)V, (long long)ld, (long long)n_logits, n_tok, n_top, LP_MAX_TOP);
        return DFX_ERR_ARG;
    }
    if (n_rows == 0) return DFX_OK;
    if (!logits || !ws || ((uintptr_t)ws & 15) || (n_tok > 0 && (!tokens || !logprob)) ||
        (n_top > 0 && (!top_id || !top_logprob))) {
        dfx_set_error("dfx_token_logprobs: logits, workspace (16-byte aligned), tokens or outputs missing");
        return DFX_ERR_ARG;
    }
    const lp_plan p = lp_plan_of(n_rows, V, n_top);
    lp_part * part = (lp_part *)ws;
    lp_cand * cand = (lp_cand *)((uint8_t *)ws + p.part_bytes);
    hipStream_t st = (hipStream_t)stream;
    const bool vec = (V & 3) == 0 && (ld & 3) == 0 && ((uintptr_t)logits & 15) == 0;
    // rows in slices that the grid's second dimension holds
    for (int64_t r0 = 0; r0 < n_rows; r0 += 65535) {
        const int64_t n = std::min<int64_t>(65535, n_rows - r0);
        const dim3 grid((unsigned)((p.pieces + 3) / 4), (unsigned)n);
        const float * lg = rows ? logits : logits + r0 * ld;
        const int64_t nl = rows ? n_logits : n_logits - r0;
        const int32_t * rw = rows ? rows + r0 : nullptr;
        lp_part * pp = part + r0 * p.pieces;
        lp_cand * cc = cand + r0 * p.pieces * p.cap;
#define PIECES(U, VEC)                                                                                                \
    hipLaunchKernelGGL((k_lp_pieces<U, VEC>), grid, dim3(256), 0, st, lg, ld, nl, rw, (int)V, p.pieces, n_top, p.cap,  \
                       pp, cc)
        if (p.u == 16) {
            if (vec) PIECES(16, true);
            else PIECES(16, false);
        } else {
            if (vec) PIECES(4, true);
            else PIECES(4, false);
        }
#undef PIECES
        DFX_CHECK_LAUNCH("dfx_token_logprobs");
    }
    hipLaunchKernelGGL(k_lp_join, dim3((unsigned)n_rows), dim3(256), 0, st, logits, ld, n_logits, rows, (int)V, p.pieces,
                       n_top, p.cap, part, cand, tokens, n_tok, logprob, entropy, top_id, top_logprob);
    DFX_CHECK_LAUNCH("dfx_token_logprobs (join)");
    return DFX_OK;
}
