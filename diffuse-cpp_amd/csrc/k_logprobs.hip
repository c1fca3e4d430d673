// k_logprobs.hip — log probabilities of given tokens, entropy and best alternatives of logits rows.
//
//   m = max x,  S = sum e,  T = sum e (x - m),  e = exp(x - m)
//   log p_t = (x_t - m) - log S,   entropy = log S - T / S
// A row is cut into pieces of LP_PIECE logits, one wave each, so that one row fills the chip as
// well as many do.  A wave keeps its piece in registers: one read gives m, S, T and the piece's
// candidates for the alternatives; no barrier, nothing shared.  A second kernel joins a row's pieces.
//
// Alternatives: of the 128 values that are the two largest of each lane, the n-th largest is a bound
// that at least n elements of the piece reach; few more do (a third one of a lane, equal values).
// It is found by halving, counting with ballots, and what reaches it is listed.  A piece where too many
// do (equal values) finds the n-th largest of all its elements the same way.
#include "dfx_device.h"

#include <algorithm>

#define LP_MAX_TOP 64
// Logits of a wave: 32 registers a lane (1024: one row with 5 alternatives no faster, 64 rows 6 % slower).
#define LP_PIECE 2048
#define LOG2E_F 1.44269504088896341f

// A candidate as one integer whose order is that of the alternatives: the value in the high word
// (larger value, larger integer; NaN as -inf, -0 as +0), the complement of the index in the low one.
// 0: none.
__device__ __forceinline__ uint32_t lp_key(float x) {
    const float y = x > -INFINITY ? x + 0.0f : -INFINITY;
    const uint32_t b = __float_as_uint(y);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t lp_cand(uint32_t key, int i) { return (uint64_t)key << 32 | (uint32_t)~i; }
__device__ __forceinline__ int lp_index(uint64_t c) { return (int)~(uint32_t)c; }
#define LP_LOWEST 0x00800000u   // key of the lowest value above -inf

struct lp_part { float m, S, T, pad; };

// A bound that at least n <= 64 of the wave's 128 keys (a >= b in each lane) reach, and, but for equal
// ones, at most n + LP_SLACK: between the least and the largest a, halved until the count is near.
#define LP_SLACK 6
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, true));
    return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
               max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}
__device__ __forceinline__ uint32_t wave_bound(uint32_t a, uint32_t b, int n) {
    uint32_t lo = ~wave_max_u(~a), hi = wave_max_u(a);              // all 64 a reach lo (0: lanes with nothing)
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        const int k = __popcll(__ballot(a >= mid)) + __popcll(__ballot(b >= mid));
        if (k < n) {
            hi = mid - 1;
            continue;
        }
        lo = mid;
        if (k <= n + LP_SLACK) break;
    }
    return lo;
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor(v, o, WAVE);
        v = w > v ? w : v;
    }
    return v;
}

// Bound by bytes: 700 rows of 152064 without alternatives (426 MB) 73 us, 5.8 TB/s (79.4 with the join); 256
// rows of 126464 with 20 alternatives (129.5 MB) 28.5 us, 4.5 TB/s, the bound's ballots and the list beside
// the loads.  VEC: rows of 16-byte pieces; element by element otherwise.
template <bool VEC>
__global__ void __launch_bounds__(256, 4) k_lp_pieces(const float * __restrict__ logits, int64_t ld, int64_t n_logits,
                                                      const int32_t * __restrict__ rows, int V, int pieces, int n_top,
                                                      int cap, lp_part * __restrict__ part,
                                                      uint64_t * __restrict__ cand) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int piece = blockIdx.x * 4 + wv;
    if (piece >= pieces) return;
    const int64_t row = rows ? (int64_t)rows[blockIdx.y] : (int64_t)blockIdx.y;
    if (row < 0 || row >= n_logits) return;
    const float * x = logits + row * ld;
    constexpr int U = LP_PIECE / 256;
    const int base = piece * LP_PIECE;
    // element e = 4 u + c of the lane
    auto index = [&](int e) { return base + (VEC ? 256 * (e >> 2) + 4 * lane + (e & 3) : 64 * e + lane); };
    float v[4 * U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if constexpr (VEC) {
            const int i = index(4 * u);
            const float4 w = *(const float4 *)(x + min(i, V - 4));
            v[4 * u] = i < V ? w.x : -INFINITY;
            v[4 * u + 1] = i < V ? w.y : -INFINITY;
            v[4 * u + 2] = i < V ? w.z : -INFINITY;
            v[4 * u + 3] = i < V ? w.w : -INFINITY;
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int i = index(4 * u + c);
                const float w = x[min(i, V - 1)];
                v[4 * u + c] = i < V ? w : -INFINITY;
            }
        }
    }
    float m1 = -INFINITY, m2 = -INFINITY;             // the lane's two largest
#pragma unroll
    for (int e = 0; e < 4 * U; e++) {
        m2 = __builtin_amdgcn_fmed3f(m1, m2, v[e]);   // with NaN the least of the others: m2
        m1 = fmaxf(m1, v[e]);
    }
    const float m = wave_max(m1);
    uint32_t bound = 0xffffffffu;
    uint64_t mask = 0;                                // the lane's elements that reach the bound
    if (n_top > 0) {
        bound = max(wave_bound(lp_key(m1), lp_key(m2), n_top), LP_LOWEST);
        const float bf = lp_value(bound);
#pragma unroll
        for (int e = 0; e < 4 * U; e++) mask |= v[e] >= bf ? 1ull << e : 0ull;
    }
    // -inf adds 0 (not 0 * -inf); NaN stays, and so does +inf - inf
    float S = 0.0f, T = 0.0f;
    const float mm = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int e = 0; e < 4 * U; e++) {
        const float d = v[e] - mm;
        const float p = __builtin_amdgcn_exp2f(d * LOG2E_F);
        S += p;
        T = fmaf(p, fmaxf(d, -256.0f), T);
    }
    const double Sd = wave_sum_d((double)S), Td = wave_sum_d((double)T);
    const int64_t slot = (int64_t)blockIdx.y * pieces + piece;
    if (lane == 0) part[slot] = {m, (float)Sd, (float)Td, 0.0f};
    if (n_top == 0) return;
    // the list: each lane's elements in turn (read again, from the cache), empty places as none
    uint64_t * out = cand + slot * cap;
    int n = 0;
    for (uint64_t any = __ballot(mask != 0); any; any = __ballot(mask != 0)) {
        const int at = n + __popcll(any & ((1ull << lane) - 1));
        if (mask != 0 && at < cap) {
            const int i = index(__ffsll((unsigned long long)mask) - 1);
            out[at] = lp_cand(lp_key(x[i]), i);
        }
        mask &= mask - 1;
        n += __popcll(any);
        if (n > cap) break;
    }
    if (n > cap) {
        // Too many, equal ones among them: the bound is taken exactly (the n_top-th largest of the piece's
        // elements, counting them all), what is above it listed, and of those that equal it the first.
        auto count = [&](uint32_t key) __attribute__((always_inline)) {
            const float f = lp_value(key);
            int k = 0;
#pragma unroll
            for (int e = 0; e < 4 * U; e++) k += __popcll(__ballot(v[e] >= f));
            return k;
        };
        uint32_t lo = bound, hi = wave_max_u(lp_key(m1));
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo + 1) / 2;
            if (count(mid) >= n_top) lo = mid;
            else hi = mid - 1;
        }
        const float at_f = lp_value(lo), above_f = lp_value(lo + 1);  // behind +inf: NaN, nothing is above
        const uint64_t lower = (1ull << lane) - 1;
        int above = 0, equal = count(lo + 1);                         // places of the next of either
#pragma unroll
        for (int u = 0; u < U; u++) {
            int mine = equal;                                         // index order: by lane (VEC), or by element
            if constexpr (VEC)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint64_t eq = __ballot(v[4 * u + c] >= at_f && !(v[4 * u + c] >= above_f));
                    mine += __popcll(eq & lower);
                    equal += __popcll(eq);
                }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int e = 4 * u + c;
                const bool gt = v[e] >= above_f, eq = v[e] >= at_f && !gt;
                const uint64_t has = __ballot(gt);
                if (gt) out[above + __popcll(has & lower)] = lp_cand(lp_key(v[e]), index(e));
                above += __popcll(has);
                if constexpr (VEC) {
                    if (eq && mine < n_top) out[mine] = lp_cand(lp_key(v[e]), index(e));
                    mine += eq;
                } else {
                    const uint64_t he = __ballot(eq);
                    const int at = equal + __popcll(he & lower);
                    if (eq && at < n_top) out[at] = lp_cand(lp_key(v[e]), index(e));
                    equal += __popcll(he);
                }
            }
        }
        n = n_top;
    }
    for (int j = n + lane; j < cap; j += 64) out[j] = 0;
}

// One workgroup per row: sums of the pieces in double, then the n_top best of the pieces' candidates
// the same way: a bound from each lane's two largest, what reaches it into LDS, places by counting.
// Bound by latency (a round of loads, two barriers, the counting): 8.5 us for 256 rows of 62 pieces and 20
// alternatives, 6.4 for one row of 75 pieces and 5, 5 for 700 rows without any.
#define LP_LIST 2048
#define LP_MANY 128
#define LP_JOIN 1024
__global__ void __launch_bounds__(LP_JOIN) k_lp_join(const float * __restrict__ logits, int64_t ld, int64_t n_logits,
                                                     const int32_t * __restrict__ rows, int V, int pieces, int n_top,
                                                     int cap, const lp_part * __restrict__ part,
                                                     const uint64_t * __restrict__ cand,
                                                     const int32_t * __restrict__ tokens, int n_tok,
                                                     float * __restrict__ logprob, float * __restrict__ entropy,
                                                     int32_t * __restrict__ top_id, float * __restrict__ top_logprob) {
    constexpr int NW = LP_JOIN / 64, HELD = 8;
    __shared__ float red_m[NW];
    __shared__ double red_s[NW], red_t[NW];
    __shared__ uint32_t red_k[NW];
    __shared__ uint64_t red_c[NW];
    __shared__ uint64_t list[LP_LIST];
    __shared__ int list_n;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, nt = blockDim.x, nw = nt >> 6;
    const int64_t r = blockIdx.x;
    const int64_t row = rows ? (int64_t)rows[r] : r;
    const float nan = __builtin_nanf("");
    if (row < 0 || row >= n_logits) {
        for (int j = tid; j < n_tok; j += nt) logprob[r * n_tok + j] = nan;
        for (int j = tid; j < n_top; j += nt) {
            top_id[r * n_top + j] = -1;
            top_logprob[r * n_top + j] = nan;
        }
        if (tid == 0 && entropy) entropy[r] = nan;
        return;
    }
    const float * x = logits + row * ld;
    const lp_part * pr = part + r * pieces;
    const uint64_t * cr = cand + r * pieces * cap;
    const int slots = pieces * cap;
    lp_part first = {-INFINITY, 0.0f, 0.0f, 0.0f};
    if (tid < pieces) first = pr[tid];
    // a given token's logit is fetched with the parts: its line is far from them
    int tok = -1;
    float xt = 0.0f;
    if (tid < n_tok) {
        tok = tokens[r * n_tok + tid];
        if (tok >= 0 && tok < V) xt = x[tok];
    }
    uint32_t k1 = 0, k2 = 0;                           // the two largest of the thread's candidates
    uint64_t held[HELD];                               // the first of them
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        held[i] = 0;
        if (tid + i * nt < slots) held[i] = cr[tid + i * nt];
    }
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const uint32_t k = (uint32_t)(held[i] >> 32);
        k2 = max(k2, min(k1, k));
        k1 = max(k1, k);
    }
#pragma unroll 4
    for (int j = tid + HELD * nt; j < slots; j += nt) {
        const uint32_t k = (uint32_t)(cr[j] >> 32);
        k2 = max(k2, min(k1, k));
        k1 = max(k1, k);
    }
    float m = first.m;
    for (int i = tid + nt; i < pieces; i += nt) m = fmaxf(m, pr[i].m);
    m = wave_max(m);
    const uint32_t tw = n_top ? wave_bound(k1, k2, n_top) : 0;
    if (lane == 0) {
        red_m[wv] = m;
        red_k[wv] = tw;
    }
    if (tid == 0) list_n = 0;
    __syncthreads();
    uint32_t bound = 1;                                // 0 is no candidate
    for (int w = 0; w < nw; w++) {
        m = fmaxf(m, red_m[w]);
        bound = max(bound, red_k[w]);
    }
    double S = 0.0, T = 0.0;
    for (int i = tid; i < pieces; i += nt) {
        const lp_part q = i == tid ? first : pr[i];
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
    auto enlist = [&](uint64_t c) {
        if ((uint32_t)(c >> 32) >= bound) {
            const int at = atomicAdd(&list_n, 1);      // any order: places are counted below
            if (at < LP_LIST) list[at] = c;
        }
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) enlist(held[i]);
    for (int j = tid + HELD * nt; j < slots; j += nt) enlist(cr[j]);
    __syncthreads();
    S = T = 0.0;
    for (int w = 0; w < nw; w++) {
        S += red_s[w];
        T += red_t[w];
    }
    // nothing above -inf: S is 0 and its logarithm no number
    const double log_s = S > 0.0 ? log(S) : (double)nan;
    if (tid == 0 && entropy) entropy[r] = (float)(log_s - T / S);
    for (int j = tid; j < n_tok; j += nt) {
        if (j != tid) {
            tok = tokens[r * n_tok + j];
            if (tok >= 0 && tok < V) xt = x[tok];
        }
        logprob[r * n_tok + j] = tok >= 0 && tok < V ? (float)(((double)xt - (double)m) - log_s) : nan;
    }
    if (n_top == 0) return;
    auto write = [&](int at, int id, float value) {
        top_id[r * n_top + at] = id;
        top_logprob[r * n_top + at] = (float)(((double)value - (double)m) - log_s);
    };
    int n = list_n;
    if (n > LP_MANY && n <= LP_LIST) {
        // more than are quickly counted: one wave takes their bound, and keeps what reaches it
        __syncthreads();                               // list_n has been read
        if (wv == 0) {
            k1 = k2 = 0;
            for (int j = lane; j < n; j += 64) {
                const uint32_t k = (uint32_t)(list[j] >> 32);
                k2 = max(k2, min(k1, k));
                k1 = max(k1, k);
            }
            bound = wave_bound(k1, k2, n_top);
            int kept = 0;
            for (int j0 = 0; j0 < n; j0 += 64) {       // places before the ones that are read next
                const uint64_t c = j0 + lane < n ? list[j0 + lane] : 0;
                const bool is = c && (uint32_t)(c >> 32) >= bound;
                const uint64_t has = __ballot(is);
                if (is) list[kept + __popcll(has & ((1ull << lane) - 1))] = c;
                kept += __popcll(has);
            }
            if (lane == 0) list_n = kept;
        }
        __syncthreads();
        n = list_n;
    }
    if (n <= LP_LIST) {
        for (int e = tid; e < n; e += nt) {
            const uint64_t c = list[e];
            int before = 0;
#pragma unroll 8
            for (int f = 0; f < n; f++) before += list[f] > c ? 1 : 0;
            if (before < n_top) write(before, lp_index(c), lp_value((uint32_t)(c >> 32)));
        }
    } else {
        // equal values throughout: one after another
        uint64_t last = ~0ull;
        for (n = 0; n < n_top; n++) {
            uint64_t best = 0;
            for (int j = tid; j < slots; j += nt) {
                const uint64_t c = cr[j];
                if (c < last && c > best) best = c;
            }
            best = wave_max_u64(best);
            __syncthreads();                           // the round before has been read
            if (lane == 0) red_c[wv] = best;
            __syncthreads();
            for (int w = 0; w < nw; w++) best = red_c[w] > best ? red_c[w] : best;
            if (tid == 0) write(n, lp_index(best), lp_value((uint32_t)(best >> 32)));
            last = best;
        }
    }
    // fewer than n_top above -inf: the rest in index order (-inf, NaN), then nothing
    if (n < n_top && wv == 0) {
        for (int i0 = 0; i0 < V && n < n_top; i0 += 64) {
            const int i = i0 + lane;
            const bool low = i < V && !(x[min(i, V - 1)] > -INFINITY);
            const uint64_t has = __ballot(low);
            const int at = n + __popcll(has & ((1ull << lane) - 1));
            if (low && at < n_top) write(at, i, x[i]);
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
struct lp_plan { int pieces, cap; size_t part_bytes, bytes; };
static lp_plan lp_plan_of(int64_t n_rows, int64_t V, int n_top) {
    lp_plan p;
    p.pieces = (int)((V + LP_PIECE - 1) / LP_PIECE);
    // n_top, the bound's slack, and the elements that are third or later in their lane: few but for large
    // n_top (64 of 2048: about 10)
    p.cap = n_top > 0 ? n_top + 12 + n_top * n_top / 100 : 0;
    p.part_bytes = align256((size_t)n_rows * p.pieces * sizeof(lp_part));
    p.bytes = p.part_bytes + (size_t)n_rows * p.pieces * p.cap * sizeof(uint64_t);
    return p;
}
static bool lp_shape_ok(int64_t n_rows, int64_t V, int n_top) {
    return n_rows >= 0 && n_rows <= (1 << 22) && V > 0 && V <= (1 << 30) && n_top >= 0 && n_top <= LP_MAX_TOP;
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
    uint64_t * cand = (uint64_t *)((uint8_t *)ws + p.part_bytes);
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
        uint64_t * cc = cand + r0 * p.pieces * p.cap;
#define PIECES(VEC)                                                                                                   \
    hipLaunchKernelGGL((k_lp_pieces<VEC>), grid, dim3(256), 0, st, lg, ld, nl, rw, (int)V, p.pieces, n_top, p.cap,  \
                       pp, cc)
        if (vec) PIECES(true);
        else PIECES(false);
#undef PIECES
        DFX_CHECK_LAUNCH("dfx_token_logprobs");
    }
    // Threads of a row's join: a wave where there are no candidates; with them, few rows take 16 waves
    // (8 candidates a thread, one round of loads), more rows 8 and 4 (256 rows of 62 pieces, 20 alternatives:
    // 39.8 us with 16 waves, 37.6 with 8, 37.9 with 4).
    const int waves = n_top == 0 ? 1 : n_rows <= 128 ? LP_JOIN / 64 : n_rows <= 512 ? 8 : 4;
    hipLaunchKernelGGL(k_lp_join, dim3((unsigned)n_rows), dim3(64 * waves), 0, st, logits, ld, n_logits, rows, (int)V,
                       p.pieces, n_top, p.cap, part, cand, tokens, n_tok, logprob, entropy, top_id, top_logprob);
    DFX_CHECK_LAUNCH("dfx_token_logprobs (join)");
    return DFX_OK;
}
