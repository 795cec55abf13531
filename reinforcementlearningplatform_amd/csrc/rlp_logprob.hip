// rlp_logprob.hip — log-probabilities of given tokens / discrete actions with the entropy and the
// top alternatives (rlp_token_logprob), and the gradient of the logits.
//
// One pass over the logits: with m the largest so far, s = sum 2^y and w = sum 2^y y of
// y = (l - m) log2(e) / temperature, rescaled when m grows,
//   logp = ln 2 (y_token - log2 s),   entropy = ln 2 (log2 s - w / s).
// In the loops y is one fma, l c - rnd(m c) with c = log2(e) / temperature: a logit's product is exact
// inside it, and what rounding m c put into every y alike (m c - rnd(m c)) is taken out of the sums at
// the end, so large logits lose nothing. Where m c is beyond 1e6 (a row of the type's lowest values, which
// is the uniform row it should be; a temperature near 0) y is formed from the difference l - m. Sums are
// f32.
#include "rlp_common.hpp"

namespace rlp {
namespace {

typedef uint32_t uintx4_any __attribute__((ext_vector_type(4), aligned(2)));  // at any element's address

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 32;
constexpr int kNoIndex = 0x7FFFFFFF;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// 16 bytes in one load at any element's address. Not as a memcpy, which might alias the stores: the gradient
// of 4096 x 32769 bf16 logits took 110 us with it, 97 so.
template <bool STREAM = false, typename T>
__device__ __forceinline__ void take16(T *to, const T *from) {
    const uintx4_any *p = (const uintx4_any *)from;
    const uintx4_any v = STREAM ? __builtin_nontemporal_load(p) : *p;
    __builtin_memcpy(to, &v, 16);
}

struct ScoreArgs {
    const void *logits;
    int64_t rows, stride;
    int vocab;
    const int64_t *tokens;
    float c, inv_t;  // log2(e) / temperature, 1 / temperature
    int k;
    float *logp, *entropy, *stats, *top_logp;
    int64_t *top_tokens;
    int slices, slice_len;  // parts of a row (one block each), joined by score_join_kernel
    float *parts;           // [rows][slices][3 + 2 k]: m, s, w, then (value, token) descending
};

struct Sums {
    float m, s, w;  // m -inf: nothing but -inf so far
};

// max(a, b, c) of numbers. With a NaN, which shows in the sums, it may be any of them: a quiet one is passed
// over, a signalling one hides those before it. As an instruction: fmaxf puts a canonicalising copy before
// every operand that comes from memory.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

// y = l c - mc of the logits of a row with maximum m; off: what is in every y beside (l - m) c
struct Shift {
    float mc, off;
    bool far;  // m c is large, its rounding too, or overflows: (l - m) c instead
    __device__ __forceinline__ Shift(float m, float c) {
        mc = m * c;
        far = !(fabsf(m) < 1e30f && fabsf(mc) < 1e6f);
        off = far ? 0.0f : __builtin_fmaf(m, c, -mc);
    }
};

__device__ __forceinline__ float base_of(float m) { return m == neg_inf() ? 0.0f : m; }

// The sums of two parts about their common maximum. -200: 2^-200 is 0 in f32, so a clamped y leaves
// 0 where 0 * -inf would leave NaN.
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float base = base_of(r.m);
    const float ya = (a.m - base) * c, yb = (b.m - base) * c;
    const float ea = __builtin_amdgcn_exp2f(ya), eb = __builtin_amdgcn_exp2f(yb);
    r.s = ea * a.s + eb * b.s;
    r.w = ea * (a.w + fmaxf(ya, -200.0f) * a.s) + eb * (b.w + fmaxf(yb, -200.0f) * b.s);
    return r;
}

// Of all lanes: first the maximum, then the sums about it.
__device__ __forceinline__ Sums join_wave(Sums v, float c) {
    float m = v.m;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float y = (v.m - base_of(m)) * c, e = __builtin_amdgcn_exp2f(y);
    v.w = e * __builtin_fmaf(fmaxf(y, -200.0f), v.s, v.w);
    v.s *= e;
    v.m = m;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        v.s += __shfl_xor(v.s, d);
        v.w += __shfl_xor(v.w, d);
    }
    return v;
}

// A value and its token as one whole number: larger for larger values, for equal ones (0 and -0 too)
// larger for the lower token.
__device__ __forceinline__ uint64_t rank_key(float v, int token) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ int key_token(uint64_t key) { return (int)~(uint32_t)key; }

// Row results from its sums (one lane). lt: the token's logit.
__device__ __forceinline__ float log2_sum(const Sums &v) {
    return v.s == 0.0f ? __builtin_inff() : __builtin_amdgcn_logf(v.s);
}
// not ln 2 times a log2, which overflows for a logit of the type's lowest value
__device__ __forceinline__ float logp_of(const Sums &v, float l, float inv_t) {
    return v.s == 0.0f ? neg_inf() : (l - base_of(v.m)) * inv_t - kLn2 * log2_sum(v);
}
__device__ __forceinline__ void write_row(const ScoreArgs &a, int64_t row, int64_t tok, float lt, const Sums &v) {
    const float l2 = log2_sum(v);
    const float ent = v.s == 0.0f ? 0.0f : kLn2 * (l2 - v.w / v.s);
    a.logp[row] = tok >= a.vocab ? __builtin_nanf("") : logp_of(v, lt, a.inv_t);
    a.entropy[row] = ent;
    if (a.stats) {
        a.stats[3 * row] = base_of(v.m);
        a.stats[3 * row + 1] = l2;
        a.stats[3 * row + 2] = ent;
    }
}
__device__ __forceinline__ void write_padded(const ScoreArgs &a, int64_t row) {
    a.logp[row] = a.entropy[row] = 0.0f;
    if (a.stats) a.stats[3 * row] = a.stats[3 * row + 1] = a.stats[3 * row + 2] = 0.0f;
    for (int i = 0; i < a.k; ++i) {
        a.top_logp[row * a.k + i] = 0.0f;
        a.top_tokens[row * a.k + i] = -1;
    }
}
__device__ __forceinline__ void write_top(const ScoreArgs &a, int64_t row, int i, const Sums &v, uint64_t key) {
    a.top_logp[row * a.k + i] = key ? logp_of(v, key_value(key), a.inv_t) : __builtin_nanf("");
    a.top_tokens[row * a.k + i] = key ? key_token(key) : -1;
}

__device__ __forceinline__ bool ahead(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// A wave's candidates for the k best, in LDS. push takes a lane's candidate where `pick`; select keeps
// the k best in order. Every key counts the keys above it, which places it at once: no chain from one
// candidate to the next, as inserting them one by one has (26 us of such chains for 8 rows' 20 best).
struct TopBuf {
    static constexpr int kCap = 128;
    uint64_t *key;
    int n, k;
    __device__ __forceinline__ void push(bool pick, uint64_t v) {
        const uint64_t mask = __ballot(pick);
        if (!mask) return;
        if (n > kCap - 64) select();
        if (pick) key[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = v;
        n += __popcll(mask);
    }
    __device__ __forceinline__ void select() {
        const int lane = threadIdx.x & 63;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // lanes read what other lanes wrote
        const uint64_t a = lane < n ? key[lane] : 0, b = lane + 64 < n ? key[lane + 64] : 0;
        int ra = 0, rb = 0;
        if (n <= 64) {
#pragma unroll 4
            for (int i = 0; i < n; ++i) ra += key[i] > a;
        } else {
#pragma unroll 4
            for (int i = 0; i < n; ++i) {
                const uint64_t o = key[i];
                ra += o > a, rb += o > b;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (lane < n && ra < k) key[ra] = a;
        if (lane + 64 < n && rb < k) key[rb] = b;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        n = min(n, k);
    }
};

// A value that k of a wave's 64 values reach: the k-th largest but for its last 16 bits, found bit by bit
// on whole numbers of the same order.
__device__ __forceinline__ float about_kth(float x, int k) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t key = b & 0x80000000u ? ~b : b | 0x80000000u;
    uint32_t lo = 0;
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = lo | 1u << bit;
        if (__popcll(__ballot(key >= t)) >= k) lo = t;
    }
    if (lo < 0x007FFFFFu) return neg_inf();  // below the number of -inf stand NaNs
    return __uint_as_float(lo & 0x80000000u ? lo ^ 0x80000000u : ~lo);
}

// Rows of up to E G logits, G lanes a row, all of it in registers: 16-byte vectors at any alignment, a lane's
// G vectors apart. Bound by instructions from 129 logits on, most of them the lanes' sums and the results,
// which a few rows a wave share: 2^20 rows of 300 bf16 logits in 199 us with 16 lanes a row, 412 with 64.
template <typename T, int G, int E = 8>
__global__ __launch_bounds__(256) void score_small_kernel(ScoreArgs a) {
    constexpr int VE = 16 / sizeof(T);
    const int g = threadIdx.x % G;
    auto token = [&](int i) { return ((i / VE) * G + g) * VE + i % VE; };  // of the lane's i-th logit
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (row >= a.rows) return;
    const int64_t tok = a.tokens[row];
    if (tok < 0) {
        if (g == 0) write_padded(a, row);
        return;
    }
    const T *l = (const T *)a.logits + row * a.stride;
    float x[E];
    Sums v = {neg_inf(), 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < E; c += VE) {
        T raw[VE];
        const int t0 = token(c);
        if (E > 8 && c * G >= a.vocab) {
#pragma unroll
            for (int e = 0; e < VE; ++e) raw[e] = (T)neg_inf();
        } else if (t0 + VE <= a.vocab) {
            take16(raw, l + t0);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) raw[e] = t0 + e < a.vocab ? l[t0 + e] : (T)neg_inf();
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            x[c + e] = to_f32(raw[e]);
            v.m = fmaxf(v.m, x[c + e]);
        }
    }
    const float lt = tok < a.vocab ? to_f32(l[tok]) : 0.0f;
#pragma unroll
    for (int d = G / 2; d > 0; d >>= 1) v.m = fmaxf(v.m, __shfl_xor(v.m, d));
    const float base = base_of(v.m);
#pragma unroll
    for (int c = 0; c < E; c += VE) {
        if (E > 8 && c * G >= a.vocab) break;
#pragma unroll
        for (int e = c; e < c + VE; ++e) {
            const float y = (x[e] - base) * a.c, p = __builtin_amdgcn_exp2f(y);
            v.s += p;
            v.w += p * fmaxf(y, -200.0f);
        }
    }
#pragma unroll
    for (int d = G / 2; d > 0; d >>= 1) {
        v.s += __shfl_xor(v.s, d);
        v.w += __shfl_xor(v.w, d);
    }
    if (g == 0) write_row(a, row, tok, lt, v);
    if constexpr (G == 64) {
        if (a.k > 2) {
            // a wave a row: what reaches a value that k of the lanes' largest reach, ranked in LDS (2^20 rows of 300
            // logits, 20 alternatives: 3.5 ms one after the other)
            __shared__ uint64_t top_s[4][TopBuf::kCap];
            TopBuf top = {top_s[threadIdx.x >> 6], 0, a.k};
            float most = neg_inf();
#pragma unroll
            for (int e = 0; e < E; ++e) most = x[e] > most ? x[e] : most;  // passes over every NaN
            const float lim = about_kth(most, a.k);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (!__any(x[e] >= lim)) continue;
                const int id = token(e);
                top.push(x[e] >= lim && id < a.vocab, rank_key(x[e], id));
            }
            top.select();
            if (g < a.k) write_top(a, row, g, v, g < top.n ? top.key[g] : 0);
            return;
        }
    }
    uint32_t open = 0;  // own tokens that are still to choose from
#pragma unroll
    for (int e = 0; e < E; ++e) open |= (token(e) < a.vocab && x[e] == x[e] ? 1u : 0u) << e;
    for (int i = 0; i < a.k; ++i) {
        float bv = neg_inf();
        int bi = kNoIndex;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if ((open >> e & 1) && ahead(x[e], token(e), bv, bi)) bv = x[e], bi = token(e);
#pragma unroll
        for (int d = G / 2; d > 0; d >>= 1) {
            const float ov = __shfl_xor(bv, d);
            const int oi = __shfl_xor(bi, d);
            if (ahead(ov, oi, bv, bi)) bv = ov, bi = oi;
        }
        if (bi != kNoIndex && bi / VE % G == g) open &= ~(1u << (bi / (VE * G) * VE + bi % VE));
        if (g == 0) write_top(a, row, i, v, bi == kNoIndex ? 0 : rank_key(bv, bi));
    }
}

// Longer rows: W waves a row, one pass. A wave takes tiles of 64 lanes x 2 16-byte vectors (any
// alignment), W tiles apart, the next tile loaded ahead: 6.0 TB/s of 4096 x 32768 bf16 logits, 5.3 of
// 4096 x 131071 (4 vectors: 6.3 and 5.5, but 65536 x 8193 takes 346 us for 245). Alternatives: each wave
// keeps its own list and a lower bound of the row's k-th value, shared between the row's waves through
// LDS; a tile is searched only where a vector's maximum reaches the bound.
template <typename T, int W, bool TOP, bool STREAM>
__global__ __launch_bounds__(256) void score_rows_kernel(ScoreArgs a) {
    constexpr int VE = 16 / sizeof(T), U = 2, TILE = 64 * VE * U;
    __shared__ float bound_s[4];
    __shared__ Sums sums_s[4];
    __shared__ int count_s[4];
    __shared__ uint64_t top_s[TOP ? 4 : 1][TopBuf::kCap];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = wave % W;
    const int64_t row = (int64_t)blockIdx.x * (4 / W) + wave / W;
    const int slice = blockIdx.y;
    if (TOP) {
        if (lane == 0 && w == 0) bound_s[wave] = neg_inf();
        if (W > 1) __syncthreads();
    }
    const int64_t tok = row < a.rows ? a.tokens[row] : -1;
    const bool padded = tok < 0;  // the same for all W waves of the row
    const T *l = (const T *)a.logits + row * a.stride;
    // STREAM: vectors begin at multiples of 16 bytes, so the first may begin before the row
    const int before = STREAM ? (uintptr_t)l / sizeof(T) % VE : 0, v0 = slice * a.slice_len - before;
    const int v1 = slice == a.slices - 1 ? a.vocab : v0 + a.slice_len;
    float lt = 0.0f;
    if (!padded && tok < a.vocab) lt = to_f32(l[tok]);
    Sums sum = {neg_inf(), 0.0f, 0.0f};
    TopBuf top = {top_s[TOP ? wave : 0], 0, a.k};
    float lv = neg_inf();  // an alternative is above (lv, li), which at least k logits of the row are not below
    int li = v1;
    volatile float *bound = &bound_s[wave / W * W];

    auto load = [&](T(&t)[U][VE], int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = at + (u * 64 + lane) * VE;
            if ((!STREAM || i >= 0) && i + VE <= v1) {
                take16<STREAM>(t[u], l + i);
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e) t[u][e] = (!STREAM || i + e >= 0) && i + e < v1 ? l[i + e] : (T)neg_inf();
            }
        }
    };
    if (!padded) {
        float off = 0.0f;  // what is in every y of the sums beside (l - sum.m) c
        auto tile = [&](const T(&cur)[U][VE], int at) {
            float x[U][VE], um[U], tm = neg_inf();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                um[u] = neg_inf();
#pragma unroll
                for (int e = 0; e < VE; e += 2) {
                    x[u][e] = to_f32(cur[u][e]), x[u][e + 1] = to_f32(cur[u][e + 1]);
                    um[u] = max3(um[u], x[u][e], x[u][e + 1]);
                }
            }
            tm = max3(tm, um[0], um[1]);
            {
                const float m = fmaxf(sum.m, tm), base = base_of(m);
                const Shift sh(base, a.c);
                // the sums so far move to the new maximum and its off, near or far (none so far: -inf)
                const float y0 = __builtin_fmaf(sum.m - base, a.c, sh.off - off);
                const float e0 = __builtin_amdgcn_exp2f(y0);
                sum.w = e0 * __builtin_fmaf(fmaxf(y0, -200.0f), sum.s, sum.w);
                sum.s *= e0;
                sum.m = m, off = sh.off;
                if (!__any(sh.far)) {
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            const float y = __builtin_fmaf(x[u][e], a.c, -sh.mc), p = __builtin_amdgcn_exp2f(y);
                            sum.s += p;
                            sum.w = __builtin_fmaf(p, fmaxf(y, -200.0f), sum.w);
                        }
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            const float y = __builtin_fmaf(x[u][e] - base, a.c, sh.off), p = __builtin_amdgcn_exp2f(y);
                            sum.s += p;
                            sum.w = __builtin_fmaf(p, fmaxf(y, -200.0f), sum.w);
                        }
                }
            }
            if (TOP) {
                if (__any(sum.s != sum.s)) {  // a NaN in the row so far: maxima that pass over it
                    tm = neg_inf();
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        um[u] = neg_inf();
#pragma unroll
                        for (int e = 0; e < VE; ++e) um[u] = x[u][e] > um[u] ? x[u][e] : um[u];
                        tm = fmaxf(tm, um[u]);
                    }
                }
                const float others = *bound;
                if (others > lv) lv = others, li = v1;
                const int many = __popcll(__ballot(tm >= lv));
                if (many > 0) {
                    // many lanes: at least k values reach what k of the lanes' maxima reach
                    if (many > a.k) {
                        const float reach = about_kth(tm, a.k);
                        if (reach > lv) lv = reach, li = v1;
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (!__any(um[u] >= lv)) continue;
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            if (!__any(x[u][e] >= lv)) continue;
                            const int id = at + (u * 64 + lane) * VE + e;
                            top.push(x[u][e] > lv || (x[u][e] == lv && (unsigned)id < (unsigned)li), rank_key(x[u][e], id));
                        }
                    }
                    if (top.n >= a.k + 8) {
                        top.select();
                        const uint64_t last = top.key[a.k - 1];
                        lv = key_value(last), li = key_token(last);
                        if (W > 1 && lane == 0 && lv > *bound) *bound = lv;
                    }
                }
            }
        };
        // two tiles in turn, the other one on its way
        T ta[U][VE], tb[U][VE];
        int at = v0 + w * TILE;
        if (at < v1) load(ta, at);
        for (; at < v1; at += 2 * W * TILE) {
            const int next = at + W * TILE;
            if (next < v1) load(tb, next);
            tile(ta, at);
            if (next >= v1) break;
            if (next + W * TILE < v1) load(ta, next + W * TILE);
            tile(tb, next);
        }
        {   // out of the sums what rounding m c put into every y
            const float e0 = __builtin_amdgcn_exp2f(-off);
            sum.w = e0 * __builtin_fmaf(-off, sum.s, sum.w);
            sum.s *= e0;
        }
        sum = join_wave(sum, a.c);
        if (TOP) top.select();
    }
    if (W > 1) {
        if (lane == 0) sums_s[wave] = sum;
        if (TOP && lane == 0) count_s[wave] = top.n;
        __syncthreads();
        if (w != 0) return;
        for (int o = 1; o < W; ++o) {
            sum = join(sum, sums_s[wave + o], a.c);
            if (!TOP) continue;
            const int n = count_s[wave + o];
            const uint64_t v = lane < n ? top_s[TOP ? wave + o : 0][lane] : 0;
            top.push(lane < n, v);
        }
        if (TOP) top.select();
    }
    if (row >= a.rows) return;
    if (a.slices > 1) {
        float *part = a.parts + (row * a.slices + slice) * (3 + 2 * a.k);
        if (lane == 0) part[0] = sum.m, part[1] = sum.s, part[2] = sum.w;
        if (TOP && lane < a.k) {  // 0: no further alternative
            const uint64_t v = lane < top.n ? top.key[lane] : 0;
            part[3 + 2 * lane] = __uint_as_float((uint32_t)v);
            part[4 + 2 * lane] = __uint_as_float((uint32_t)(v >> 32));
        }
        return;
    }
    if (padded) {
        if (lane == 0) write_padded(a, row);
        return;
    }
    if (lane == 0) write_row(a, row, tok, lt, sum);
    if (TOP && lane < a.k) write_top(a, row, lane, sum, lane < top.n ? top.key[lane] : 0);
}

// Joins the slices (at most 64) of a row: one wave a row, one slice a lane.
template <typename T>
__global__ __launch_bounds__(256) void score_join_kernel(ScoreArgs a) {
    __shared__ uint64_t top_s[4][TopBuf::kCap];
    const int lane = threadIdx.x & 63;
    const int64_t row = blockIdx.x * 4LL + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    const int64_t tok = a.tokens[row];
    if (tok < 0) {
        if (lane == 0) write_padded(a, row);
        return;
    }
    const float lt = tok < a.vocab ? to_f32(((const T *)a.logits)[row * a.stride + tok]) : 0.0f;
    const float *part = a.parts + (row * a.slices + min(lane, a.slices - 1)) * (3 + 2 * a.k);
    const bool on = lane < a.slices;
    Sums sum = {on ? part[0] : neg_inf(), on ? part[1] : 0.0f, on ? part[2] : 0.0f};
    sum = join_wave(sum, a.c);
    if (lane == 0) write_row(a, row, tok, lt, sum);
    if (a.k == 0) return;
    TopBuf top = {top_s[threadIdx.x >> 6], 0, a.k};
    uint64_t last = 0;
    for (int i = 0; i < a.k; ++i) {  // every slice's i-th entry
        const uint64_t v = on ? (uint64_t)__float_as_uint(part[4 + 2 * i]) << 32 | __float_as_uint(part[3 + 2 * i]) : 0;
        const bool pick = v > last;
        if (!__any(pick)) break;  // the slices' further entries are no better
        top.push(pick, v);
        if (top.n >= a.k + 8) {
            top.select();
            last = top.key[a.k - 1];
        }
    }
    top.select();
    if (lane < a.k) write_top(a, row, lane, sum, lane < top.n ? top.key[lane] : 0);
}

struct GradArgs {
    const void *logits;
    void *d_logits;
    int64_t rows, stride, d_stride;
    int vocab, span;  // span: logits of a row per block in y
    const int64_t *tokens;
    float c, inv_t;
    const float *stats, *d_logp, *d_entropy;
};

// d logit = (g (1[token] - p) - h p (log p + entropy)) / temperature; L lanes a row, 16 bytes each. With
// y = log2 p: -p (A + B y) of the row's A = g + h entropy and B = h ln 2, and g more at the token.
template <typename T, bool STREAM, bool ALIGNED, int U>
__global__ __launch_bounds__(256) void score_grad_kernel(GradArgs a, int L) {
    constexpr int VE = 16 / sizeof(T);
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (row >= a.rows) return;
    const int64_t tok = a.tokens[row];
    const bool padded = tok < 0;
    const T *l = (const T *)a.logits + row * a.stride;
    T *d = (T *)a.d_logits + row * a.d_stride;
    // U vectors on their way before the row's numbers are waited for
    // ALIGNED: vectors begin at multiples of 16 bytes of d, so the first may begin before the row
    const int before = ALIGNED ? (int)((uintptr_t)d / sizeof(T) % VE) : 0;
    const int v0 = (int)blockIdx.y * a.span - before, v1 = min(a.vocab, v0 + a.span);
    for (int i0 = v0 + threadIdx.x % L * VE; i0 < v1; i0 += U * L * VE) {
        T x[U][VE] = {};
        if (!padded) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * L * VE;
                if ((!ALIGNED || i >= 0) && i + VE <= v1) {
                    take16(x[u], l + i);
                } else {
#pragma unroll
                    for (int e = 0; e < VE; ++e) x[u][e] = (!ALIGNED || i + e >= 0) && i + e < v1 ? l[i + e] : (T)neg_inf();
                }
            }
        }
        const float m = a.stats[3 * row];
        float g = a.d_logp ? a.d_logp[row] * a.inv_t : 0.0f;
        const float h = a.d_entropy ? a.d_entropy[row] * a.inv_t : 0.0f;
        const Shift sh(m, a.c);
        const float l2 = a.stats[3 * row + 1] + sh.off;
        if (l2 == __builtin_inff()) g = 0.0f;  // nothing but -inf
        if (tok >= a.vocab) g = __builtin_nanf("");
        const float A = __builtin_fmaf(h, a.stats[3 * row + 2], g), B = h * kLn2;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * L * VE;
            if (i >= v1) break;
            float v[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float xe = to_f32(x[u][e]);
                const float y = (sh.far ? __builtin_fmaf(xe - m, a.c, sh.off) : __builtin_fmaf(xe, a.c, -sh.mc)) - l2;
                v[e] = -__builtin_amdgcn_exp2f(y) * __builtin_fmaf(B, fmaxf(y, -200.0f), A);
            }
            if (tok - i >= 0 && tok - i < VE) {
#pragma unroll
                for (int e = 0; e < VE; ++e) v[e] += tok - i == e ? g : 0.0f;
            }
            T r[VE];
#pragma unroll
            for (int e = 0; e < VE; ++e) r[e] = (T)(padded ? 0.0f : v[e]);
            if ((!ALIGNED || i >= 0) && i + VE <= v1) {
                uintx4_any out;
                __builtin_memcpy(&out, r, 16);
                if (STREAM) __builtin_nontemporal_store(out, (uintx4_any *)(d + i));
                else *(uintx4_any *)(d + i) = out;
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    if ((!ALIGNED || i + e >= 0) && i + e < v1) d[i + e] = r[e];
            }
        }
    }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
constexpr int kSmallVocab = 512;

// Rows a block takes: 256 threads over the lanes of a row. A launch has at most 2^24 - 1 such blocks (2^32 - 1
// threads along x).
bool rows_fit(int64_t rows, int lanes) { return rows * lanes <= 256LL * ((1 << 24) - 1); }
int score_lanes(int64_t vocab) { return vocab <= 8192 ? 64 : 256; }
// Lanes of a row's gradient, up to four vectors a lane (300 bf16 logits: 167 us of 2^19 rows, 268 with one), two
// up to 64 logits (2^20 rows of 64 f32: 98 us for 121). At least 256 bytes of a row at a time beyond that, as
// stores past the caches of less fill no line (2^20 rows of 100 bf16: 122 us for 220), and 256 lanes, not 128
// (65536 rows of 2000 f32: 175 us for 204).
int grad_lanes(int64_t vocab, int dtype) {
    int L = vocab <= 64 ? 1 : 16;
    while (L < 256 && L * (dtype == RLP_F32 ? 4 : 8) * (vocab <= 64 ? 2 : 4) < vocab) L *= 2;
    return L == 128 ? 256 : L;
}

// Few long rows: each over several blocks of at least one tile per wave.
int slices_of(int64_t rows, int64_t vocab, int dtype, int *len) {
    *len = (int)vocab;
    if (rows < 1 || rows >= 512 || vocab <= kSmallVocab) return 1;
    const int64_t tile = 4 * (dtype == RLP_F32 ? 512 : 1024);  // four waves' tiles
    int64_t want = (1024 + rows - 1) / rows;
    const int64_t most = (vocab + tile - 1) / tile;
    if (want > most) want = most;
    if (want > 64) want = 64;
    if (want <= 1) return 1;
    const int64_t each = ((vocab + want - 1) / want + tile - 1) / tile * tile;
    *len = (int)each;
    return (int)((vocab + each - 1) / each);
}

template <typename T>
void launch_score(const ScoreArgs &a, hipStream_t s) {
    auto blocks = [&](int per) { return (unsigned)((a.rows + per - 1) / per); };
    // logits of twice the 256 MB last-level cache and more: loads past it and aligned, as vectors over two cache
    // lines cost time then (bf16, 4096 x 131071 254 -> 205 us, with 8 alternatives 268 -> 213; 16384 x 32769
    // 226 -> 177). Fewer stay in the cache for the gradient, and are summed in an order that does not
    // depend on a row's address.
    const bool past = a.rows * a.vocab * (int64_t)sizeof(T) > (512LL << 20);
    auto rows = [&](auto kept, auto stream, dim3 grid) { (past ? stream : kept)<<<grid, 256, 0, s>>>(a); };
    if (a.vocab <= 32) score_small_kernel<T, 2, 16><<<blocks(128), 256, 0, s>>>(a);
    else if (a.vocab <= 128) score_small_kernel<T, 4, 32><<<blocks(64), 256, 0, s>>>(a);
    else if (a.vocab <= 256 && a.k <= 2) score_small_kernel<T, 8, 32><<<blocks(32), 256, 0, s>>>(a);
    else if (a.vocab <= kSmallVocab && a.k <= 2) score_small_kernel<T, 16, 32><<<blocks(16), 256, 0, s>>>(a);
    else if (a.vocab <= kSmallVocab) score_small_kernel<T, 64><<<blocks(4), 256, 0, s>>>(a);
    else if (a.slices == 1 && (a.vocab <= 8192 || (a.rows >= 2048 && (a.k > 0 || a.vocab <= 16384)))) {
        // a wave a row: short rows, and rows enough to fill the card where a search for alternatives begins
        // and ends in every wave (bf16, 16384 x 32769, 8 alternatives: 226 us, four waves a row 296; without,
        // 65536 x 8193 takes 189 us so and 245 with four, 4096 x 32768 49 and 45)
        if (a.k) rows(score_rows_kernel<T, 1, true, false>, score_rows_kernel<T, 1, true, true>, blocks(4));
        else rows(score_rows_kernel<T, 1, false, false>, score_rows_kernel<T, 1, false, true>, blocks(4));
    } else {
        const dim3 grid((unsigned)a.rows, a.slices);
        if (a.k) rows(score_rows_kernel<T, 4, true, false>, score_rows_kernel<T, 4, true, true>, grid);
        else rows(score_rows_kernel<T, 4, false, false>, score_rows_kernel<T, 4, false, true>, grid);
        if (a.slices > 1) score_join_kernel<T><<<blocks(4), 256, 0, s>>>(a);
    }
}

template <typename T>
void launch_grad(GradArgs a, hipStream_t s) {
    constexpr int VE = 16 / sizeof(T);
    const int L = grad_lanes(a.vocab, VE == 4 ? RLP_F32 : RLP_BF16);
    const int64_t blocks = (a.rows + 256 / L - 1) / (256 / L);
    // a block takes 4 vectors a lane of a long row; at most 65535 blocks in y
    a.span = 256 * VE * 4;
    const int64_t most = (int64_t)a.vocab + VE - 1;  // with what lies before the row
    int64_t ny = (most + a.span - 1) / a.span;
    while (ny > 65535) a.span *= 2, ny = (most + a.span - 1) / a.span;
    // logits and gradient beyond the 256 MB last-level cache: stores past it (4096 x 32768 bf16 102 us for
    // 153), else the gradient stays there for what reads it next. Twice that and more also aligned, where a row's
    // ends cost less than vectors over two cache lines (16384 x 32769 bf16 450 us for 483; 4096 x 32769 97 for 96)
    const dim3 grid((unsigned)blocks, (unsigned)ny);
    const int64_t bytes = a.rows * a.vocab * (int64_t)sizeof(T);
    const bool past = bytes > (128LL << 20);
    if (L * VE >= a.vocab) {
        if (past) score_grad_kernel<T, true, false, 1><<<grid, 256, 0, s>>>(a, L);
        else score_grad_kernel<T, false, false, 1><<<grid, 256, 0, s>>>(a, L);
    } else {
        if (L == 256 && bytes > (512LL << 20)) score_grad_kernel<T, true, true, 4><<<grid, 256, 0, s>>>(a, L);
        else if (past) score_grad_kernel<T, true, false, 4><<<grid, 256, 0, s>>>(a, L);
        else score_grad_kernel<T, false, false, 4><<<grid, 256, 0, s>>>(a, L);
    }
}

int check_rows(const char *who, int dtype, int64_t rows, int64_t vocab, int64_t stride, float temperature) {
    RLP_REQUIRE(dtype == RLP_F32 || dtype == RLP_F16 || dtype == RLP_BF16, "%s: dtype %d", who, dtype);
    RLP_REQUIRE(rows >= 0 && rows <= 0x7FFFFFFFLL, "%s: %lld rows", who, (long long)rows);
    RLP_REQUIRE(vocab >= 1 && vocab <= 0x7FF00000LL, "%s: vocab %lld", who, (long long)vocab);
    RLP_REQUIRE(stride >= 0, "%s: row stride %lld", who, (long long)stride);
    RLP_REQUIRE(temperature >= 1e-30f && temperature <= 1e30f, "%s: temperature %g (1e-30 to 1e30)", who,
                temperature);
    return RLP_OK;
}

}  // namespace
}  // namespace rlp

using namespace rlp;

extern "C" {

int64_t rlp_token_logprob_workspace_bytes(int64_t rows, int64_t vocab, int top_k, int dtype) {
    const int rc = check_rows("rlp_token_logprob_workspace_bytes", dtype, rows, vocab, 0, 1.0f);
    if (rc != RLP_OK) return rc;
    RLP_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= vocab,
                "rlp_token_logprob_workspace_bytes: top_k %d (0 to min(vocab, %d))", top_k, kMaxTop);
    int len;
    const int n = slices_of(rows, vocab, dtype, &len);
    return n > 1 ? rows * n * (3 + 2 * top_k) * 4 : 0;
}

int rlp_token_logprob(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                      const int64_t *tokens, float temperature, int top_k, float *logp, float *entropy,
                      float *stats, float *top_logp, int64_t *top_tokens, void *workspace,
                      int64_t workspace_bytes, rlp_stream_t stream) {
    take_pending();
    const int rc = check_rows("rlp_token_logprob", dtype, rows, vocab, row_stride, temperature);
    if (rc != RLP_OK) return rc;
    RLP_REQUIRE(top_k >= 0 && top_k <= kMaxTop && top_k <= vocab,
                "rlp_token_logprob: top_k %d (0 to min(vocab, %d))", top_k, kMaxTop);
    if (rows == 0) return RLP_OK;
    RLP_REQUIRE(logits && tokens && logp && entropy && (top_k == 0 || (top_logp && top_tokens)),
                "rlp_token_logprob: null argument");
    RLP_REQUIRE(rows_fit(rows, score_lanes(vocab)), "rlp_token_logprob: %lld rows of %lld logits are too many for one launch",
                (long long)rows, (long long)vocab);
    const int64_t need = rlp_token_logprob_workspace_bytes(rows, vocab, top_k, dtype);
    RLP_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
                "rlp_token_logprob: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)need);
    ScoreArgs a = {};
    a.logits = logits, a.rows = rows, a.stride = row_stride, a.vocab = (int)vocab, a.tokens = tokens;
    a.c = (float)(1.4426950408889634 / (double)temperature), a.inv_t = 1.0f / temperature, a.k = top_k;
    a.logp = logp, a.entropy = entropy, a.stats = stats, a.top_logp = top_logp, a.top_tokens = top_tokens;
    a.slices = slices_of(rows, vocab, dtype, &a.slice_len);
    a.parts = (float *)workspace;
    hipStream_t s = as_stream(stream);
    if (dtype == RLP_F32) launch_score<float>(a, s);
    else if (dtype == RLP_F16) launch_score<_Float16>(a, s);
    else launch_score<__bf16>(a, s);
    RLP_CHECK_LAUNCH("rlp_token_logprob");
    return RLP_OK;
}

int rlp_token_logprob_backward(const void *logits, int dtype, int64_t rows, int64_t vocab,
                               int64_t row_stride, const int64_t *tokens, float temperature,
                               const float *stats, const float *d_logp, const float *d_entropy,
                               void *d_logits, int64_t d_row_stride, rlp_stream_t stream) {
    take_pending();
    const int rc = check_rows("rlp_token_logprob_backward", dtype, rows, vocab, row_stride, temperature);
    if (rc != RLP_OK) return rc;
    RLP_REQUIRE(rows <= 1 || d_row_stride >= vocab, "rlp_token_logprob_backward: rows of d_logits overlap");
    if (rows == 0) return RLP_OK;
    RLP_REQUIRE(logits && tokens && stats && d_logits, "rlp_token_logprob_backward: null argument");
    RLP_REQUIRE(rows_fit(rows, grad_lanes(vocab, dtype)),
                "rlp_token_logprob_backward: %lld rows of %lld logits are too many for one launch", (long long)rows,
                (long long)vocab);
    GradArgs a = {};
    a.logits = logits, a.d_logits = d_logits, a.rows = rows, a.stride = row_stride, a.d_stride = d_row_stride;
    a.vocab = (int)vocab, a.tokens = tokens;
    a.c = (float)(1.4426950408889634 / (double)temperature), a.inv_t = 1.0f / temperature;
    a.stats = stats, a.d_logp = d_logp, a.d_entropy = d_entropy;
    hipStream_t s = as_stream(stream);
    if (dtype == RLP_F32) launch_grad<float>(a, s);
    else if (dtype == RLP_F16) launch_grad<_Float16>(a, s);
    else launch_grad<__bf16>(a, s);
    RLP_CHECK_LAUNCH("rlp_token_logprob_backward");
    return RLP_OK;
}

}  // extern "C"
