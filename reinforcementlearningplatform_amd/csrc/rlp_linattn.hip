// rlp_linattn.hip — linear attention with one decay per head (rlp_linear_attention*): the memory of
// a sequence policy over rollout segments and prompts, forward, backward and for one token.
//
//   S_t = lam_h S_{t-1} + k_t v_t^T     (S_{t-1} dropped where an episode begins at token t)
//   o_t = scale * q_t S_t
//
// Every direction is the same sum with its operands in other roles,
//   out_i = sum_{j <= i} lam^(i-j) (x_i . y_j) z_j   over the pairs of one episode:
//   forward  x = q,  y = k,  z = v;            dq  x = do, y = v,  z = k;
//   dv       x = k,  y = q,  z = do, reversed; dk  x = v,  y = do, z = q, reversed in time,
// so one kernel computes all of them. It walks a sequence in chunks: within a chunk the decayed,
// masked products P = X Y^T times Z, before it lam^(i+1) x_i S with the state S = sum_j y_j z_j^T
// of what came before, S [dx][dz] held in the MFMA accumulators of the block for the whole walk.
#include <type_traits>

#include "rlp_common.hpp"

namespace rlp {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned short ushortx2 __attribute__((ext_vector_type(2)));
typedef uintx4 uintx4_any __attribute__((aligned(2)));  // 16 bytes at any element's address

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(__bf16 x) { return (float)x; }

// One walk over the sequences: operand strides in elements (batch, token, head), D contiguous.
struct WalkArgs {
    const void *x, *y, *z;
    void *out;               // nullable: only the state is wanted
    int64_t xb, xt, xh, yb, yt, yh, zb, zt, zh, ob, ot, oh;
    int gx, gy, gz;          // states per x / y / z head (shared heads)
    const float *log_decay;  // [H]
    const uint8_t *reset;    // nullable
    int64_t rb, rt;
    const int32_t *lengths;  // nullable
    const float *init;       // nullable: state in; element (a, n) at bh * dx * dz + a * ia + n * in
    float *fin;              // nullable: state out, same layout as init
    int64_t ia, in;
    float *seg;              // [B * H][nseg][dx * dz] states of the segments (nseg > 1), element (a, n) at
    int64_t sa, sn;          //   a * sa + n * sn
    float *segf;             // [B * H][nseg] the segment's decay, -1 where it holds a reset
    int B, T, H, dx, dz;
    int nseg, seglen;
    int mode;                // 0 one walk, 1 only the segments' own states, 2 outputs from seg
    int rev;                 // walk from the last token to the first
    int e0;                  // decay of the carried state at a chunk's token i: lam^(i + e0)
    float s1, s2, s3;        // factors of P, of x_i S and of the state's increments
    int out_f32;             // out is f32 (a partial of a shared head), not T
};

// Whether the walk's link into position p is cut (not 0): walking forward by an episode that begins at
// p's token, backward by one that begins at the token behind. As it was loaded, to be waited for later.
__device__ __forceinline__ uint32_t cut_at(const WalkArgs &a, int b, int p, int len) {
    if (!a.reset || (a.rev && p == 0)) return 0;
    return a.reset[b * a.rb + (int64_t)(a.rev ? len - p : p) * a.rt];
}

// log2 lam; a log_decay of -inf (no memory) becomes a finite number, so that lam^0 is 1 and lam^1 is 0
__device__ __forceinline__ float log2_decay(float log_decay) {
    const float l = log_decay * kLog2e;
    return l < -1e6f ? -1e6f : l;  // a NaN stays one
}
__device__ __forceinline__ float decay_pow(float lam2, int n) {
    return __builtin_amdgcn_exp2f(lam2 * (float)n);
}

// The value as if computed anew: keeps what a loop derives from lane numbers and powers inside the loop.
// Hoisted, those invariants (addresses, comparisons, products of powers) took 200 registers more than a
// wave has and went to scratch.
template <typename T>
__device__ __forceinline__ T anew(T v) {
    asm volatile("" : "+v"(v));
    return v;
}

// The sequence of a grid's slot-th H blocks, of up to 64 by their lengths. A sequence's chunks follow one another,
// so that the longest ends last. Up to two blocks a CU all start at once: the longest get a CU alone, the
// others share theirs with the shortest, the longer with the shorter. More start in order, the longest
// first. 24 of 256 .. 2047 tokens with 16 heads, 128 x 128 bf16: 213 us, 238 as they stand (221 longest
// first); 60 of 125 .. 1000 with 8, 64 x 64 f32: 112 for 140.
__device__ __forceinline__ int by_length(const WalkArgs &a, int slot) {
    if (!a.lengths || a.nseg > 1 || a.B > 64 || gridDim.x <= 256) return slot;
    const int lane = threadIdx.x & 63, n = lane < a.B ? a.lengths[lane] : 0;
    int rank = 0;
    for (int j = 0; j < a.B; ++j) {
        const int m = __builtin_amdgcn_readlane(n, j);
        rank += m > n || (m == n && j < lane);
    }
    if (gridDim.x <= 512) {
        const int first = 256 / a.H, shared = min(a.B - first, first);  // sequences in the CUs' first places
        slot = slot < shared ? slot + first - shared : slot < first ? slot - shared : a.B - 1 - (slot - first);
    }
    return __builtin_ctzll(__ballot(lane < a.B && rank == slot));
}

typedef floatx4 floatx4_any __attribute__((aligned(4)));

// A wave's 16 columns of a state, rows row0 + 16 at .. + 3 a lane. Of a transposed one these four are 16 bytes;
// and without the masks of narrower states the loads are all in flight together (1611 x 16 states of 64 x 128
// through training on 6 tokens 1158 us for 1556).
template <int DZ, int N>
__device__ __forceinline__ void load_state(floatx4 (&S)[N], const float *src, int64_t ia, int64_t in, int dx, int dz,
                                           int row0, int col) {
    if (src && dx == 16 * N && dz == DZ) {
        if (ia == 1) {
#pragma unroll
            for (int at = 0; at < N; ++at) S[at] = *(const floatx4_any *)(src + col * in + row0 + 16 * at);
        } else {
#pragma unroll
            for (int at = 0; at < N; ++at)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[at][r] = src[(row0 + 16 * at + r) * ia + col * in];
        }
        return;
    }
#pragma unroll
    for (int at = 0; at < N; ++at)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + 16 * at + r;
            S[at][r] = src && row < dx && col < dz ? src[row * ia + col * in] : 0.0f;
        }
}

// Highest set bit of m at or below i (the chunk position where i's episode begins), -1: none.
__device__ __forceinline__ int begin_of(uint32_t m, int i) {
    const uint32_t below = m & (0xFFFFFFFFu >> (31 - i));
    return below ? 31 - __builtin_clz(below) : -1;
}

// 32 rows of D columns of T on their way from global memory to f32 rows in LDS: 16 bytes a thread and
// step at any alignment; rows >= n and columns >= d become 0.
template <typename T, int D, int NT>
struct Rows32 {
    static constexpr int VE = 16 / sizeof(T), VR = D / VE, N = (32 * VR + NT - 1) / NT;
    uintx4 v[N];
    __device__ __forceinline__ void load(const T *src, int64_t st, int n, int d, unsigned tid) {
        const int row = tid / VR, c = tid % VR * VE;
        const T *p = src + row * st + c;
        if (n == 32 && d == D && 32 * VR % NT == 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = *(const uintx4_any *)(p + k * (NT / VR) * st);
            return;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = (uintx4){0, 0, 0, 0};
            if (row + k * (NT / VR) >= n) continue;
            const T *pk = p + k * (NT / VR) * st;
            if (c + VE <= d) {
                v[k] = *(const uintx4_any *)pk;
            } else if constexpr (sizeof(T) == 4) {
                if (c < d) v[k][0] = *(const uint32_t *)pk;
                if (c + 1 < d) v[k][1] = *(const uint32_t *)(pk + 1);
                if (c + 2 < d) v[k][2] = *(const uint32_t *)(pk + 2);
            } else {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (c + e < d) v[k][e / 2] |= (uint32_t)__builtin_bit_cast(unsigned short, pk[e]) << (16 * (e & 1));
            }
        }
    }
    // Also says whether a value is inf or NaN.
    __device__ __forceinline__ bool store(float (*dst)[D + 4], unsigned tid) const {
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const unsigned id = k * NT + tid;
            const int row = id / VR, c = id % VR * VE;
            if (32 * VR % NT != 0 && row >= 32) break;
            float f[VE];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < VE; ++e) f[e] = __uint_as_float(v[k][e]);
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    f[e] = to_f32(__builtin_bit_cast(T, (unsigned short)(v[k][e / 2] >> (16 * (e & 1)))));
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) most = max(most, __float_as_uint(f[e]) & 0x7FFFFFFFu);
#pragma unroll
            for (int e = 0; e < VE; e += 4)
                *(floatx4 *)&dst[row][c + e] = (floatx4){f[e], f[e + 1], f[e + 2], f[e + 3]};
        }
        return most >= 0x7F800000u;
    }
};

__device__ __forceinline__ floatx4 mfma_f32(float a, float b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// The walk in exact f32 products (v_mfma_f32_16x16x4_f32), 32 tokens a chunk, for every type. A block
// of NW waves owns one (batch, head, segment); wave w owns columns [16 w, 16 w + 16) of the state and
// the output, so no wave ever needs another's state.
//
// A 16x16 accumulator holds rows 4 q + r (q = lane >> 4) of column lane & 15 in register r, and an
// operand one value of row q of four. With the order of a contraction free, register r of an
// accumulator is the operand of rows q -> 4 q + r as it stands: S goes from accumulator to operand
// without leaving its wave, and so does P, computed transposed as Y X^T and shared out over the waves.
//
// Bound by HBM and matrix instructions together up to 64 x 64 (4096 x 4 sequences of 64 tokens: 1.6 GB in
// 343 us, 4.7 TB/s, with 50 % of the cycles in f32 products), by the latter at 128 x 128 (16 x 16 of 4096:
// 858 us for 2.15 GB, 100 TF/s). 32 columns a wave with 32x32 products, at one wave a SIMD, took three
// times as long (that training segment 4.86 ms for 1.68).
template <typename T, int DXB, int NW>
__global__ __launch_bounds__(64 * NW, 32 * DXB <= 32 * NW ? 4 : 2) void la_walk_kernel(WalkArgs a) {
    constexpr int C = 32, DX = 32 * DXB, DZ = 16 * NW, NT = 64 * NW;
    __shared__ __align__(16) float xs[C][DX + 4];
    __shared__ __align__(16) float ys[C][DX + 4];
    __shared__ __align__(16) float zs[C][DZ + 4];
    __shared__ __align__(16) floatx4 ps[3][64];
    __shared__ __align__(16) float into_s[C], from_s[C];
    __shared__ int bad_s, first_s;
    unsigned tid = threadIdx.x;
    int lane = tid & 63, q = lane >> 4, l15 = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % a.H, b = by_length(a, blockIdx.x / a.H), g = blockIdx.y;
    const int64_t bh = (int64_t)b * a.H + h;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    const int p0 = g * a.seglen, p1 = min(len, p0 + a.seglen);
    const float lam2 = log2_decay(a.log_decay[h]);
    const int64_t tok0 = a.rev ? len - 1 : 0, dir = a.rev ? -1 : 1;
    const T *x = (const T *)a.x + b * a.xb + (h / a.gx) * a.xh + tok0 * a.xt;
    const T *y = (const T *)a.y + b * a.yb + (h / a.gy) * a.yh + tok0 * a.yt;
    const T *z = (const T *)a.z + b * a.zb + (h / a.gz) * a.zh + tok0 * a.zt;
    const int64_t out0 = b * a.ob + h * a.oh + tok0 * a.ot;
    const bool want_out = a.mode != 1 && a.out;
    const int c0 = 16 * w;
    int col = c0 + l15;

    floatx4 S[2 * DXB];
    {
        const float *src = nullptr;
        int64_t ia = a.ia, in = a.in;
        if (a.mode == 0 && a.init) src = a.init + (int64_t)bh * a.dx * a.dz;
        if (a.mode == 2) src = a.seg + ((int64_t)bh * a.nseg + g) * a.dx * a.dz, ia = a.sa, in = a.sn;
        load_state<DZ>(S, src, ia, in, a.dx, a.dz, 4 * q, col);
    }
    bool seg_cut = false;
    if (tid == 0) bad_s = -1;
    Rows32<T, DX, NT> rx, ry;
    Rows32<T, DZ, NT> rz;
    const int64_t xs_t = dir * a.xt, ys_t = dir * a.yt, zs_t = dir * a.zt;
    x += p0 * xs_t, y += p0 * ys_t, z += p0 * zs_t;  // of the chunk to load next, at position `ahead`
    int ahead = p0;
    uint32_t cut = 0;
    auto load = [&](int n) {
        cut = lane < n ? cut_at(a, b, ahead + lane, len) : 0;
        if (want_out) rx.load(x, xs_t, n, a.dx, tid);
        ry.load(y, ys_t, n, a.dx, tid);
        rz.load(z, zs_t, n, a.dz, tid);
    };
    auto step = [&](int n) { x += n * xs_t, y += n * ys_t, z += n * zs_t, ahead += n; };
    if (p0 < p1) load(min(C, p1 - p0));
    for (int pos = p0; pos < p1;) {
        tid = anew(tid), lane = tid & 63, q = lane >> 4, l15 = lane & 15, col = c0 + l15;
        int n = min(C, p1 - pos);
        // what a token takes from the state that comes in, and what it leaves to the one that goes out: only
        // tokens of the episodes that came in and that goes out
        auto factors = [&](uint32_t cuts) {
            if (tid < C) {
                const int i = tid;
                into_s[i] = cuts & (~0u >> (31 - i)) ? 0.0f : a.s2 * decay_pow(lam2, i + a.e0);
                from_s[i] = i < n && i >= begin_of(cuts, n - 1) ? a.s3 * decay_pow(lam2, n - a.e0 - i) : 0.0f;
            }
        };
        uint32_t cuts = (uint32_t)__ballot(cut != 0);
        __syncthreads();  // the chunk before is done with the tiles
        if (want_out) rx.store(xs, tid);
        bool bad = ry.store(ys, tid);
        bad |= rz.store(zs, tid);
        if (bad) bad_s = pos;
        factors(cuts);
        step(n);
        if (ahead < p1) load(min(C, p1 - ahead));
        __syncthreads();
        if (bad_s == pos) {
            // An inf or NaN would reach rows it has no part in, through 0 * x in the products: the
            // chunk ends before a row that holds one, and such a row's chunk before the next episode.
            if (tid == 0) first_s = n;
            __syncthreads();
            bool head = false;
            for (int j = 0; j < n; ++j) {
                bool here = false;
                for (unsigned c = tid; c < DX; c += NT) here |= (__float_as_uint(ys[j][c]) & 0x7F800000u) == 0x7F800000u;
                for (unsigned c = tid; c < DZ; c += NT) here |= (__float_as_uint(zs[j][c]) & 0x7F800000u) == 0x7F800000u;
                if (j == 0) head = __syncthreads_or(here);
                else if (here) atomicMin(&first_s, j);
            }
            __syncthreads();
            step(-n);
            n = first_s;
            if (head && (cuts & ~1u)) n = min(n, (int)__builtin_ctz(cuts & ~1u));
            cuts &= ~0u >> (32 - n);
            for (unsigned id = tid; id < (C - n) * DX; id += NT) ys[n + id / DX][id % DX] = 0.0f;
            for (unsigned id = tid; id < (C - n) * DZ; id += NT) zs[n + id / DZ][id % DZ] = 0.0f;
            step(n);
            if (ahead < p1) load(min(C, p1 - ahead));
            factors(cuts);
            __syncthreads();
        }
        floatx4 zv[2], O[2];  // zv: z rows 16 jt + 4 q + r of the wave's columns
#pragma unroll
        for (int jt = 0; jt < 2; ++jt)
#pragma unroll
            for (int r = 0; r < 4; ++r) zv[jt][r] = zs[16 * jt + 4 * q + r][col];
        if (want_out) {
            // P^T = s1 lam^(i-j) Y X^T of the pairs j <= i of one episode: tiles (j, i) on and above the diagonal
            for (int t = w; t < 3; t += NW) {
                const int it = t > 0, jt = t > 1;
                floatx4 P = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int at = 0; at < 2 * DXB; ++at) {
                    const floatx4 yv = *(const floatx4 *)&ys[16 * jt + l15][16 * at + 4 * q];
                    const floatx4 xv = *(const floatx4 *)&xs[16 * it + l15][16 * at + 4 * q];
#pragma unroll
                    for (int r = 0; r < 4; ++r) P = mfma_f32(yv[r], xv[r], P);
                }
                const int d0 = 16 * (it - jt) + l15 - 4 * q;
                const int j0 = cuts ? begin_of(cuts, 16 * it + l15) - 16 * jt - 4 * q : -C;  // of i's episode
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    P[r] *= a.s1 * decay_pow(lam2, d0 - r);
                    P[r] = r <= d0 && r >= j0 ? P[r] : 0.0f;  // 0 whatever stood there
                }
                ps[t][lane] = P;
            }
            // x S, decayed to each row
#pragma unroll
            for (int it = 0; it < 2; ++it) O[it] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int at = 0; at < 2 * DXB; ++at)
#pragma unroll
                for (int it = 0; it < 2; ++it) {
                    const floatx4 xv = *(const floatx4 *)&xs[16 * it + l15][16 * at + 4 * q];
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[it] = mfma_f32(xv[r], S[at][r], O[it]);
                }
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const floatx4 f = *(const floatx4 *)&into_s[16 * it + 4 * q];
#pragma unroll
                for (int r = 0; r < 4; ++r) O[it][r] *= f[r];
                if (cuts) {  // not 0 * inf
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[it][r] = f[r] != 0.0f ? O[it][r] : 0.0f;
                }
            }
            __syncthreads();  // P is there
            const floatx4 p00 = ps[0][lane], p01 = ps[1][lane], p11 = ps[2][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                O[0] = mfma_f32(p00[r], zv[0][r], O[0]);
                O[1] = mfma_f32(p01[r], zv[0][r], O[1]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) O[1] = mfma_f32(p11[r], zv[1][r], O[1]);
            if (col < a.dz) {
                const int64_t at0 = out0 + (pos + 4 * q) * dir * a.ot + col;
#pragma unroll
                for (int it = 0; it < 2; ++it)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (16 * it + 4 * q + r >= n) continue;
                        const int64_t at = at0 + (16 * it + r) * dir * a.ot;
                        if (a.out_f32) ((float *)a.out)[at] = O[it][r];
                        else ((T *)a.out)[at] = (T)O[it][r];
                    }
            }
        }
        // S = lam^n S + sum_j s3 lam^(n - e0 - j) y_j z_j^T
        {
            const float keep = decay_pow(lam2, n);
#pragma unroll
            for (int at = 0; at < 2 * DXB; ++at)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[at][r] *= keep;
        }
        if (cuts) {
#pragma unroll
            for (int at = 0; at < 2 * DXB; ++at) S[at] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int jt = 0; jt < 2; ++jt) {
            const floatx4 f = *(const floatx4 *)&from_s[16 * jt + 4 * q];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float wz = zv[jt][r] * f[r];
#pragma unroll
                for (int at = 0; at < 2 * DXB; ++at)
                    S[at] = mfma_f32(ys[16 * jt + 4 * q + r][16 * at + l15], wz, S[at]);
            }
        }
        seg_cut |= cuts != 0;
        pos += n;
    }
    // rows behind the sequence's end are 0
    if (want_out)
        for (int t = max(p0, len) + (int)tid / DZ; t < min(a.T, p0 + a.seglen); t += NT / DZ)
            if (const int c = tid % DZ; c < a.dz) {
                const int64_t at = b * a.ob + h * a.oh + t * a.ot + c;
                if (a.out_f32) ((float *)a.out)[at] = 0.0f;
                else ((T *)a.out)[at] = (T)0.0f;
            }
    float *dst = nullptr;
    int64_t da = a.ia, dn = a.in;
    if (a.mode == 0 && a.fin) dst = a.fin + (int64_t)bh * a.dx * a.dz;
    if (a.mode == 1) dst = a.seg + ((int64_t)bh * a.nseg + g) * a.dx * a.dz, da = a.sa, dn = a.sn;
    if (dst) {
        // walking backward, what is left belongs to the state before token 0
        const bool drop = a.mode == 0 && a.rev && a.reset && len > 0 && a.reset[b * a.rb] != 0;
#pragma unroll
        for (int at = 0; at < 2 * DXB; ++at)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * at + 4 * q + r;
                if (row < a.dx && col < a.dz) dst[row * da + col * dn] = drop ? 0.0f : S[at][r];
            }
    }
    if (a.mode == 1 && tid == 0)
        a.segf[(int64_t)bh * a.nseg + g] = seg_cut ? -1.0f : decay_pow(lam2, max(p1 - p0, 0));
}

// ------------------------------------------------------------------------------------------
// The walk on bfloat16 operands
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack2(float a, float b) {  // two roundings to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2){a, b}, bf16x2));
}
__device__ __forceinline__ float lo_half(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_half(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

// An f32 value as the sum of three bf16 operands: each piece takes what the pieces before left over, at most
// 2^-9 of it, so the three hold a value to less than 2^-24 of itself, as f32 does.
constexpr int kPieces = 3;

__device__ __forceinline__ void split8(const float *v, bf16x8 (&out)[kPieces]) {
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
        uintx4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = pack2(rest[2 * e], rest[2 * e + 1]);
            rest[2 * e] -= lo_half(w[e]);
            rest[2 * e + 1] -= hi_half(w[e]);
        }
        out[p] = __builtin_bit_cast(bf16x8, w);
    }
}

__device__ __forceinline__ int begin_of64(uint64_t m, int i) {
    const uint64_t below = m & (~0ull >> (63 - i));
    return below ? 63 - __builtin_clzll(below) : -1;
}

// C rows of D bf16 columns on their way from global memory to LDS: 16 bytes a thread and step at any
// alignment; rows >= n and columns >= d become 0.
template <int C, int D, int NT>
struct Rows16 {
    static constexpr int VR = D / 8, N = (C * VR + NT - 1) / NT;
    uintx4 v[N];
    __device__ __forceinline__ void load(const __bf16 *src, int64_t st, int n, int d, unsigned tid) {
        const int row = tid / VR, c = tid % VR * 8;
        const __bf16 *p = src + row * st + c;
        if (n == C && d == D && C * VR >= NT) {
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = *(const uintx4_any *)(p + k * (NT / VR) * st);
            return;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = (uintx4){0, 0, 0, 0};
            if (row + k * (NT / VR) >= n) continue;
            const __bf16 *pk = p + k * (NT / VR) * st;
            if (c + 8 <= d) {
                v[k] = *(const uintx4_any *)pk;
            } else {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (c + e < d) v[k][e / 2] |= (uint32_t)__builtin_bit_cast(unsigned short, pk[e]) << (16 * (e & 1));
            }
        }
    }
    // PERM: of 32 columns the four-column groups in the order 0 4 1 5 2 6 3 7, in which a quarter wave's
    // eight columns are 16 bytes and match two accumulators' rows (see the kernel).
    template <bool PERM, int P>
    __device__ __forceinline__ void store(unsigned short (*dst)[P], unsigned tid) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const unsigned id = k * NT + tid;
            const int row = id / VR, c = id % VR * 8;
            if (C * VR < NT && row >= C) break;
            if (PERM) {
                const int at = (c & ~31) + (c & 8) * 2 + (c & 16) / 4;
                *(uintx2 *)&dst[row][at] = (uintx2){v[k][0], v[k][1]};
                *(uintx2 *)&dst[row][at + 8] = (uintx2){v[k][2], v[k][3]};
            } else {
                *(uintx4 *)&dst[row][c] = v[k];
            }
        }
    }
    __device__ __forceinline__ bool not_finite() const {
        ushortx2 m = {0, 0};
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                m = __builtin_elementwise_max(m, __builtin_bit_cast(ushortx2, v[k][e] & 0x7FFF7FFFu));
        return m[0] >= 0x7F80 || m[1] >= 0x7F80;
    }
};

// Rows j0 + 4 q .. + 3 of column c0 + (lane & 15), q = lane >> 4: the transposing LDS read, in which 16
// lanes give the addresses of 4 rows x 16 columns and get a column each. column32: also the rows 16 on,
// together the operand of 32 rows.
template <bool PERM, int P>
__device__ __forceinline__ uintx2 column4(const unsigned short (*t)[P], int j0, int c0, int lane) {
    typedef __attribute__((address_space(3))) shortx4 *lds4;
    const int row = j0 + (lane >> 2);
    const int c = PERM ? (c0 & ~31) + (c0 & 16) / 4 + (lane & 3) * 8 : c0 + (lane & 3) * 4;
    return __builtin_bit_cast(uintx2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)&t[row][c]));
}
template <bool PERM, int P>
__device__ __forceinline__ uintx4 column32(const unsigned short (*t)[P], int j0, int c0, int lane) {
    const uintx2 a = column4<PERM>(t, j0, c0, lane), b = column4<PERM>(t, j0 + 16, c0, lane);
    return (uintx4){a[0], a[1], b[0], b[1]};
}

// la_walk_kernel for bf16 operands on v_mfma_f32_16x16x32_bf16, C tokens a chunk. Products of the
// operands are exact in f32; what is not an operand (P and S for the output, the weighted z of the state's
// sum) is split into three bf16 pieces where it meets the matrix cores, so that outputs, gradients and states
// are those of f32 sums. With two pieces (2^-17 of each term) an output that is small beside its terms had
// wrong digits, for 7 to 14 % less time (65536 tokens 433 us for 487, the ragged prompts 179 for 197).
//
// A 16x16 accumulator holds rows 4 q + r (q = lane >> 4) of column lane & 15, so the accumulators of two
// row tiles are the operand of 32 rows in the order 4 q .. 4 q + 3, 16 + 4 q .. of the quarter waves. With
// the other operand read in that order (the order of a contraction is free) S goes from accumulator
// to operand without leaving its wave, and so does P, computed transposed as Y X^T.
//
// 16 columns a wave, not 32: with 32x32 tiles at two waves a SIMD the same work waited on LDS and on
// its own products (9 us a chunk of 128 x 128); half the registers a wave let four waves run.
//
// Bound by issue: of the cycles of 16 sequences of 65536 tokens, 128 x 128 (outputs in 335 us for 1.07 GB),
// vector instructions take 44 % and matrix instructions 34 %, and they seldom run at once. Without
// the check for infs and NaNs it takes 1 to 2 % less.
template <int DXB, int NW, int C>
__global__ __launch_bounds__(64 * NW, 32 * DXB <= 32 * NW ? 4 : 2) void la_walk_bf16_kernel(WalkArgs a) {
    constexpr int CT = C / 16, NP = CT * (CT + 1) / 2, SLOTS = C == 64 ? 6 : 2;  // token tiles, P's, their operands
    constexpr int DX = 32 * DXB, DZ = 16 * NW, NT = 64 * NW, PAD = 16;
    __shared__ __align__(16) unsigned short xs[C][DX + PAD];
    __shared__ __align__(16) unsigned short ys[C][DX + PAD];
    __shared__ __align__(16) unsigned short zs[C][DZ + PAD];
    __shared__ __align__(16) uintx2 ps[SLOTS][kPieces][64][2];  // (token tile, 32 tokens), piece, lane, half
    __shared__ __align__(16) float into_s[C], from_s[C];
    __shared__ int bad_s, first_s;
    unsigned tid = threadIdx.x;
    int lane = tid & 63, q = lane >> 4, l15 = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % a.H, b = by_length(a, blockIdx.x / a.H), g = blockIdx.y;
    const int64_t bh = (int64_t)b * a.H + h;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    const int p0 = g * a.seglen, p1 = min(len, p0 + a.seglen);
    const float lam2 = log2_decay(a.log_decay[h]);
    const int64_t tok0 = a.rev ? len - 1 : 0, dir = a.rev ? -1 : 1;
    const __bf16 *x = (const __bf16 *)a.x + b * a.xb + (h / a.gx) * a.xh + tok0 * a.xt;
    const __bf16 *y = (const __bf16 *)a.y + b * a.yb + (h / a.gy) * a.yh + tok0 * a.yt;
    const __bf16 *z = (const __bf16 *)a.z + b * a.zb + (h / a.gz) * a.zh + tok0 * a.zt;
    const int64_t out0 = b * a.ob + h * a.oh + tok0 * a.ot;
    const bool want_out = a.mode != 1 && a.out;
    const int c0 = 16 * w;
    int col = c0 + l15;

    floatx4 S[2 * DXB];
    {
        const float *src = nullptr;
        int64_t ia = a.ia, in = a.in;
        if (a.mode == 0 && a.init) src = a.init + (int64_t)bh * a.dx * a.dz;
        if (a.mode == 2) src = a.seg + ((int64_t)bh * a.nseg + g) * a.dx * a.dz, ia = a.sa, in = a.sn;
        load_state<DZ>(S, src, ia, in, a.dx, a.dz, 4 * q, col);
    }
    bool seg_cut = false;
    if (tid == 0) bad_s = -1;
    for (unsigned id = tid; id < SLOTS * kPieces * 64 * 2; id += NT) (&ps[0][0][0][0])[id] = (uintx2){0, 0};  // stays above the diagonal
    Rows16<C, DX, NT> rx, ry;
    Rows16<C, DZ, NT> rz;
    const int64_t xs_t = dir * a.xt, ys_t = dir * a.yt, zs_t = dir * a.zt;
    x += p0 * xs_t, y += p0 * ys_t, z += p0 * zs_t;  // of the chunk to load next, at position `ahead`
    int ahead = p0;
    uint32_t cut = 0;
    auto load = [&](int n) {
        cut = lane < n ? cut_at(a, b, ahead + lane, len) : 0;
        if (want_out) rx.load(x, xs_t, n, a.dx, tid);
        ry.load(y, ys_t, n, a.dx, tid);
        rz.load(z, zs_t, n, a.dz, tid);
    };
    auto step = [&](int n) { x += n * xs_t, y += n * ys_t, z += n * zs_t, ahead += n; };
    if (p0 < p1) load(min(C, p1 - p0));
    for (int pos = p0; pos < p1;) {
        tid = anew(tid), lane = tid & 63, q = lane >> 4, l15 = lane & 15, col = c0 + l15;
        int n = min(C, p1 - pos);
        // what a token takes from the state that comes in, and what it leaves to the one that goes out: only
        // tokens of the episodes that came in and that goes out
        auto factors = [&](uint64_t cuts) {
            if (tid < C) {
                const int i = tid;
                into_s[i] = cuts & (~0ull >> (63 - i)) ? 0.0f : a.s2 * decay_pow(lam2, i + a.e0);
                from_s[i] = i < n && i >= begin_of64(cuts, n - 1) ? a.s3 * decay_pow(lam2, n - a.e0 - i) : 0.0f;
            }
        };
        uint64_t cuts = __ballot(cut != 0);
        __syncthreads();  // the chunk before is done with the tiles
        if (want_out) rx.template store<true>(xs, tid);
        ry.template store<true>(ys, tid);
        rz.template store<false>(zs, tid);
        factors(cuts);
        if (ry.not_finite() || rz.not_finite()) bad_s = pos;
        step(n);
        if (ahead < p1) load(min(C, p1 - ahead));
        __syncthreads();
        if (bad_s == pos) {
            // An inf or NaN would reach rows it has no part in, through 0 * x in the products: the
            // chunk ends before a row that holds one, and such a row's chunk before the next episode.
            if (tid == 0) first_s = n;
            __syncthreads();
            bool head = false;
            for (int j = 0; j < n; ++j) {
                bool bad = false;
                for (unsigned c = tid; c < DX; c += NT) bad |= (ys[j][c] & 0x7F80) == 0x7F80;
                for (unsigned c = tid; c < DZ; c += NT) bad |= (zs[j][c] & 0x7F80) == 0x7F80;
                if (j == 0) head = __syncthreads_or(bad);
                else if (bad) atomicMin(&first_s, j);
            }
            __syncthreads();
            step(-n);
            n = first_s;
            if (head && (cuts & ~1ull)) n = min(n, (int)__builtin_ctzll(cuts & ~1ull));
            cuts &= ~0ull >> (64 - n);
            for (unsigned id = tid; id < (C - n) * DX; id += NT) ys[n + id / DX][id % DX] = 0;
            for (unsigned id = tid; id < (C - n) * DZ; id += NT) zs[n + id / DZ][id % DZ] = 0;
            step(n);
            if (ahead < p1) load(min(C, p1 - ahead));
            factors(cuts);
            __syncthreads();
        }
        floatx4 O[CT];
        uintx4 zv[CT / 2];  // z rows 32 js .. of the wave's columns: the operand of P Z, weighted that of S
        auto load_z = [&] {
#pragma unroll
            for (int js = 0; js < CT / 2; ++js) zv[js] = column32<false>(zs, 32 * js, c0, lane);
        };
        if (want_out) {
            // P^T = s1 lam^(i-j) Y X^T of the pairs j <= i of one episode in 16 x 16 tiles (j, i), shared
            // out over the waves and handed to all of them as operands, in pieces
            for (int t = w; t < NP; t += NW) {
                const int it = (t > 0) + (t > 2) + (t > 5), jt = t - it * (it + 1) / 2;
                floatx4 P = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < DXB; ++s)
                    P = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8 *)&ys[16 * jt + l15][32 * s + 8 * q],
                                                                *(const bf16x8 *)&xs[16 * it + l15][32 * s + 8 * q],
                                                                P, 0, 0, 0);
                const int d0 = 16 * (it - jt) + l15 - 4 * q;
                const int j0 = cuts ? begin_of64(cuts, 16 * it + l15) - 16 * jt - 4 * q : -C;  // of i's episode
                float pv[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    pv[r] = P[r] * (a.s1 * decay_pow(lam2, d0 - r));
                    pv[r] = r <= d0 && r >= j0 ? pv[r] : 0.0f;  // 0 whatever stood there
                }
                const int slot = it + (it == 3) + (jt >> 1);
#pragma unroll
                for (int p = 0; p < kPieces; ++p) {
                    const uintx2 o = {pack2(pv[0], pv[1]), pack2(pv[2], pv[3])};
                    ps[slot][p][lane][jt & 1] = o;
                    pv[0] -= lo_half(o[0]), pv[1] -= hi_half(o[0]), pv[2] -= lo_half(o[1]), pv[3] -= hi_half(o[1]);
                }
            }
            // x S, decayed to each row
#pragma unroll
            for (int it = 0; it < CT; ++it) O[it] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < DXB; ++s) {
                bf16x8 Sp[kPieces];
                float sv[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) sv[e] = S[2 * s + (e >> 2)][e & 3];
                split8(sv, Sp);
#pragma unroll
                for (int it = 0; it < CT; ++it) {
                    const bf16x8 X = *(const bf16x8 *)&xs[16 * it + l15][32 * s + 8 * q];
#pragma unroll
                    for (int p = 0; p < kPieces; ++p) O[it] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(X, Sp[p], O[it], 0, 0, 0);
                }
            }
#pragma unroll
            for (int it = 0; it < CT; ++it) {
                const floatx4 f = *(const floatx4 *)&into_s[16 * it + 4 * q];
#pragma unroll
                for (int r = 0; r < 4; ++r) O[it][r] *= f[r];
                if (cuts) {  // not 0 * inf
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[it][r] = f[r] != 0.0f ? O[it][r] : 0.0f;
                }
            }
            load_z();
            __syncthreads();  // P is there
#pragma unroll
            for (int it = 0; it < CT; ++it)
#pragma unroll
                for (int js = 0; js < (it >> 1) + 1; ++js)
#pragma unroll
                    for (int p = 0; p < kPieces; ++p)
                        O[it] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            *(const bf16x8 *)&ps[it + (it == 3) + js][p][lane], __builtin_bit_cast(bf16x8, zv[js]), O[it],
                            0, 0, 0);
        }
        if (!want_out) load_z();
        // S = lam^n S + sum_j s3 lam^(n - e0 - j) y_j z_j^T
        {
            const float keep = decay_pow(lam2, n);
#pragma unroll
            for (int at = 0; at < 2 * DXB; ++at)
#pragma unroll
                for (int r = 0; r < 4; ++r) S[at][r] *= keep;
        }
        if (cuts) {
#pragma unroll
            for (int at = 0; at < 2 * DXB; ++at) S[at] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int js = 0; js < CT / 2; ++js) {
            float wz[8];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const floatx4 f = *(const floatx4 *)&from_s[32 * js + 16 * m + 4 * q];
                wz[4 * m] = lo_half(zv[js][2 * m]) * f[0], wz[4 * m + 1] = hi_half(zv[js][2 * m]) * f[1];
                wz[4 * m + 2] = lo_half(zv[js][2 * m + 1]) * f[2], wz[4 * m + 3] = hi_half(zv[js][2 * m + 1]) * f[3];
            }
            bf16x8 Zp[kPieces];
            split8(wz, Zp);
#pragma unroll
            for (int at = 0; at < 2 * DXB; ++at) {
                const bf16x8 Y = __builtin_bit_cast(bf16x8, column32<true>(ys, 32 * js, 16 * at, lane));
#pragma unroll
                for (int p = 0; p < kPieces; ++p) S[at] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(Y, Zp[p], S[at], 0, 0, 0);
            }
        }
        if (want_out) {
            // out through the wave's own columns of the z tile, which it is done with: 16-byte stores
            if (!a.out_f32) {
#pragma unroll
                for (int it = 0; it < CT; ++it)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const uint32_t o = pack2(O[it][r], O[it][r + 1]);
                        zs[16 * it + 4 * q + r][col] = (unsigned short)o;
                        zs[16 * it + 4 * q + r + 1][col] = (unsigned short)(o >> 16);
                    }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // lanes read what other lanes wrote
                const int row = lane >> 1, c = c0 + (lane & 1) * 8;
                __bf16 *o = (__bf16 *)a.out + out0 + (pos + row) * dir * a.ot + c;
#pragma unroll
                for (int k = 0; k < CT / 2; ++k) {
                    if (row + 32 * k >= n) continue;
                    __bf16 *ok = o + 32 * k * dir * a.ot;
                    if (c + 8 <= a.dz) {
                        *(uintx4_any *)ok = *(uintx4 *)&zs[row + 32 * k][c];
                    } else {
                        for (int e = 0; c + e < a.dz; ++e) ok[e] = __builtin_bit_cast(__bf16, zs[row + 32 * k][c + e]);
                    }
                }
            } else {
                float *o = (float *)a.out + out0 + (pos + 4 * q) * dir * a.ot + col;
                if (col < a.dz)
#pragma unroll
                    for (int it = 0; it < CT; ++it)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (16 * it + 4 * q + r < n) o[(16 * it + r) * dir * a.ot] = O[it][r];
            }
        }
        seg_cut |= cuts != 0;
        pos += n;
    }
    // rows behind the sequence's end are 0
    if (want_out)
        for (int t = max(p0, len) + (int)tid / DZ; t < min(a.T, p0 + a.seglen); t += NT / DZ)
            if (const int c = tid % DZ; c < a.dz) {
                const int64_t at = b * a.ob + h * a.oh + t * a.ot + c;
                if (a.out_f32) ((float *)a.out)[at] = 0.0f;
                else ((__bf16 *)a.out)[at] = (__bf16)0.0f;
            }
    float *dst = nullptr;
    int64_t da = a.ia, dn = a.in;
    if (a.mode == 0 && a.fin) dst = a.fin + (int64_t)bh * a.dx * a.dz;
    if (a.mode == 1) dst = a.seg + ((int64_t)bh * a.nseg + g) * a.dx * a.dz, da = a.sa, dn = a.sn;
    if (dst) {
        const bool drop = a.mode == 0 && a.rev && a.reset && len > 0 && a.reset[b * a.rb] != 0;
#pragma unroll
        for (int at = 0; at < 2 * DXB; ++at)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = 16 * at + 4 * q + r;
                if (row < a.dx && col < a.dz) dst[row * da + col * dn] = drop ? 0.0f : S[at][r];
            }
    }
    if (a.mode == 1 && tid == 0)
        a.segf[(int64_t)bh * a.nseg + g] = seg_cut ? -1.0f : decay_pow(lam2, max(p1 - p0, 0));
}

// Joins the segments of a split sequence: seg[g] becomes the state that comes into segment g.
__global__ __launch_bounds__(256) void la_join_kernel(WalkArgs a) {
    const int bh = blockIdx.x, b = bh / a.H, e = blockIdx.y * 256 + threadIdx.x;
    if (e >= a.dx * a.dz) return;
    const int64_t size = (int64_t)a.dx * a.dz, at = bh * size + (e / a.dz) * a.ia + (e % a.dz) * a.in;
    float carry = a.init ? a.init[at] : 0.0f;
    float *seg = a.seg + bh * a.nseg * size + e;
    const float *f = a.segf + (int64_t)bh * a.nseg;
    for (int g = 0; g < a.nseg; g += 8) {
        float u[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = g + k < a.nseg ? seg[(g + k) * size] : 0.0f;  // in flight together
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (g + k >= a.nseg) break;
            seg[(g + k) * size] = carry;
            carry = f[g + k] < 0.0f ? u[k] : f[g + k] * carry + u[k];
        }
    }
    if (a.fin) {
        const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
        const bool drop = a.rev && a.reset && len > 0 && a.reset[b * a.rb] != 0;
        a.fin[at] = drop ? 0.0f : carry;
    }
}

// Gradient of a shared head: the sum of its states' f32 partials [B][T][H][D], in head order.
template <typename T>
__global__ __launch_bounds__(256) void la_share_kernel(const float *part, T *out, int64_t ob, int64_t ot,
                                                       int64_t oh, int B, int T_, int Hs, int group, int D) {
    const int64_t total = (int64_t)B * T_ * Hs * D;
    for (int64_t id = blockIdx.x * 256LL + threadIdx.x; id < total; id += gridDim.x * 256LL) {
        const int d = id % D;
        int64_t rest = id / D;
        const int hs = rest % Hs;
        rest /= Hs;
        const int t = rest % T_, b = (int)(rest / T_);
        const float *p = part + ((((int64_t)b * T_ + t) * Hs + hs) * group) * D + d;
        float s = 0.0f;
        for (int k = 0; k < group; ++k) s += p[(int64_t)k * D];
        out[b * ob + t * ot + hs * oh + d] = (T)s;
    }
}

// One token for every sequence: reads and writes each state once, 4 columns a lane, LC lanes a row, four
// rows' loads in flight. A block owns 4 LC columns of one (batch, head) state. Bound by HBM: 16384 x 4
// states of 64 x 64 from one buffer to another in 346 us, 6.2 TB/s. STREAM: loads and stores that pass
// the caches by, for states that do not stay in them (see the launch).
struct StepArgs {
    const void *q, *k, *v;
    void *out;
    int64_t qb, qh, kb, kh, vb, vh, ob, oh;
    int gq, gk, gv;
    const float *log_decay;
    const float *state;
    float *state_out;
    const uint8_t *reset;
    int64_t rb;
    float scale;
    int H, dk, dv;
};

template <typename T, int LC, bool STREAM>
__global__ __launch_bounds__(256) void la_step_kernel(StepArgs a) {
    constexpr int R = 256 / LC, U = 4;  // rows at a time, times in flight
    __shared__ float part[R][4 * LC + 1];
    const int64_t bh = blockIdx.x;
    const int b = (int)(bh / a.H), h = (int)(bh % a.H);
    const int lc = threadIdx.x % LC, r0 = threadIdx.x / LC, c0 = (blockIdx.y * LC + lc) * 4;
    const T *q = (const T *)a.q + b * a.qb + (h / a.gq) * a.qh;
    const T *k = (const T *)a.k + b * a.kb + (h / a.gk) * a.kh;
    const T *v = (const T *)a.v + b * a.vb + (h / a.gv) * a.vh;
    const bool drop = a.reset && a.reset[b * a.rb] != 0;
    const float lam = decay_pow(log2_decay(a.log_decay[h]), 1);
    const bool full = c0 + 4 <= a.dv;
    float vc[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) vc[e] = c0 + e < a.dv ? to_f32(v[c0 + e]) : 0.0f;
    const float *src = a.state + bh * a.dk * a.dv + c0;
    float *dst = a.state_out + bh * a.dk * a.dv + c0;
    for (int rb = r0; rb < a.dk; rb += R * U) {
        floatx4 s[U];
        float kr[U], qr[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = rb + u * R;
            s[u] = (floatx4){0.f, 0.f, 0.f, 0.f};
            if (r >= a.dk) continue;
            kr[u] = to_f32(k[r]), qr[u] = to_f32(q[r]);
            if (drop) continue;
            if (full) {
                const floatx4_any *p = (const floatx4_any *)(src + r * a.dv);
                s[u] = STREAM ? __builtin_nontemporal_load(p) : *p;
            } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (c0 + e < a.dv) s[u][e] = src[r * a.dv + e];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = rb + u * R;
            if (r >= a.dk) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[u][e] = lam * s[u][e] + kr[u] * vc[e];
                o[e] += qr[u] * s[u][e];
            }
            if (full) {
                if (STREAM) __builtin_nontemporal_store(s[u], (floatx4_any *)(dst + r * a.dv));
                else *(floatx4_any *)(dst + r * a.dv) = s[u];
            } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (c0 + e < a.dv) dst[r * a.dv + e] = s[u][e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[r0][lc * 4 + e] = o[e];
    __syncthreads();
    if (threadIdx.x < 4 * LC) {
        const int c = blockIdx.y * 4 * LC + threadIdx.x;
        float s = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) s += part[r][threadIdx.x];
        if (c < a.dv) ((T *)a.out)[b * a.ob + h * a.oh + c] = (T)(a.scale * s);
    }
}

// ------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------
constexpr int kMaxD = 128;

// A sequence is split where batch x heads leave most CUs idle, into as many segments as fill the card
// with the two blocks a CU holds at D = 128. A segment has 256 tokens at least, so that its state's way
// through memory stays below the walk. The split walk reads y and z twice: 384 sequences of up to 2047
// tokens take 305 us in two parts each, 213 us whole (128 x 128 bf16); 16 of 65536 tokens 480 us in 512
// blocks, 552 in 256 and 502 in 768.
int segments(int64_t bh, int T, int *seglen) {
    *seglen = T > 0 ? T : 1;
    if (bh < 1 || bh > 128 || T < 512) return 1;
    const int want = (int)(512 / bh);
    int len = (T + want - 1) / want;
    len = (len + 63) / 64 * 64;
    if (len < 256) len = 256;
    *seglen = len;
    return (T + len - 1) / len;
}

int64_t segment_floats(int64_t bh, int T, int Dk, int Dv) {
    int len;
    const int64_t ns = segments(bh, T, &len);
    return ns > 1 ? bh * ns * ((int64_t)Dk * Dv + 1) : 0;
}

template <typename T, int DXB>
void launch_walk(const WalkArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)a.B * a.H), a.nseg);
    auto go = [&](auto nw) {
        constexpr int NW = decltype(nw)::value;
        if constexpr (std::is_same_v<T, __bf16>) {
            // 64 tokens a chunk: half the barriers and state steps. Up to 64 columns 32 tokens leave LDS for twice
            // the blocks, which pays where there are blocks enough: 16384 of 128 tokens, 64 x 64, in 260 us for
            // 322, 1024 of 1000 tokens in 137 for 169, 512 of 2048 tokens in 168 for 174, but 512 of 128 tokens in 16.2
            // for 15.3, 256 of 2048 in 139 for 132, 512 parts of 65536 tokens in 260 for 255. So do sequences that end
            // within them (8192 of 32 tokens, 128 x 128, 118 us for 165; 800 of 24 tokens 19 for 25)
            auto chunk = [&](auto c) {
                constexpr int C = decltype(c)::value;
                la_walk_bf16_kernel<DXB, NW, C><<<grid, 64 * NW, 0, s>>>(a);
            };
            if ((NW <= 4 && grid.x >= 512) || a.T <= 32) return chunk(std::integral_constant<int, 32>{});
            chunk(std::integral_constant<int, 64>{});
        } else {
            la_walk_kernel<T, DXB, NW><<<grid, 64 * NW, 0, s>>>(a);
        }
    };
    if (a.dz <= 32) go(std::integral_constant<int, 2>{});
    else if (a.dz <= 64) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
}

template <typename T>
void launch_walk(const WalkArgs &a, hipStream_t s) {
    if (a.dx <= 32) launch_walk<T, 1>(a, s);
    else if (a.dx <= 64) launch_walk<T, 2>(a, s);
    else launch_walk<T, 4>(a, s);
}

// have_states: ws holds the segments' states of another walk, which were this one's transposed; they are
// read only.
template <typename T>
void walk(WalkArgs a, float *ws, hipStream_t s, bool have_states = false) {
    const int64_t bh = (int64_t)a.B * a.H;
    a.nseg = segments(bh, a.T, &a.seglen);
    a.seg = ws;
    if (a.nseg > 1 && have_states) {
        a.sa = 1, a.sn = a.dx;
        a.mode = 2;
    } else if (a.nseg > 1) {
        a.sa = a.dz, a.sn = 1;
        a.segf = ws + bh * a.nseg * a.dx * a.dz;
        a.mode = 1;
        launch_walk<T>(a, s);
        la_join_kernel<<<dim3((unsigned)bh, (a.dx * a.dz + 255) / 256), 256, 0, s>>>(a);
        a.mode = 2;
    }
    if (a.mode == 0 || a.out) launch_walk<T>(a, s);
}

WalkArgs base_args(const rlp_la_cfg &c, const float *log_decay, const uint8_t *reset, const int32_t *lengths) {
    WalkArgs a = {};
    a.B = c.B, a.T = c.T, a.H = c.H;
    a.log_decay = log_decay, a.reset = reset, a.lengths = lengths;
    a.rb = c.reset_stride[0], a.rt = c.reset_stride[1];
    return a;
}

void set(const void *&p, int64_t &b, int64_t &t, int64_t &h, const void *src, const int64_t *st) {
    p = src, b = st[0], t = st[1], h = st[2];
}

template <typename T>
void forward(const rlp_la_cfg &c, const void *q, const void *k, const void *v, const float *log_decay,
             const uint8_t *reset, const int32_t *lengths, const float *init, void *out, float *fin,
             float *ws, hipStream_t s) {
    WalkArgs a = base_args(c, log_decay, reset, lengths);
    set(a.x, a.xb, a.xt, a.xh, q, c.q_stride);
    set(a.y, a.yb, a.yt, a.yh, k, c.k_stride);
    set(a.z, a.zb, a.zt, a.zh, v, c.v_stride);
    a.gx = c.H / c.Hq, a.gy = c.H / c.Hk, a.gz = c.H / c.Hv;
    a.out = out, a.ob = c.o_stride[0], a.ot = c.o_stride[1], a.oh = c.o_stride[2];
    a.dx = c.Dk, a.dz = c.Dv;
    a.init = init, a.fin = fin, a.ia = c.Dv, a.in = 1;
    a.e0 = 1, a.s1 = a.s2 = c.scale, a.s3 = 1.0f;
    walk<T>(a, ws, s);
}

template <typename T>
void share(const rlp_la_cfg &c, const float *part, void *out, const int64_t *st, int Hs, int D, hipStream_t s) {
    const int64_t total = (int64_t)c.B * c.T * Hs * D;
    if (total == 0) return;
    const int64_t blocks = (total + 255) / 256;
    la_share_kernel<T><<<(unsigned)(blocks < 16384 ? blocks : 16384), 256, 0, s>>>(
        part, (T *)out, st[0], st[1], st[2], c.B, c.T, Hs, c.H / Hs, D);
}

template <typename T>
void backward(const rlp_la_cfg &c, const void *q, const void *k, const void *v, const float *log_decay,
              const uint8_t *reset, const int32_t *lengths, const float *init, const void *d_out,
              const float *d_fin, void *dq, void *dk, void *dv, float *d_init, const float *forward_ws, float *ws,
              hipStream_t s) {
    const int64_t bh = (int64_t)c.B * c.H;
    float *part = ws + segment_floats(bh, c.T, c.Dk, c.Dv);
    // a gradient of unshared heads goes straight out, of shared heads through f32 partials
    auto target = [&](WalkArgs &a, void *out, const int64_t *st, int Hs, int D) {
        if (!out || Hs == c.H) {
            a.out = out, a.ob = st[0], a.ot = st[1], a.oh = st[2];
        } else {
            a.out = part, a.out_f32 = 1;
            a.oh = D, a.ot = (int64_t)c.H * D, a.ob = a.ot * c.T;
        }
    };
    if (dq) {
        WalkArgs a = base_args(c, log_decay, reset, lengths);
        set(a.x, a.xb, a.xt, a.xh, d_out, c.o_stride);
        set(a.y, a.yb, a.yt, a.yh, v, c.v_stride);
        set(a.z, a.zb, a.zt, a.zh, k, c.k_stride);
        a.gx = 1, a.gy = c.H / c.Hv, a.gz = c.H / c.Hk;
        a.dx = c.Dv, a.dz = c.Dk;
        a.init = init, a.ia = 1, a.in = c.Dv;  // S transposed
        a.e0 = 1, a.s1 = a.s2 = c.scale, a.s3 = 1.0f;
        target(a, dq, c.dq_stride, c.Hq, c.Dk);
        walk<T>(a, forward_ws ? const_cast<float *>(forward_ws) : ws, s, forward_ws != nullptr);
        if (c.Hq != c.H) share<T>(c, part, dq, c.dq_stride, c.Hq, c.Dk, s);
    }
    if (dv || d_init) {
        WalkArgs a = base_args(c, log_decay, reset, lengths);
        set(a.x, a.xb, a.xt, a.xh, k, c.k_stride);
        set(a.y, a.yb, a.yt, a.yh, q, c.q_stride);
        set(a.z, a.zb, a.zt, a.zh, d_out, c.o_stride);
        a.gx = c.H / c.Hk, a.gy = c.H / c.Hq, a.gz = 1;
        a.dx = c.Dk, a.dz = c.Dv;
        a.init = d_fin, a.fin = d_init, a.ia = c.Dv, a.in = 1;
        a.rev = 1, a.e0 = 0, a.s1 = c.scale, a.s2 = 1.0f, a.s3 = c.scale;
        target(a, dv, c.dv_stride, c.Hv, c.Dv);
        walk<T>(a, ws, s);
        if (dv && c.Hv != c.H) share<T>(c, part, dv, c.dv_stride, c.Hv, c.Dv, s);
    }
    if (dk) {
        WalkArgs a = base_args(c, log_decay, reset, lengths);
        set(a.x, a.xb, a.xt, a.xh, v, c.v_stride);
        set(a.y, a.yb, a.yt, a.yh, d_out, c.o_stride);
        set(a.z, a.zb, a.zt, a.zh, q, c.q_stride);
        a.gx = c.H / c.Hv, a.gy = 1, a.gz = c.H / c.Hq;
        a.dx = c.Dv, a.dz = c.Dk;
        a.init = d_fin, a.ia = 1, a.in = c.Dv;  // R transposed
        a.rev = 1, a.e0 = 0, a.s1 = c.scale, a.s2 = 1.0f, a.s3 = c.scale;
        target(a, dk, c.dk_stride, c.Hk, c.Dk);
        walk<T>(a, ws, s, dv || d_init);
        if (c.Hk != c.H) share<T>(c, part, dk, c.dk_stride, c.Hk, c.Dk, s);
    }
}

int check_cfg(const rlp_la_cfg *c, const char *who) {
    RLP_REQUIRE(c, "%s: null cfg", who);
    RLP_REQUIRE(c->dtype == RLP_F32 || c->dtype == RLP_F16 || c->dtype == RLP_BF16, "%s: dtype %d", who, c->dtype);
    RLP_REQUIRE(c->B >= 0 && c->T >= 0 && c->H >= 1, "%s: B %d, T %d, H %d", who, c->B, c->T, c->H);
    RLP_REQUIRE(c->Hq >= 1 && c->Hk >= 1 && c->Hv >= 1 && c->H % c->Hq == 0 && c->H % c->Hk == 0 &&
                    c->H % c->Hv == 0,
                "%s: %d states for %d / %d / %d heads of q / k / v (each has to divide it)", who, c->H,
                c->Hq, c->Hk, c->Hv);
    RLP_REQUIRE(c->Dk >= 1 && c->Dk <= kMaxD && c->Dv >= 1 && c->Dv <= kMaxD,
                "%s: Dk %d, Dv %d (1 to %d)", who, c->Dk, c->Dv, kMaxD);
    RLP_REQUIRE((int64_t)c->B * c->H < (1 << 23) && c->T <= (1 << 30), "%s: B x H or T too large", who);
    return RLP_OK;
}

int64_t workspace_bytes(const rlp_la_cfg &c, bool backward) {
    const int64_t bh = (int64_t)c.B * c.H;
    int64_t f = segment_floats(bh, c.T, c.Dk, c.Dv);
    if (backward) {
        int D = 0;
        if (c.Hq != c.H || c.Hk != c.H) D = c.Dk;
        if (c.Hv != c.H && c.Dv > D) D = c.Dv;
        f += bh * c.T * D;
    }
    return f * 4;
}

// The bytes from the first to behind the last of B x H rows of D elements.
struct Span {
    const char *first, *behind;
    Span(const void *p, int64_t B, int64_t b, int64_t H, int64_t h, int64_t D, int64_t size) {
        const int64_t db = (B - 1) * b, dh = (H - 1) * h;
        first = (const char *)p + size * ((db < 0 ? db : 0) + (dh < 0 ? dh : 0));
        behind = (const char *)p + size * ((db > 0 ? db : 0) + (dh > 0 ? dh : 0) + D);
    }
    bool meets(const Span &o) const { return first < o.behind && o.first < behind; }
};

template <typename F>
void by_type(int dtype, F &&f) {
    if (dtype == RLP_F32) f((float *)nullptr);
    else if (dtype == RLP_F16) f((_Float16 *)nullptr);
    else f((__bf16 *)nullptr);
}

}  // namespace
}  // namespace rlp

using namespace rlp;

extern "C" {

int64_t rlp_linear_attention_workspace_bytes(const rlp_la_cfg *cfg, int backward) {
    const int rc = check_cfg(cfg, "rlp_linear_attention_workspace_bytes");
    return rc != RLP_OK ? rc : workspace_bytes(*cfg, backward != 0);
}

int rlp_linear_attention(const rlp_la_cfg *cfg, const void *q, const void *k, const void *v,
                         const float *log_decay, const uint8_t *reset, const int32_t *lengths,
                         const float *state, void *out, float *state_out, void *workspace,
                         int64_t workspace_bytes_, rlp_stream_t stream) {
    take_pending();
    const int rc = check_cfg(cfg, "rlp_linear_attention");
    if (rc != RLP_OK) return rc;
    if (cfg->B == 0 || (cfg->T == 0 && !state_out)) return RLP_OK;
    RLP_REQUIRE(log_decay && (cfg->T == 0 || (q && k && v && out)), "rlp_linear_attention: null argument");
    const int64_t need = workspace_bytes(*cfg, false);
    RLP_REQUIRE(need == 0 || (workspace && workspace_bytes_ >= need),
                "rlp_linear_attention: workspace of %lld bytes, %lld needed", (long long)workspace_bytes_,
                (long long)need);
    by_type(cfg->dtype, [&](auto *t) {
        forward<std::remove_pointer_t<decltype(t)>>(*cfg, q, k, v, log_decay, reset, lengths, state, out,
                                                    state_out, (float *)workspace, as_stream(stream));
    });
    RLP_CHECK_LAUNCH("rlp_linear_attention");
    return RLP_OK;
}

int rlp_linear_attention_backward(const rlp_la_cfg *cfg, const void *q, const void *k, const void *v,
                                  const float *log_decay, const uint8_t *reset, const int32_t *lengths,
                                  const float *state, const void *d_out, const float *d_state_out,
                                  const void *forward_workspace, void *dq, void *dk, void *dv,
                                  float *d_state, void *workspace, int64_t workspace_bytes_,
                                  rlp_stream_t stream) {
    take_pending();
    const int rc = check_cfg(cfg, "rlp_linear_attention_backward");
    if (rc != RLP_OK) return rc;
    if (cfg->B == 0 || (cfg->T == 0 && !d_state)) return RLP_OK;
    if (!dq && !dk && !dv && !d_state) return RLP_OK;
    RLP_REQUIRE(log_decay && (cfg->T == 0 || (q && k && v && d_out)),
                "rlp_linear_attention_backward: null argument");
    const int64_t need = workspace_bytes(*cfg, true);
    RLP_REQUIRE(need == 0 || (workspace && workspace_bytes_ >= need),
                "rlp_linear_attention_backward: workspace of %lld bytes, %lld needed",
                (long long)workspace_bytes_, (long long)need);
    by_type(cfg->dtype, [&](auto *t) {
        backward<std::remove_pointer_t<decltype(t)>>(*cfg, q, k, v, log_decay, reset, lengths, state, d_out,
                                                     d_state_out, dq, dk, dv, d_state,
                                                     (const float *)forward_workspace, (float *)workspace,
                                                     as_stream(stream));
    });
    RLP_CHECK_LAUNCH("rlp_linear_attention_backward");
    return RLP_OK;
}

int rlp_linear_attention_step(const rlp_la_cfg *cfg, const void *q, const void *k, const void *v,
                              const float *log_decay, const uint8_t *reset, const float *state,
                              float *state_out, void *out, rlp_stream_t stream) {
    take_pending();
    const int rc = check_cfg(cfg, "rlp_linear_attention_step");
    if (rc != RLP_OK) return rc;
    RLP_REQUIRE(cfg->T == 1, "rlp_linear_attention_step: T = %d (one token)", cfg->T);
    if (cfg->B == 0) return RLP_OK;
    RLP_REQUIRE(q && k && v && log_decay && state && state_out && out, "rlp_linear_attention_step: null argument");
    {   // blocks of other heads and columns read the inputs while one writes; out's rows may lie between theirs
        const int64_t B = cfg->B, H = cfg->H, D = (int64_t)cfg->Dk * cfg->Dv, size = cfg->dtype == RLP_F32 ? 4 : 2;
        const Span in[5] = {{q, B, cfg->q_stride[0], cfg->Hq, cfg->q_stride[2], cfg->Dk, size},
                            {k, B, cfg->k_stride[0], cfg->Hk, cfg->k_stride[2], cfg->Dk, size},
                            {v, B, cfg->v_stride[0], cfg->Hv, cfg->v_stride[2], cfg->Dv, size},
                            {log_decay, 1, 0, 1, 0, H, 4},
                            {reset, reset ? B : 0, cfg->reset_stride[0], 1, 0, reset ? 1 : 0, 1}};
        const Span before(state, 1, 0, 1, 0, B * H * D, 4), after(state_out, 1, 0, 1, 0, B * H * D, 4);
        const Span o(out, B, cfg->o_stride[0], H, cfg->o_stride[2], cfg->Dv, size);
        RLP_REQUIRE(state == state_out || !after.meets(before), "rlp_linear_attention_step: state_out overlaps state");
        RLP_REQUIRE(!o.meets(before) && !o.meets(after), "rlp_linear_attention_step: out overlaps a state");
        for (int i = 0; i < (reset ? 5 : 4); ++i)
            RLP_REQUIRE(!in[i].meets(after), "rlp_linear_attention_step: the updated state overlaps another argument");
    }
    StepArgs a = {};
    a.q = q, a.k = k, a.v = v, a.out = out, a.log_decay = log_decay, a.state = state, a.state_out = state_out;
    a.qb = cfg->q_stride[0], a.qh = cfg->q_stride[2], a.kb = cfg->k_stride[0], a.kh = cfg->k_stride[2];
    a.vb = cfg->v_stride[0], a.vh = cfg->v_stride[2], a.ob = cfg->o_stride[0], a.oh = cfg->o_stride[2];
    a.gq = cfg->H / cfg->Hq, a.gk = cfg->H / cfg->Hk, a.gv = cfg->H / cfg->Hv;
    a.reset = reset, a.rb = cfg->reset_stride[0];
    a.scale = cfg->scale, a.H = cfg->H, a.dk = cfg->Dk, a.dv = cfg->Dv;
    // few states: narrow blocks, more of them on the card; many: whole 256-byte rows
    const int64_t bh = (int64_t)cfg->B * cfg->H;
    const bool narrow = cfg->Dv <= 32 || bh < 512;
    // states beyond the 256 MB last-level cache: past it, 512 MB in place in 167 us for 196 (within it the
    // next step finds them: 128 MB 41 us for 44)
    const bool stream_by = bh * cfg->Dk * cfg->Dv * (state == state_out ? 4 : 8) > (256LL << 20);
    const dim3 grid((unsigned)bh, narrow ? (cfg->Dv + 31) / 32 : (cfg->Dv + 63) / 64);
    by_type(cfg->dtype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (stream_by) {
            if (narrow) la_step_kernel<T, 8, true><<<grid, 256, 0, as_stream(stream)>>>(a);
            else la_step_kernel<T, 16, true><<<grid, 256, 0, as_stream(stream)>>>(a);
        } else {
            if (narrow) la_step_kernel<T, 8, false><<<grid, 256, 0, as_stream(stream)>>>(a);
            else la_step_kernel<T, 16, false><<<grid, 256, 0, as_stream(stream)>>>(a);
        }
    });
    RLP_CHECK_LAUNCH("rlp_linear_attention_step");
    return RLP_OK;
}

}  // extern "C"
