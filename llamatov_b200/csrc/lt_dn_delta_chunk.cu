// Gated delta rule over prompt rows in chunks of 64 tokens on the tensor cores (mma.sync m16n8k16, bf16 operands, fp32 sums).
// Of a chunk, with b_i the sum of its log decays up to and including token i, K and Q its raw rows, r_i = 1 / |k_i|, S the state
// it starts from:
//   A_ij = beta_i e^(b_i - b_j) r_i r_j k_i . k_j  (j < i),   T = (I + A)^-1 diag(beta)
//   U = T (V - diag(e^b r) K S^T)
//   S <- e^(b_end) S + U^T diag(r e^(b_end - b)) K
//   O = rq q_scale (diag(e^b) Q S^T + tril(Q K^T .* r_j e^(b_i - b_j)) U)
//
// With W = T diag(e^b r) K and U0 = T V, which need no state, U = U0 - W S^T.
//
//   k_delta_prep    every chunk and head at once: T by forward substitution in blocks, in fp32; W, U0
//   k_delta_states  walks the chunks: a CTA owns 16 value columns of one head of one sequence, its warps the key channels; the state
//                   stays in their accumulators, transposed (rows are value columns), so that it is the A operand of the next
//                   product as it stands; stores the state a chunk starts from, and U
//   k_delta_out     every chunk and head at once
//
// What is bf16 in memory (q, k, v) enters exactly.  Everything else is fp32: it enters as the sum of three bf16 (24 significant
// bits), three products against bf16 and six against another such sum, so that chunks are as exact as token order.  The
// tensor cores cut sums off instead of rounding them, which costs up to 2^-23 of the accumulator at every step.  So the products of the
// leading parts have accumulators of their own in U0, in the update of the state and in the outputs; in W and W S^T all parts share one,
// the smallest first, as there the leading ones are four steps and at most two.
//
// A row that is not finite (infinities, NaN) makes the outputs of its heads not finite over its whole chunk, earlier tokens' among them: products
// over a chunk have zeros where token order has nothing.  Other heads, other sequences and earlier chunks are as they would be.
//
// The walk over the chunks is the longest of the three, and bound by the instructions and waits of a chunk's dependent chain.  So W, U0
// and the keys lie in memory as the lanes hold them (16 bytes a lane, side by side) and go straight into registers, asked for when
// the chunk before has used them; a chunk passes two barriers.  (16 heads of 128, 2048 rows: 32, 70 and 37 us; four
// sequences of them 437 together.  With T in place of W, one product and barrier more, and operands through shared memory: 17, 76 and 38;
// 484.)
#include "lt_dn_delta.cuh"
#include "lt_dn_mma.cuh"

namespace lt {
namespace dn {

constexpr int DC = 64;                          // tokens of a chunk
constexpr float DLOG2E = 1.4426950408889634f;
constexpr int TS = DC + 8;                      // row stride of 64-column bf16 tiles: an odd number of 16-byte units
constexpr int DVEC = DC + 4;                    // r e^(b_end - b), e^(b_end)

struct DeltaChunkP {
    const bf16 *q, *k, *v;
    const float *la, *beta;
    float* o;
    // [chunk][H], in lanes' order: W [dp/16][64/16][3] of uint4 x 32; starting states [dvp/16][dp/16][3] of uint4 x 32; U0, then U
    // [dvp/16][64/8] of float4 x 32; vec [DVEC].  [chunk][G]: keys [dp/16][64/16] of uint4 x 32
    uint4 *W, *S0, *Kf;
    float4* U;
    float* vec;
    int nkt, nvt;            // tiles of 16 key channels, of 16 value columns
    int ld, ldla, ldb, ldo;
    int first[LT_DN_SEQS + 1];    // chunks before a sequence's
    lt_dn_delta D;
    lt_dn_seqs Q;
};

// x, y as three packed pairs of bf16 that add up to them
__device__ __forceinline__ void split3(float x, float y, unsigned& h, unsigned& m, unsigned& l) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x, y);
    x -= __low2float(a);
    y -= __high2float(a);
    const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
    const __nv_bfloat162 c = __floats2bfloat162_rn(x - __low2float(b), y - __high2float(b));
    h = *(const unsigned*)&a;
    m = *(const unsigned*)&b;
    l = *(const unsigned*)&c;
}

struct Chunk {
    int b, t0, rows;         // sequence, first token in it, tokens
    long row0;               // row of the first token
};
__device__ __forceinline__ Chunk chunk_of(const DeltaChunkP& P, int c) {
    Chunk r;
    r.b = 0;
    while (c >= P.first[r.b + 1]) r.b++;
    r.t0 = (c - P.first[r.b]) * DC;
    r.rows = min(DC, P.Q.rows[r.b] - r.t0);
    r.row0 = (long)P.Q.start[r.b] + r.t0;
    return r;
}

// sums of a chunk's log decays (base 2), by one warp: doubles, so that a difference of two sums is as near as its own terms, which are
// fp32 products (2^-24 of each, and 2^-26 of the constant)
__device__ __forceinline__ void log_sums(const DeltaChunkP& P, const Chunk& c, int h, int lane, double* sb) {
    const int t = 2 * lane;
    const double l0 = t < c.rows ? (double)(delta_log(P.la[(c.row0 + t) * P.ldla + h]) * DLOG2E) : 0.0;
    const double l1 = t + 1 < c.rows ? (double)(delta_log(P.la[(c.row0 + t + 1) * P.ldla + h]) * DLOG2E) : 0.0;
    double p = l0 + l1;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, p, s);
        if (lane >= s) p += x;
    }
    double before = __shfl_up_sync(0xffffffffu, p, 1);
    if (lane == 0) before = 0.0;
    sb[t] = before + l0;
    sb[t + 1] = p;
}

// rows of q or k of a group, zeros outside; stride in elements, `units` of 16 bytes a row
__device__ __forceinline__ void load_rows(bf16* dst, int stride, int units, const bf16* src, const Chunk& c, int ld, int col, int width) {
    for (int e = threadIdx.x; e < DC * units; e += blockDim.x) {
        const int t = e / units, x = (e - t * units) * 8;
        const bool ok = t < c.rows && x < width;
        cp16(dst + t * stride + x, src + (ok ? (c.row0 + t) * ld + col + x : 0), ok);
    }
}
// scale / |row| of 64 rows, eight lanes per row
__device__ __forceinline__ void row_norms(const bf16* s, int stride, int units, float eps, float scale, float* out) {
    const int sub = threadIdx.x & 7;
    for (int t = threadIdx.x >> 3; t < DC; t += blockDim.x >> 3) {
        float a = 0.0f;
        for (int x = sub; x < units; x += 8) {
            float f[8];
            Vec<bf16>::unpack(*(const uint4*)(s + t * stride + x * 8), f);
#pragma unroll
            for (int i = 0; i < 8; i++) a = fmaf(f[i], f[i], a);
        }
        a += __shfl_xor_sync(0xffffffffu, a, 1);
        a += __shfl_xor_sync(0xffffffffu, a, 2);
        a += __shfl_xor_sync(0xffffffffu, a, 4);
        if (sub == 0) out[t] = scale / sqrtf(a + eps);
    }
}

// ---------------------------------------------------------------------------- T of every chunk

constexpr int MS = DC + 4;       // row stride of fp32 tiles
constexpr int PREP_THREADS = 256;

// four numbers of a row as three rows of bf16
__device__ __forceinline__ void store_parts(bf16* p, float4 x) {
    uint2 p0, p1, p2;
    split3(x.x, x.y, p0.x, p1.x, p2.x);
    split3(x.z, x.w, p0.y, p1.y, p2.y);
    *(uint2*)p = p0;
    *(uint2*)(p + DC * TS) = p1;
    *(uint2*)(p + 2 * DC * TS) = p2;
}

// I + A is inverted in place: diagonal blocks of 16 by forward substitution, a column per lane, then the blocks below them,
// X21 = -X22 (A21 X11), first of 16, then of 32.
__global__ void __launch_bounds__(PREP_THREADS, 4) k_delta_prep(const __grid_constant__ DeltaChunkP P) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) double sb[DC];
    __shared__ __align__(16) float sr[DC], sbeta[DC], sgrow[DC];
    const int dpr = (P.D.dp + 31) & ~31, KS = dpr + 8, dvr = P.nvt * 16, VS = dvr + 8, per = P.D.H / P.D.G;
    float* sA = (float*)smem;                 // [64][MS]
    float* sT = sA + DC * MS;                 // [32][36]
    bf16* sP = (bf16*)smem;                   // [3][64][TS]: parts of T, once its numbers are in registers
    bf16* sk = sP + 3 * DC * TS;              // keys, then values, then keys again
    bf16* sv = sk;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int h = blockIdx.y, hq = h / per;
    const Chunk c = chunk_of(P, blockIdx.x);
    const long at = (long)blockIdx.x * P.D.H + h;
    load_rows(sk, KS, dpr / 8, P.k, c, P.ld, hq * P.D.dp, P.D.dp);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (warp == 0) log_sums(P, c, h, lane, sb);
    if (tid >= 64 && tid < 128) sbeta[tid - 64] = tid - 64 < c.rows ? P.beta[(c.row0 + tid - 64) * P.ldb + h] : 0.0f;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    row_norms(sk, KS, dpr / 8, P.D.eps, 1.0f, sr);
    if (h == hq * per) {                      // the keys as the update of the state takes them
        uint4* out = P.Kf + ((long)blockIdx.x * P.D.G + hq) * P.nkt * 4 * 32 + lane;
        for (int e = warp; e < P.nkt * 4; e += PREP_THREADS / 32) {
            unsigned r[4];
            ldsm4t(r, sk + ((e & 3) * 16 + (lane & 15)) * KS + (e >> 2) * 16 + (lane >> 4) * 8);
            out[e * 32] = make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
    const int m = warp & 3;      // k_i . k_j: rows 16 m + g (+ 8), columns 16 n + 2 tg (+ 1, + 8, + 9) of every other n up to m
    float a[2][2][4];
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) a[n][0][e] = a[n][1][e] = 0.0f;
    for (int kk = 0; kk < dpr / 16; kk++) {
        unsigned x[4];
        ldsm4(x, sk + (m * 16 + (lane & 15)) * KS + kk * 16 + (lane >> 4) * 8);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int col = 2 * n + (warp >> 2);
            if (col > m) break;
            unsigned r[4];
            ldsm4(r, sk + (col * 16 + (lane & 7) + ((lane >> 4) << 3)) * KS + kk * 16 + ((lane >> 3) & 1) * 8);
            mma16816(a[n][0], x, r[0], r[1]);
            mma16816(a[n][1], x, r[2], r[3]);
        }
    }
    __syncthreads();
    load_rows(sv, VS, dvr / 8, P.v, c, P.ld, h * P.D.dvp, P.D.dvp);
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int n = 0; n < 2; n++) {
        const int col = 2 * n + (warp >> 2);
        if (col > m) break;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int i = m * 16 + g + ((e >> 1) & 1) * 8, j = col * 16 + (e >> 2) * 8 + 2 * tg + (e & 1);
            sA[i * MS + j] = j < i ? a[n][e >> 2][e & 3] * sbeta[i] * sr[i] * sr[j] * exp2f((float)(sb[i] - sb[j])) : 0.0f;
        }
    }
    if (tid < DC) {
        float* vec = P.vec + at * DVEC;
        sgrow[tid] = exp2f((float)sb[tid]) * sr[tid];
        vec[tid] = exp2f((float)(sb[DC - 1] - sb[tid])) * sr[tid];
        if (tid == 0) vec[DC] = exp2f((float)sb[DC - 1]);
    }
    __syncthreads();
    if (warp < 4 && lane < 16) {
        float* d = sA + warp * 16 * MS + warp * 16;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = i == lane ? 1.0f : 0.0f;
#pragma unroll
        for (int k = 0; k < 15; k++)
#pragma unroll
            for (int i = k + 1; i < 16; i++) x[i] = fmaf(-d[i * MS + k], x[k], x[i]);
        __syncwarp(0xffffu);
#pragma unroll
        for (int i = 0; i < 16; i++) d[i * MS + lane] = x[i];
    }
    __syncthreads();
    {
        const int p = tid >> 7, i = (tid >> 3) & 15, j = (tid & 7) * 2, r = 32 * p + 16 + i, q = 32 * p;
        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const float x = sA[r * MS + q + k];
            const float2 y = *(const float2*)(sA + (q + k) * MS + q + j);
            s0 = fmaf(x, y.x, s0);
            s1 = fmaf(x, y.y, s1);
        }
        *(float2*)(sT + (p * 16 + i) * 36 + j) = make_float2(s0, s1);
        __syncthreads();
        s0 = s1 = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const float x = -sA[r * MS + q + 16 + k];
            const float2 y = *(const float2*)(sT + (p * 16 + k) * 36 + j);
            s0 = fmaf(x, y.x, s0);
            s1 = fmaf(x, y.y, s1);
        }
        *(float2*)(sA + r * MS + q + j) = make_float2(s0, s1);
        *(float2*)(sA + (q + i) * MS + q + 16 + j) = make_float2(0, 0);
    }
    __syncthreads();
    {
        const int i = tid >> 3, j = (tid & 7) * 4;
        float4 s = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 32; k++) {
            const float x = sA[(32 + i) * MS + k];
            const float4 y = *(const float4*)(sA + k * MS + j);
            s.x = fmaf(x, y.x, s.x); s.y = fmaf(x, y.y, s.y); s.z = fmaf(x, y.z, s.z); s.w = fmaf(x, y.w, s.w);
        }
        *(float4*)(sT + i * 36 + j) = s;
        __syncthreads();
        s = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 32; k++) {
            const float x = -sA[(32 + i) * MS + 32 + k];
            const float4 y = *(const float4*)(sT + k * 36 + j);
            s.x = fmaf(x, y.x, s.x); s.y = fmaf(x, y.y, s.y); s.z = fmaf(x, y.z, s.z); s.w = fmaf(x, y.w, s.w);
        }
        *(float4*)(sA + (32 + i) * MS + j) = s;
        *(float4*)(sA + i * MS + 32 + j) = make_float4(0, 0, 0, 0);
    }
    __syncthreads();
    {   // parts of T = (I + A)^-1 diag(beta), over its numbers
        float4 T[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int e = tid + u * PREP_THREADS, j = (e & 15) * 4;
            const float4 x = *(const float4*)(sA + (e >> 4) * MS + j), be = *(const float4*)(sbeta + j);
            T[u] = make_float4(x.x * be.x, x.y * be.y, x.z * be.z, x.w * be.w);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int e = tid + u * PREP_THREADS;
            store_parts(sP + (e >> 4) * TS + (e & 15) * 4, T[u]);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    for (int vt = warp; vt < P.nvt; vt += PREP_THREADS / 32) {       // U0, transposed
        float4* out = P.U + (at * P.nvt + vt) * 8 * 32 + lane;
        unsigned x[4][4];
#pragma unroll
        for (int j = 0; j < 4; j++) ldsm4t(x[j], sv + (j * 16 + (lane >> 4) * 8 + (lane & 7)) * VS + vt * 16 + ((lane >> 3) & 1) * 8);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float d[3][4];
#pragma unroll
            for (int p = 0; p < 3; p++) {
                d[p][0] = d[p][1] = d[p][2] = d[p][3] = 0.0f;
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++) {
                    if (4 * k2 > i) break;
                    unsigned r[4];
                    ldsm4(r, sP + (p * DC + i * 8 + (lane & 7)) * TS + k2 * 32 + (lane >> 3) * 8);
                    mma16816(d[p], x[2 * k2], r[0], r[1]);
                    if (4 * k2 + 2 <= i) mma16816(d[p], x[2 * k2 + 1], r[2], r[3]);
                }
            }
            out[i * 32] = make_float4(d[0][0] + (d[1][0] + d[2][0]), d[0][1] + (d[1][1] + d[2][1]), d[0][2] + (d[1][2] + d[2][2]),
                                      d[0][3] + (d[1][3] + d[2][3]));
        }
    }
    __syncthreads();
    load_rows(sk, KS, dpr / 8, P.k, c, P.ld, hq * P.D.dp, P.D.dp);
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int u = 0; u < 4; u++) {             // of T diag(e^b r): the parts add up to T again
        const int e = tid + u * PREP_THREADS, j = (e & 15) * 4;
        bf16* p = sP + (e >> 4) * TS + j;
        float x[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 2; i >= 0; i--) {
            const uint2 w = *(const uint2*)(p + i * DC * TS);
            x[0] += lo_f(w.x); x[1] += hi_f(w.x); x[2] += lo_f(w.y); x[3] += hi_f(w.y);
        }
        const float4 f = *(const float4*)(sgrow + j);
        store_parts(p, make_float4(x[0] * f.x, x[1] * f.y, x[2] * f.z, x[3] * f.w));
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    // W: tokens 16 m .., every other tile of channels, two tiles at a time
    for (int kt = warp >> 2; kt < P.nkt; kt += 4) {
        float d[2][2][4];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) d[u][0][e] = d[u][1][e] = 0.0f;
#pragma unroll
        for (int p = 2; p >= 0; p--)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j > m) break;
                unsigned x[4];
                ldsm4(x, sP + (p * DC + m * 16 + (lane & 15)) * TS + j * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (kt + 2 * u >= P.nkt) break;
                    unsigned r[4];
                    ldsm4t(r, sk + (j * 16 + (lane & 15)) * KS + (kt + 2 * u) * 16 + (lane >> 4) * 8);
                    mma16816(d[u][0], x, r[0], r[1]);
                    mma16816(d[u][1], x, r[2], r[3]);
                }
            }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            if (kt + 2 * u >= P.nkt) break;
            uint4 q0, q1, q2;
            split3(d[u][0][0], d[u][0][1], q0.x, q1.x, q2.x);
            split3(d[u][1][0], d[u][1][1], q0.y, q1.y, q2.y);
            split3(d[u][0][2], d[u][0][3], q0.z, q1.z, q2.z);
            split3(d[u][1][2], d[u][1][3], q0.w, q1.w, q2.w);
            uint4* o = P.W + ((at * P.nkt + kt + 2 * u) * 4 + m) * 3 * 32 + lane;
            o[0] = q0;
            o[32] = q1;
            o[64] = q2;
        }
    }
}
static size_t prep_smem(int dp, int nvt) {
    const int dpr = (dp + 31) & ~31, dvr = nvt * 16;
    return (size_t)3 * DC * TS * 2 + (size_t)DC * ((dpr > dvr ? dpr : dvr) + 8) * 2;
}
static_assert(DC * MS * 4 + 32 * 36 * 4 <= 3 * DC * TS * 2, "A and its products lie where the parts of T do later");

// ---------------------------------------------------------------------------- states

// NW warps, each with KT tiles of 16 key channels
template <int NW, int KT>
__global__ void __launch_bounds__(NW * 32, NW == 8 && KT == 1 ? 2 : 1) k_delta_states(const __grid_constant__ DeltaChunkP P) {
    constexpr int YS = DC + 8, NT = 8 / NW;              // blocks of 8 tokens that a warp makes U of
    // Keys are asked for a chunk ahead, or half a chunk where the registers of two CTAs an SM leave no room: with one CTA 16 heads of
    // 128 take as long, 32 heads or four sequences of 16 a fifth longer.
    constexpr bool AHEAD = NW != 8 || KT != 1;
    __shared__ __align__(16) float sY[NW * 16 * YS];     // shares of (W S^T)^T
    __shared__ __align__(16) bf16 sZ[3 * 16 * TS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int vt = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hq = h / (P.D.H / P.D.G);
    const int nchunk = P.first[b + 1] - P.first[b], dp = P.D.dp, dvp = P.D.dvp;
    if (nchunk == 0) return;
    const int active = (P.nkt + KT - 1) / KT;            // warps with key channels
    const int kt0 = warp * KT, va = vt * 16 + g, vb = va + 8;
    const long at0 = (long)P.first[b] * P.D.H + h;

    float s[2 * KT][4];              // S[va or vb][16 kt0 + 8 i + 2 tg + (0, 1)]
    const long sa = (long)va * dp + kt0 * 16 + 2 * tg, sd = sa + 8L * dp;
    float* S = P.Q.S[b] + (long)h * dvp * dp;
#pragma unroll
    for (int i = 0; i < 2 * KT; i++) {
        float2 a = make_float2(0, 0), d = a;
        if (kt0 * 16 + 8 * i < dp && va < dvp) a = *(const float2*)(S + sa + 8 * i);
        if (kt0 * 16 + 8 * i < dp && vb < dvp) d = *(const float2*)(S + sd + 8 * i);
        s[i][0] = a.x; s[i][1] = a.y; s[i][2] = d.x; s[i][3] = d.y;
    }
    // what a chunk needs beside the state, asked for as soon as the registers are free
    const uint4* Wp = P.W + (at0 * P.nkt + kt0) * 12 * 32 + lane;
    const uint4* Kp = P.Kf + (((long)P.first[b] * P.D.G + hq) * P.nkt + kt0) * 4 * 32 + lane;
    float4* Up = P.U + ((at0 * P.nvt + vt) * 8 + warp) * 32 + lane;
    const float* vp = P.vec + at0 * DVEC + warp * 8 + 2 * tg;
    uint4* S0 = P.S0 + ((at0 * P.nvt + vt) * P.nkt + kt0) * 3 * 32 + lane;
    uint4 w[KT][4][3], kf[KT][4];
    float4 u0[NT];
    float2 z[NT];
    float end = 0.0f;
    bool mine[KT];
#pragma unroll
    for (int kt = 0; kt < KT; kt++) mine[kt] = kt0 + kt < P.nkt;
    auto ask_w = [&]() {
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int p = 0; p < 3; p++)
                    if (mine[kt]) w[kt][t][p] = Wp[((kt * 4 + t) * 3 + p) * 32];
        Wp += (long)P.D.H * P.nkt * 12 * 32;
    };
    auto ask_k = [&]() {
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                if (mine[kt]) kf[kt][t] = Kp[(kt * 4 + t) * 32];
        Kp += (long)P.D.G * P.nkt * 4 * 32;
    };
    auto ask_u = [&]() {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            u0[n] = Up[n * NW * 32];
            z[n] = *(const float2*)(vp + n * NW * 8);
        }
        end = vp[DC - warp * 8 - 2 * tg];
        vp += (long)P.D.H * DVEC;
    };
#pragma unroll
    for (int kt = 0; kt < KT; kt++)
#pragma unroll
        for (int t = 0; t < 4; t++) {
            kf[kt][t] = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int p = 0; p < 3; p++) w[kt][t][p] = make_uint4(0, 0, 0, 0);
        }
    ask_w();
    ask_u();
    if (AHEAD) ask_k();
    for (int chunk = 0; chunk < nchunk; chunk++) {
        const bool more = chunk + 1 < nchunk;
        if (warp < active) {         // this warp's share of (W S^T)^T
            float y[8][4];
#pragma unroll
            for (int n = 0; n < 8; n++) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.0f;
#pragma unroll
            for (int kt = 0; kt < KT; kt++) {
                unsigned a[3][4];
                split3(s[2 * kt][0], s[2 * kt][1], a[0][0], a[1][0], a[2][0]);
                split3(s[2 * kt][2], s[2 * kt][3], a[0][1], a[1][1], a[2][1]);
                split3(s[2 * kt + 1][0], s[2 * kt + 1][1], a[0][2], a[1][2], a[2][2]);
                split3(s[2 * kt + 1][2], s[2 * kt + 1][3], a[0][3], a[1][3], a[2][3]);
                if (mine[kt]) {
#pragma unroll
                    for (int p = 0; p < 3; p++) S0[(kt * 3 + p) * 32] = make_uint4(a[p][0], a[p][1], a[p][2], a[p][3]);
                }
#pragma unroll
                for (int sum = 2; sum >= 0; sum--)       // parts i and j with i + j = sum, the smallest first
#pragma unroll
                    for (int p = 0; p <= sum; p++)
#pragma unroll
                        for (int t = 0; t < 4; t++) {
                            mma16816(y[2 * t], a[p], w[kt][t][sum - p].x, w[kt][t][sum - p].y);
                            mma16816(y[2 * t + 1], a[p], w[kt][t][sum - p].z, w[kt][t][sum - p].w);
                        }
            }
            if (more) ask_w();
            if (!AHEAD) ask_k();
            float* o = sY + (warp * 16 + g) * YS + 2 * tg;
#pragma unroll
            for (int n = 0; n < 8; n++) {
                *(float2*)(o + 8 * n) = make_float2(y[n][0], y[n][1]);
                *(float2*)(o + 8 * YS + 8 * n) = make_float2(y[n][2], y[n][3]);
            }
        }
        S0 += (long)P.D.H * P.nvt * P.nkt * 3 * 32;
        const float decay = end;
        __syncthreads();             // shares are there; nobody reads Z of the chunk before
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int t = (n * NW + warp) * 8 + 2 * tg;
            float2 ya = *(const float2*)(sY + g * YS + t), yb = *(const float2*)(sY + (8 + g) * YS + t);
#pragma unroll
            for (int k = 1; k < NW; k++)
                if (k < active) {
                    const float2 xa = *(const float2*)(sY + (k * 16 + g) * YS + t), xb = *(const float2*)(sY + (k * 16 + 8 + g) * YS + t);
                    ya.x += xa.x; ya.y += xa.y; yb.x += xb.x; yb.y += xb.y;
                }
            const float4 u = make_float4(u0[n].x - ya.x, u0[n].y - ya.y, u0[n].z - yb.x, u0[n].w - yb.y);
            Up[n * NW * 32] = u;
            unsigned a, m, l;
            split3(u.x * z[n].x, u.y * z[n].y, a, m, l);
            *(unsigned*)(sZ + g * TS + t) = a;
            *(unsigned*)(sZ + (16 + g) * TS + t) = m;
            *(unsigned*)(sZ + (32 + g) * TS + t) = l;
            split3(u.z * z[n].x, u.w * z[n].y, a, m, l);
            *(unsigned*)(sZ + (8 + g) * TS + t) = a;
            *(unsigned*)(sZ + (24 + g) * TS + t) = m;
            *(unsigned*)(sZ + (40 + g) * TS + t) = l;
        }
        Up += (long)P.D.H * P.nvt * 8 * 32;
        if (more) ask_u();
        __syncthreads();             // Z is there, and the shares are used
        if (warp < active) {
            float d[3][2 * KT][4];
#pragma unroll
            for (int p = 0; p < 3; p++)
#pragma unroll
                for (int i = 0; i < 2 * KT; i++) d[p][i][0] = d[p][i][1] = d[p][i][2] = d[p][i][3] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < DC / 16; kk++) {
                unsigned za[3][4];
#pragma unroll
                for (int p = 0; p < 3; p++) ldsm4(za[p], sZ + (p * 16 + (lane & 15)) * TS + kk * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int kt = 0; kt < KT; kt++)
#pragma unroll
                    for (int p = 0; p < 3; p++) {
                        mma16816(d[p][2 * kt], za[p], kf[kt][kk].x, kf[kt][kk].y);
                        mma16816(d[p][2 * kt + 1], za[p], kf[kt][kk].z, kf[kt][kk].w);
                    }
            }
            if (AHEAD && more) ask_k();
#pragma unroll
            for (int i = 0; i < 2 * KT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[i][e] = fmaf(decay, s[i][e], d[0][i][e] + (d[1][i][e] + d[2][i][e]));
        }
    }
#pragma unroll
    for (int i = 0; i < 2 * KT; i++) {
        if (kt0 * 16 + 8 * i < dp && va < dvp) *(float2*)(S + sa + 8 * i) = make_float2(s[i][0], s[i][1]);
        if (kt0 * 16 + 8 * i < dp && vb < dvp) *(float2*)(S + sd + 8 * i) = make_float2(s[i][2], s[i][3]);
    }
}

template <int NW, int KT>
static int launch_states(const DeltaChunkP& P, cudaStream_t s) {
    k_delta_states<NW, KT><<<dim3(P.nvt, P.D.H, P.Q.n), NW * 32, 0, s>>>(P);
    return check_launch("lt_dn_delta_chunked (states)");
}

// ---------------------------------------------------------------------------- outputs

// NK: blocks of 16 key channels at most; a warp owns 16 value columns at a time
template <int NK, int NW>
struct DeltaOut {
    static constexpr int QS = NK * 16 + 8;
    static constexpr int SMEM = 2 * DC * QS * 2 + 3 * DC * TS * 2;
    static constexpr int CTAS = NK > 8 ? 1 : NW == 4 ? 4 : 2;       // of an SM
};

template <int NK, int NW>
__global__ void __launch_bounds__(NW * 32, DeltaOut<NK, NW>::CTAS) k_delta_out(const __grid_constant__ DeltaChunkP P) {
    constexpr int QS = DeltaOut<NK, NW>::QS;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) double sb[DC];
    __shared__ float sr[DC], srq[DC];
    bf16* sq = (bf16*)smem;
    bf16* sk = sq + DC * QS;
    bf16* sP = sk + DC * QS;                     // [3][64][TS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int h = blockIdx.y, hq = h / (P.D.H / P.D.G), dp = P.D.dp, dvp = P.D.dvp, nk = P.nkt;
    const Chunk c = chunk_of(P, blockIdx.x);
    const long at = (long)blockIdx.x * P.D.H + h;
    load_rows(sq, QS, NK * 2, P.q, c, P.ld, hq * dp, dp);
    load_rows(sk, QS, NK * 2, P.k, c, P.ld, hq * dp, dp);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (warp == 0) log_sums(P, c, h, lane, sb);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    row_norms(sk, QS, NK * 2, P.D.eps, 1.0f, sr);
    row_norms(sq, QS, NK * 2, P.D.eps, P.D.q_scale, srq);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 8 / NW; u++) {           // q_t . k_j: columns 8 i .. of all rows that see them
        const int i = NW == 8 ? (warp < 4 ? warp : 11 - warp) : (u == 0 ? warp : 7 - warp);
        float a[4][4];
#pragma unroll
        for (int m = 0; m < 4; m++) a[m][0] = a[m][1] = a[m][2] = a[m][3] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < NK; kk += 2) {
            if (kk >= nk) break;
            unsigned r[4];
            ldsm4(r, sk + (i * 8 + (lane & 7)) * QS + kk * 16 + (lane >> 3) * 8);
#pragma unroll
            for (int m = 0; m < 4; m++) {
                if (2 * m + 1 < i) continue;
#pragma unroll
                for (int k1 = 0; k1 < 2; k1++) {
                    unsigned x[4];
                    ldsm4(x, sq + (m * 16 + (lane & 15)) * QS + (kk + k1) * 16 + (lane >> 4) * 8);
                    mma16816(a[m], x, r[2 * k1], r[2 * k1 + 1]);
                }
            }
        }
        const int j = i * 8 + 2 * tg;
        const double bj0 = sb[j], bj1 = sb[j + 1];
        const float r0 = sr[j], r1 = sr[j + 1];
#pragma unroll
        for (int m = 0; m < 4; m++) {
            if (2 * m + 1 < i) continue;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int t = m * 16 + g + 8 * e;
                const double bt = sb[t];
                const float x = j <= t ? a[m][2 * e] * r0 * exp2f((float)(bt - bj0)) : 0.0f;
                const float y = j + 1 <= t ? a[m][2 * e + 1] * r1 * exp2f((float)(bt - bj1)) : 0.0f;
                unsigned p0, p1, p2;
                split3(x, y, p0, p1, p2);
                *(unsigned*)(sP + t * TS + j) = p0;
                *(unsigned*)(sP + (DC + t) * TS + j) = p1;
                *(unsigned*)(sP + (2 * DC + t) * TS + j) = p2;
            }
        }
    }
    __syncthreads();
    for (int vt = warp; vt < P.nvt; vt += NW) {
        const uint4* S0 = P.S0 + (at * P.nvt + vt) * nk * 3 * 32 + lane;
        const float4* U = P.U + (at * P.nvt + vt) * 8 * 32 + lane;
        float acc[4][2][4], low[4][2][4];
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[m][n][e] = low[m][n][e] = 0.0f;
        uint4 next[3];
#pragma unroll
        for (int p = 0; p < 3; p++) next[p] = __ldcs(S0 + p * 32);
#pragma unroll
        for (int kk = 0; kk < NK; kk++) {
            if (kk >= nk) break;
            uint4 f[3];
#pragma unroll
            for (int p = 0; p < 3; p++) {
                f[p] = next[p];
                if (kk + 1 < nk) next[p] = __ldcs(S0 + ((kk + 1) * 3 + p) * 32);
            }
#pragma unroll
            for (int m = 0; m < 4; m++) {
                unsigned x[4];
                ldsm4(x, sq + (m * 16 + (lane & 15)) * QS + kk * 16 + (lane >> 4) * 8);
                mma16816(acc[m][0], x, f[0].x, f[0].z);
                mma16816(acc[m][1], x, f[0].y, f[0].w);
#pragma unroll
                for (int p = 2; p > 0; p--) {
                    mma16816(low[m][0], x, f[p].x, f[p].z);
                    mma16816(low[m][1], x, f[p].y, f[p].w);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const float fa = exp2f((float)sb[m * 16 + g]), fb = exp2f((float)sb[m * 16 + g + 8]);
#pragma unroll
            for (int n = 0; n < 2; n++) {
                acc[m][n][0] *= fa; acc[m][n][1] *= fa; acc[m][n][2] *= fb; acc[m][n][3] *= fb;
                low[m][n][0] *= fa; low[m][n][1] *= fa; low[m][n][2] *= fb; low[m][n][3] *= fb;
            }
        }
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            const float4 ua = __ldcs(U + 2 * kt * 32), ub = __ldcs(U + (2 * kt + 1) * 32);
            unsigned b0[2][3], b1[2][3];
            split3(ua.x, ua.y, b0[0][0], b0[0][1], b0[0][2]);
            split3(ub.x, ub.y, b1[0][0], b1[0][1], b1[0][2]);
            split3(ua.z, ua.w, b0[1][0], b0[1][1], b0[1][2]);
            split3(ub.z, ub.w, b1[1][0], b1[1][1], b1[1][2]);
#pragma unroll
            for (int m = kt; m < 4; m++) {
                unsigned x[3][4];
#pragma unroll
                for (int p = 0; p < 3; p++) ldsm4(x[p], sP + (p * DC + m * 16 + (lane & 15)) * TS + kt * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    mma16816(low[m][n], x[0], b0[n][2], b1[n][2]);
                    mma16816(acc[m][n], x[0], b0[n][0], b1[n][0]);
                    mma16816(low[m][n], x[2], b0[n][0], b1[n][0]);
                    mma16816(low[m][n], x[1], b0[n][1], b1[n][1]);
                    mma16816(low[m][n], x[0], b0[n][1], b1[n][1]);
                    mma16816(low[m][n], x[1], b0[n][0], b1[n][0]);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int t = m * 16 + g + 8 * e;
                if (t >= c.rows) continue;
                const float f = srq[t];
                float* o = P.o + (c.row0 + t) * P.ldo + (long)h * dvp + vt * 16 + 2 * tg;
#pragma unroll
                for (int n = 0; n < 2; n++)
                    if (vt * 16 + 8 * n < dvp)
                        *(float2*)(o + 8 * n) = make_float2(f * (acc[m][n][2 * e] + low[m][n][2 * e]), f * (acc[m][n][2 * e + 1] + low[m][n][2 * e + 1]));
            }
    }
}

template <int NK, int NW>
static int launch_delta_out(const DeltaChunkP& P, int chunks, cudaStream_t s) {
    static PerDeviceOnce once;
    LT_ONCE(once, LT_CUDA(cudaFuncSetAttribute(k_delta_out<NK, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, DeltaOut<NK, NW>::SMEM)));
    k_delta_out<NK, NW><<<dim3(chunks, P.D.H), NW * 32, DeltaOut<NK, NW>::SMEM, s>>>(P);
    return check_launch("lt_dn_delta_chunked (outputs)");
}

static long delta_chunks(const lt_dn_seqs* Q) {
    long n = 0;
    for (int i = 0; i < Q->n && i < LT_DN_SEQS; i++) n += ((long)Q->rows[i] + DC - 1) / DC;
    return n;
}
// fp32 elements of one chunk, all heads
static long delta_chunk_floats(const lt_dn_delta* D) {
    const long nkt = (D->dp + 15) / 16, nvt = (D->dvp + 15) / 16;
    return D->H * (nkt * 12 * 128 + nvt * nkt * 3 * 128 + nvt * 8 * 128 + DVEC) + D->G * nkt * 4 * 128;
}

}  // namespace dn
}  // namespace lt

using namespace lt;
using namespace lt::dn;

extern "C" long lt_dn_delta_chunked_ws(const lt_dn_delta* h_d, const lt_dn_seqs* h_q) {
    int rows = 0;      // of a call that would be refused: nothing
    if (delta_error(h_d) != nullptr || delta_seqs_error(h_q, &rows) != nullptr) return 0;
    return delta_chunks(h_q) * delta_chunk_floats(h_d);
}

extern "C" int lt_dn_delta_chunked(const void* q, const void* k, const void* v, int ld, const float* la, int ldla, const float* beta, int ldb, float* o,
                                   int ldo, const lt_dn_delta* h_d, const lt_dn_seqs* h_q, float* ws, void* stream) {
    int rows = 0;
    const char* bad = delta_error(h_d);
    if (bad == nullptr) bad = delta_seqs_error(h_q, &rows);
    LT_REQUIRE(bad == nullptr, "lt_dn_delta_chunked: %s", bad);
    LT_REQUIRE(q && k && v && la && beta && o && ws, "lt_dn_delta_chunked: null pointer");
    LT_REQUIRE(h_d->dp <= 256 && h_d->dvp <= 512, "lt_dn_delta_chunked: head sizes %d and %d are above 256 and 512", h_d->dp, h_d->dvp);
    LT_REQUIRE(ld >= h_d->G * h_d->dp && ld >= h_d->H * h_d->dvp && ldla >= h_d->H && ldb >= h_d->H && ldo >= h_d->H * h_d->dvp, "lt_dn_delta_chunked: ld=%d ldla=%d ldb=%d ldo=%d",
               ld, ldla, ldb, ldo);
    LT_REQUIRE(ld % 8 == 0 && ldo % 2 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o) && aligned16(ws), "lt_dn_delta_chunked: alignment");
    if (rows == 0) return LT_OK;
    DeltaChunkP P = {};
    P.q = (const bf16*)q; P.k = (const bf16*)k; P.v = (const bf16*)v; P.la = la; P.beta = beta; P.o = o;
    P.ld = ld; P.ldla = ldla; P.ldb = ldb; P.ldo = ldo; P.D = *h_d; P.Q = *h_q;
    for (int i = 0; i < P.Q.n; i++) P.first[i + 1] = P.first[i] + (int)(((long)P.Q.rows[i] + DC - 1) / DC);
    for (int i = P.Q.n; i < LT_DN_SEQS; i++) P.first[i + 1] = P.first[P.Q.n];
    const int chunks = P.first[P.Q.n];
    const long n = (long)chunks * P.D.H;
    P.nkt = (P.D.dp + 15) / 16;
    P.nvt = (P.D.dvp + 15) / 16;
    P.W = (uint4*)ws;
    P.S0 = P.W + n * P.nkt * 12 * 32;
    P.U = (float4*)(P.S0 + n * P.nvt * P.nkt * 3 * 32);
    P.Kf = (uint4*)(P.U + n * P.nvt * 8 * 32);
    P.vec = (float*)(P.Kf + (long)chunks * P.D.G * P.nkt * 4 * 32);
    cudaStream_t s = (cudaStream_t)stream;
    const int dp = P.D.dp;
    static PerDeviceOnce once;
    LT_ONCE(once, LT_CUDA(cudaFuncSetAttribute(k_delta_prep, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prep_smem(256, 32))));
    k_delta_prep<<<dim3(chunks, P.D.H), PREP_THREADS, prep_smem(dp, P.nvt), s>>>(P);
    int rc = check_launch("lt_dn_delta_chunked (prepare)");
    if (rc != LT_OK) return rc;
    rc = dp <= 64 ? launch_states<4, 1>(P, s) : dp <= 128 ? launch_states<8, 1>(P, s) : launch_states<8, 2>(P, s);
    if (rc != LT_OK) return rc;
    const bool few = P.D.dvp <= 64;
    if (dp <= 64) return few ? launch_delta_out<4, 4>(P, chunks, s) : launch_delta_out<4, 8>(P, chunks, s);
    if (dp <= 128) return few ? launch_delta_out<8, 4>(P, chunks, s) : launch_delta_out<8, 8>(P, chunks, s);
    return few ? launch_delta_out<16, 4>(P, chunks, s) : launch_delta_out<16, 8>(P, chunks, s);
}
