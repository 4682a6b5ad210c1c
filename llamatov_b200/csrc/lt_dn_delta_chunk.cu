// Gated delta rule over prompt rows in chunks of 64 tokens on the tensor cores (mma.sync m16n8k16, bf16 operands, fp32 sums).
// Of a chunk, with b_i the sum of its log decays up to and including token i, K and Q its raw rows, r_i = 1 / |k_i|, S the state
// it starts from:
//   A_ij = beta_i e^(b_i - b_j) r_i r_j k_i . k_j  (j < i),   T = (I + A)^-1 diag(beta)
//   U = T (V - diag(e^b r) K S^T)
//   S <- e^(b_end) S + U^T diag(r e^(b_end - b)) K
//   O = rq q_scale (diag(e^b) Q S^T + tril(Q K^T .* r_j e^(b_i - b_j)) U)
//
//   k_delta_prep    every chunk and head at once: T by forward substitution in blocks, in fp32
//   k_delta_states  walks the chunks: a CTA owns 16 value columns of one head of one sequence, its warps the key channels; the state
//                   stays in their accumulators, transposed (rows are value columns), so that it is the A operand of the next
//                   product as it stands; stores the state a chunk starts from, and U
//   k_delta_out     every chunk and head at once
//
// What is bf16 in memory (q, k) enters exactly.  Everything else is fp32: it enters as the sum of three bf16 (24 significant
// bits), three products against bf16 and six against another such sum, so that chunks are as exact as token order.  The
// products of the leading parts have accumulators of their own: the tensor cores cut sums off instead of rounding them, which costs
// up to 2^-24 of the accumulator at every step.
#include "lt_dn_delta.cuh"
#include "lt_dn_mma.cuh"

namespace lt {
namespace dn {

constexpr int DC = 64;                          // tokens of a chunk
constexpr float DLOG2E = 1.4426950408889634f;
constexpr int TS = DC + 8;                      // row stride of 64-column bf16 tiles: an odd number of 16-byte units
constexpr int DVEC = 2 * DC + 4;                // e^b r, r e^(b_end - b), e^(b_end)

struct DeltaChunkP {
    const bf16 *q, *k, *v;
    const float *la, *beta;
    float* o;
    bf16* T3;                // [chunk][H][3][64][64]
    float *vec, *S0, *U;     // [chunk][H]: [DVEC], [dvp][dp], [dvp][64]
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

// sums of a chunk's log decays (base 2), by one warp: doubles, so that differences are exact
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

// I + A is inverted in place: diagonal blocks of 16 by forward substitution, a column per lane, then the blocks below them,
// X21 = -X22 (A21 X11), first of 16, then of 32.
__global__ void __launch_bounds__(PREP_THREADS) k_delta_prep(const __grid_constant__ DeltaChunkP P) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) double sb[DC];
    __shared__ __align__(16) float sr[DC], sbeta[DC];
    const int dpr = (P.D.dp + 31) & ~31, KS = dpr + 8;
    float* sA = (float*)smem;                 // [64][MS]
    bf16* sk = (bf16*)(sA + DC * MS);
    float* sT = (float*)sk;                   // [32][36], once the keys are used
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int h = blockIdx.y, hq = h / (P.D.H / P.D.G);
    const Chunk c = chunk_of(P, blockIdx.x);
    const long at = (long)blockIdx.x * P.D.H + h;
    load_rows(sk, KS, dpr / 8, P.k, c, P.ld, hq * P.D.dp, P.D.dp);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (warp == 0) log_sums(P, c, h, lane, sb);
    if (tid >= 64 && tid < 128) sbeta[tid - 64] = tid - 64 < c.rows ? P.beta[(c.row0 + tid - 64) * P.ldb + h] : 0.0f;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    row_norms(sk, KS, dpr / 8, P.D.eps, 1.0f, sr);
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
        vec[tid] = exp2f((float)sb[tid]) * sr[tid];
        vec[DC + tid] = exp2f((float)(sb[DC - 1] - sb[tid])) * sr[tid];
        if (tid == 0) vec[2 * DC] = exp2f((float)sb[DC - 1]);
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
    bf16* out = P.T3 + at * 3 * DC * DC;
#pragma unroll
    for (int e = tid; e < DC * DC / 4; e += PREP_THREADS) {
        const int i = e >> 4, j = (e & 15) * 4;
        const float4 x = *(const float4*)(sA + i * MS + j), be = *(const float4*)(sbeta + j);
        uint2 t0, t1, t2;
        split3(x.x * be.x, x.y * be.y, t0.x, t1.x, t2.x);
        split3(x.z * be.z, x.w * be.w, t0.y, t1.y, t2.y);
        *(uint2*)(out + i * DC + j) = t0;
        *(uint2*)(out + DC * DC + i * DC + j) = t1;
        *(uint2*)(out + 2 * DC * DC + i * DC + j) = t2;
    }
}
static size_t prep_smem(int dp) {
    const size_t keys = (size_t)DC * (((dp + 31) & ~31) + 8) * 2, T = 32 * 36 * 4;
    return (size_t)DC * MS * 4 + (keys > T ? keys : T);
}

// ---------------------------------------------------------------------------- states

// NW warps, each with 16 KT key channels
template <int NW, int KT, int STAGES_>
struct DeltaStates {
    static constexpr int STAGES = STAGES_, DPR = NW * 16 * KT, KS = DPR + 8, VS = 24, YS = DC + 8;
    static constexpr int K_B = DC * KS * 2, T_B = 3 * DC * TS * 2, V_B = DC * VS * 2, VEC_B = DVEC * 4;
    static constexpr int STAGE = K_B + T_B + V_B + VEC_B;
    static constexpr int Y_B = NW * 16 * YS * 4, X_B = 3 * 16 * TS * 2;
    static constexpr int SMEM = STAGES * STAGE + Y_B + 2 * X_B;
    static_assert(STAGE % 16 == 0 && SMEM <= 227 * 1024, "shared memory");
};

template <int NW, int KT, int ST>
__global__ void __launch_bounds__(NW * 32) k_delta_states(const __grid_constant__ DeltaChunkP P) {
    using L = DeltaStates<NW, KT, ST>;
    constexpr int KS = L::KS, THREADS = NW * 32;
    extern __shared__ __align__(16) unsigned char smem[];
    float* sY = (float*)(smem + L::STAGES * L::STAGE);       // [warp][16][YS]
    bf16* sXp = (bf16*)((unsigned char*)sY + L::Y_B);        // [3][16][TS]
    bf16* sZp = (bf16*)((unsigned char*)sXp + L::X_B);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int v0 = blockIdx.x * 16, h = blockIdx.y, b = blockIdx.z, hq = h / (P.D.H / P.D.G);
    const int nchunk = P.first[b + 1] - P.first[b], dp = P.D.dp, dvp = P.D.dvp;
    if (nchunk == 0) return;
    const int active = (dp + 16 * KT - 1) / (16 * KT);       // warps with key channels
    const int cw = warp * 16 * KT;
    const int va = v0 + g, vb = va + 8;

    // this thread's 16-byte units of a stage: one column of the keys, one of T, one of the values; pointers go on by chunks
    constexpr int KU = L::DPR / 8, KR = THREADS / KU;        // units of a row of keys, rows of them at a time
    const int kt_ = tid / KU, kx = (tid % KU) * 8, tt = tid >> 3, tx = (tid & 7) * 8, vt = tid >> 1, vx = (tid & 1) * 8;
    const bool k_ok = kx < dp, v_ok = tid < 2 * DC && v0 + vx < dvp;
    const bf16* kp = P.k + ((long)P.Q.start[b] + kt_) * P.ld + (long)hq * dp + kx;
    const bf16* vp = P.v + ((long)P.Q.start[b] + vt) * P.ld + (long)h * dvp + v0 + vx;
    const long at0 = (long)P.first[b] * P.D.H + h;
    const bf16* tp = P.T3 + at0 * 3 * DC * DC + tid * 8;
    const float* cp = P.vec + at0 * DVEC + tid * 4;
    int left = P.Q.rows[b], next = 0;         // rows not yet asked for, chunk that is asked for next
    auto load = [&]() {
        if (next < nchunk) {
            unsigned char* st = smem + (next % L::STAGES) * L::STAGE;
            bf16* sk = (bf16*)st + kt_ * KS + kx;
            bf16* sT = (bf16*)(st + L::K_B) + tt * TS + tx;
#pragma unroll
            for (int i = 0; i < DC / KR; i++) {
                const bool ok = k_ok && kt_ + i * KR < left;
                cp16(sk + i * KR * KS, ok ? kp + (long)i * KR * P.ld : P.k, ok);
            }
#pragma unroll
            for (int i = 0; i < 3 * DC * 8 / THREADS; i++) cp16(sT + i * (THREADS / 8) * TS, tp + i * THREADS * 8, true);
            if (tid < 2 * DC) {
                const bool ok = v_ok && vt < left;
                cp16((bf16*)(st + L::K_B + L::T_B) + vt * L::VS + vx, ok ? vp : P.v, ok);
            }
            if (tid < DVEC / 4) cp16((float*)(st + L::K_B + L::T_B + L::V_B) + tid * 4, cp, true);
            kp += (long)DC * P.ld;
            vp += (long)DC * P.ld;
            tp += (long)P.D.H * 3 * DC * DC;
            cp += (long)P.D.H * DVEC;
            left -= DC;
            next++;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float s[2 * KT][4];              // S[va or vb][cw + 8 i + 2 tg + (0, 1)]
    const long sa = (long)va * dp + cw + 2 * tg, sd = (long)vb * dp + cw + 2 * tg;
    const bool a_ok = va < dvp, b_ok = vb < dvp;
    float* S = P.Q.S[b] + (long)h * dvp * dp;
#pragma unroll
    for (int i = 0; i < 2 * KT; i++) {
        float2 a = make_float2(0, 0), d = a;
        if (cw + 8 * i < dp && a_ok) a = *(const float2*)(S + sa + 8 * i);
        if (cw + 8 * i < dp && b_ok) d = *(const float2*)(S + sd + 8 * i);
        s[i][0] = a.x; s[i][1] = a.y; s[i][2] = d.x; s[i][3] = d.y;
    }
    auto keep = [&](float* to) {
#pragma unroll
        for (int i = 0; i < 2 * KT; i++) {
            if (cw + 8 * i < dp && a_ok) *(float2*)(to + sa + 8 * i) = make_float2(s[i][0], s[i][1]);
            if (cw + 8 * i < dp && b_ok) *(float2*)(to + sd + 8 * i) = make_float2(s[i][2], s[i][3]);
        }
    };
    // operands that do not wait for the state are read ahead of the barrier that the state's own share waits at
    auto keys = [&](unsigned (&r)[KT][4][4], const bf16* sk) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int n = 0; n < 4; n++)
                ldsm4(r[kt][n], sk + (n * 16 + (lane & 7) + ((lane >> 4) << 3)) * KS + cw + kt * 16 + ((lane >> 3) & 1) * 8);
    };
#pragma unroll
    for (int i = 0; i < L::STAGES - 1; i++) load();
    asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 2) : "memory");
    __syncthreads();
    unsigned kf[KT][4][4];
    keys(kf, (const bf16*)smem);
    float* S0 = P.S0 + at0 * dvp * dp;
    float* U = P.U + at0 * dvp * DC;
    for (int chunk = 0; chunk < nchunk; chunk++) {
        const unsigned char* st = smem + (chunk % L::STAGES) * L::STAGE;
        const bf16* sk = (const bf16*)st;
        const bf16* sT = (const bf16*)(st + L::K_B);
        const bf16* sv = (const bf16*)(st + L::K_B + L::T_B);
        const float* sc = (const float*)(st + L::K_B + L::T_B + L::V_B);
        if (warp < active) {         // this warp's share of (K S^T)^T
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
#pragma unroll
                for (int p = 2; p >= 0; p--)
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        mma16816(y[2 * n], a[p], kf[kt][n][0], kf[kt][n][1]);
                        mma16816(y[2 * n + 1], a[p], kf[kt][n][2], kf[kt][n][3]);
                    }
            }
            float* o = sY + (warp * 16 + g) * L::YS + 2 * tg;
#pragma unroll
            for (int n = 0; n < 8; n++) {
                *(float2*)(o + 8 * n) = make_float2(y[n][0], y[n][1]);
                *(float2*)(o + 8 * L::YS + 8 * n) = make_float2(y[n][2], y[n][3]);
            }
        }
        keep(S0);
        S0 += (long)P.D.H * dvp * dp;
        __syncthreads();             // shares are there; nobody works on the chunk before
        load();
#pragma unroll
        for (int e = tid; e < 256; e += THREADS) {       // X = V - e^b r (K S^T), transposed
            const int v = e >> 4, t = (e & 15) * 4;
            float4 y = *(const float4*)(sY + v * L::YS + t);
#pragma unroll
            for (int w = 1; w < NW; w++)
                if (w < active) {
                    const float4 z = *(const float4*)(sY + (w * 16 + v) * L::YS + t);
                    y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
                }
            const float4 f = *(const float4*)(sc + t);
            uint2 a, d, l;
            split3(fmaf(-f.x, y.x, to_f(sv[t * L::VS + v])), fmaf(-f.y, y.y, to_f(sv[(t + 1) * L::VS + v])), a.x, d.x, l.x);
            split3(fmaf(-f.z, y.z, to_f(sv[(t + 2) * L::VS + v])), fmaf(-f.w, y.w, to_f(sv[(t + 3) * L::VS + v])), a.y, d.y, l.y);
            *(uint2*)(sXp + v * TS + t) = a;
            *(uint2*)(sXp + (16 + v) * TS + t) = d;
            *(uint2*)(sXp + (32 + v) * TS + t) = l;
        }
        unsigned kb[4][KT][4];       // the keys again, as rows of tokens
#pragma unroll
        for (int kk = 0; kk < 4; kk++)
#pragma unroll
            for (int i = 0; i < KT; i++) ldsm4t(kb[kk][i], sk + (kk * 16 + (lane & 15)) * KS + cw + i * 16 + (lane >> 4) * 8);
#pragma unroll
        for (int u = 0; u < 8 / NW; u++) {       // U^T = X^T T^T: tokens 8 i ..; warps that share a scheduler have as much together
            const int i = NW == 8 ? (warp < 4 ? warp : 11 - warp) : (u == 0 ? warp : 7 - warp);
            unsigned tb[3][2][4];
#pragma unroll
            for (int p = 0; p < 3; p++)
#pragma unroll
                for (int k2 = 0; k2 < 2; k2++)
                    if (4 * k2 <= i) ldsm4(tb[p][k2], sT + (p * DC + i * 8 + (lane & 7)) * TS + k2 * 32 + (lane >> 3) * 8);
            if (u == 0) __syncthreads();         // X is there
            float d[6][4];
#pragma unroll
            for (int p = 0; p < 6; p++) d[p][0] = d[p][1] = d[p][2] = d[p][3] = 0.0f;
#pragma unroll
            for (int kt = 0; kt < 4; kt++) {
                if (2 * kt > i) break;
                unsigned xa[3][4];
#pragma unroll
                for (int p = 0; p < 3; p++) ldsm4(xa[p], sXp + (p * 16 + (lane & 15)) * TS + kt * 16 + (lane >> 4) * 8);
                const int lo = 2 * (kt & 1);
                mma16816(d[0], xa[0], tb[0][kt >> 1][lo], tb[0][kt >> 1][lo + 1]);
                mma16816(d[1], xa[0], tb[1][kt >> 1][lo], tb[1][kt >> 1][lo + 1]);
                mma16816(d[2], xa[1], tb[0][kt >> 1][lo], tb[0][kt >> 1][lo + 1]);
                mma16816(d[3], xa[0], tb[2][kt >> 1][lo], tb[2][kt >> 1][lo + 1]);
                mma16816(d[4], xa[1], tb[1][kt >> 1][lo], tb[1][kt >> 1][lo + 1]);
                mma16816(d[5], xa[2], tb[0][kt >> 1][lo], tb[0][kt >> 1][lo + 1]);
            }
            const int t = i * 8 + 2 * tg;
            const float2 z = *(const float2*)(sc + DC + t);
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = d[0][e] + ((d[1][e] + d[2][e]) + (d[3][e] + (d[4][e] + d[5][e])));
            unsigned a, m, l;
            split3(x[0] * z.x, x[1] * z.y, a, m, l);
            *(unsigned*)(sZp + g * TS + t) = a;
            *(unsigned*)(sZp + (16 + g) * TS + t) = m;
            *(unsigned*)(sZp + (32 + g) * TS + t) = l;
            split3(x[2] * z.x, x[3] * z.y, a, m, l);
            *(unsigned*)(sZp + (8 + g) * TS + t) = a;
            *(unsigned*)(sZp + (24 + g) * TS + t) = m;
            *(unsigned*)(sZp + (40 + g) * TS + t) = l;
            if (a_ok) *(float2*)(U + (long)va * DC + t) = make_float2(x[0], x[1]);
            if (b_ok) *(float2*)(U + (long)vb * DC + t) = make_float2(x[2], x[3]);
        }
        U += (long)P.D.H * dvp * DC;
        const float end = sc[2 * DC];
        asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 2) : "memory");
        __syncthreads();             // Z is there, and the next chunk
        if (chunk + 1 < nchunk) keys(kf, (const bf16*)(smem + ((chunk + 1) % L::STAGES) * L::STAGE));
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
                for (int p = 0; p < 3; p++) ldsm4(za[p], sZp + (p * 16 + (lane & 15)) * TS + kk * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int i = 0; i < KT; i++)
#pragma unroll
                    for (int p = 0; p < 3; p++) {
                        mma16816(d[p][2 * i], za[p], kb[kk][i][0], kb[kk][i][1]);
                        mma16816(d[p][2 * i + 1], za[p], kb[kk][i][2], kb[kk][i][3]);
                    }
            }
#pragma unroll
            for (int i = 0; i < 2 * KT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[i][e] = fmaf(end, s[i][e], d[0][i][e] + (d[1][i][e] + d[2][i][e]));
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    keep(S);
}

template <int NW, int KT, int ST>
static int launch_states(const DeltaChunkP& P, cudaStream_t s) {
    using L = DeltaStates<NW, KT, ST>;
    static PerDeviceOnce once;
    if (once.first()) LT_CUDA(cudaFuncSetAttribute(k_delta_states<NW, KT, ST>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM));
    k_delta_states<NW, KT, ST><<<dim3((P.D.dvp + 15) / 16, P.D.H, P.Q.n), NW * 32, L::SMEM, s>>>(P);
    return check_launch("lt_dn_delta_chunked (states)");
}

// ---------------------------------------------------------------------------- outputs

// NK: blocks of 16 key channels at most; a warp owns 8 value columns at a time
template <int NK, int NW>
struct DeltaOut {
    static constexpr int QS = NK * 16 + 8;
    static constexpr int SMEM = 2 * DC * QS * 2 + 3 * DC * TS * 2;
    static constexpr int CTAS = NW == 4 ? 4 : NK <= 8 ? 2 : 1;      // of an SM
};

template <int NK, int NW>
__global__ void __launch_bounds__(NW * 32, DeltaOut<NK, NW>::CTAS) k_delta_out(const __grid_constant__ DeltaChunkP P) {
    constexpr int QS = DeltaOut<NK, NW>::QS, KB = NK < 8 ? NK : 8;      // blocks of channels whose state is fetched together
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) double sb[DC];
    __shared__ float sr[DC], srq[DC];
    bf16* sq = (bf16*)smem;
    bf16* sk = sq + DC * QS;
    bf16* sP = sk + DC * QS;                     // [3][64][TS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tg = lane & 3;
    const int h = blockIdx.y, hq = h / (P.D.H / P.D.G), dp = P.D.dp, dvp = P.D.dvp, nk = (dp + 15) >> 4;
    const Chunk c = chunk_of(P, blockIdx.x);
    const long at = (long)blockIdx.x * P.D.H + h;
    load_rows(sq, QS, NK * 2, P.q, c, P.ld, hq * dp, dp);
    load_rows(sk, QS, NK * 2, P.k, c, P.ld, hq * dp, dp);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float* S0 = P.S0 + at * dvp * dp + 2 * tg;
    const float* U = P.U + at * dvp * DC + 2 * tg;
    float2 fS[KB][2], fU[4][2];
    auto fetch_state = [&](int v, int kb) {
#pragma unroll
        for (int k = 0; k < KB; k++) {
            const int x = (kb + k) * 16;
            const float* p = S0 + (long)(v + g) * dp + x;
            fS[k][0] = v < dvp && x < dp ? __ldcs((const float2*)p) : make_float2(0, 0);
            fS[k][1] = v < dvp && x + 8 < dp ? __ldcs((const float2*)(p + 8)) : make_float2(0, 0);
        }
    };
    auto fetch_u = [&](int v) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float* p = U + (long)(v + g) * DC + k * 16;
            fU[k][0] = v < dvp ? __ldcs((const float2*)p) : make_float2(0, 0);
            fU[k][1] = v < dvp ? __ldcs((const float2*)(p + 8)) : make_float2(0, 0);
        }
    };
    fetch_state(warp * 8, 0);
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
    for (int v0 = warp * 8; v0 < dvp; v0 += NW * 8) {
        if (v0 != warp * 8) fetch_state(v0, 0);
        float acc[4][4], low[4][4];
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[m][e] = low[m][e] = 0.0f;
#pragma unroll
        for (int kb = 0; kb < NK; kb += KB) {
            if (kb >= nk) break;
            if (kb > 0) fetch_state(v0, kb);
#pragma unroll
            for (int k = 0; k < KB; k++) {
                if (kb + k >= nk) break;
                unsigned b0[3], b1[3];
                split3(fS[k][0].x, fS[k][0].y, b0[0], b0[1], b0[2]);
                split3(fS[k][1].x, fS[k][1].y, b1[0], b1[1], b1[2]);
                if (k == 0 && kb == 0) fetch_u(v0);
#pragma unroll
                for (int m = 0; m < 4; m++) {
                    unsigned x[4];
                    ldsm4(x, sq + (m * 16 + (lane & 15)) * QS + (kb + k) * 16 + (lane >> 4) * 8);
                    mma16816(acc[m], x, b0[0], b1[0]);
                    mma16816(low[m], x, b0[2], b1[2]);
                    mma16816(low[m], x, b0[1], b1[1]);
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const float fa = exp2f((float)sb[m * 16 + g]), fb = exp2f((float)sb[m * 16 + g + 8]);
            acc[m][0] *= fa; acc[m][1] *= fa; acc[m][2] *= fb; acc[m][3] *= fb;
            low[m][0] *= fa; low[m][1] *= fa; low[m][2] *= fb; low[m][3] *= fb;
        }
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            unsigned b0[3], b1[3];
            split3(fU[kt][0].x, fU[kt][0].y, b0[0], b0[1], b0[2]);
            split3(fU[kt][1].x, fU[kt][1].y, b1[0], b1[1], b1[2]);
#pragma unroll
            for (int m = kt; m < 4; m++) {
                unsigned x[3][4];
#pragma unroll
                for (int p = 0; p < 3; p++) ldsm4(x[p], sP + (p * DC + m * 16 + (lane & 15)) * TS + kt * 16 + (lane >> 4) * 8);
                mma16816(acc[m], x[0], b0[0], b1[0]);
                mma16816(low[m], x[0], b0[2], b1[2]);
                mma16816(low[m], x[2], b0[0], b1[0]);
                mma16816(low[m], x[1], b0[1], b1[1]);
                mma16816(low[m], x[0], b0[1], b1[1]);
                mma16816(low[m], x[1], b0[0], b1[0]);
            }
        }
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int t = m * 16 + g + 8 * e;
                if (t >= c.rows) continue;
                const float f = srq[t];
                *(float2*)(P.o + (c.row0 + t) * P.ldo + (long)h * dvp + v0 + 2 * tg) =
                    make_float2(f * (acc[m][2 * e] + low[m][2 * e]), f * (acc[m][2 * e + 1] + low[m][2 * e + 1]));
            }
    }
}

template <int NK, int NW>
static int launch_delta_out(const DeltaChunkP& P, int chunks, cudaStream_t s) {
    static PerDeviceOnce once;
    if (once.first()) LT_CUDA(cudaFuncSetAttribute(k_delta_out<NK, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, DeltaOut<NK, NW>::SMEM));
    k_delta_out<NK, NW><<<dim3(chunks, P.D.H), NW * 32, DeltaOut<NK, NW>::SMEM, s>>>(P);
    return check_launch("lt_dn_delta_chunked (outputs)");
}

static long delta_chunks(const lt_dn_seqs* Q) {
    long n = 0;
    for (int i = 0; i < Q->n && i < LT_DN_SEQS; i++) n += (Q->rows[i] + DC - 1) / DC;
    return n;
}
// fp32 elements of one chunk and head
static long delta_chunk_floats(const lt_dn_delta* D) { return 3L * DC * DC / 2 + DVEC + (long)D->dvp * D->dp + (long)D->dvp * DC; }

}  // namespace dn
}  // namespace lt

using namespace lt;
using namespace lt::dn;

extern "C" long lt_dn_delta_chunked_ws(const lt_dn_delta* h_d, const lt_dn_seqs* h_q) {
    return delta_chunks(h_q) * h_d->H * delta_chunk_floats(h_d);
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
    for (int i = 0; i < P.Q.n; i++) P.first[i + 1] = P.first[i] + (P.Q.rows[i] + DC - 1) / DC;
    for (int i = P.Q.n; i < LT_DN_SEQS; i++) P.first[i + 1] = P.first[P.Q.n];
    const int chunks = P.first[P.Q.n];
    const long n = (long)chunks * P.D.H;
    P.T3 = (bf16*)ws;
    P.vec = ws + n * (3 * DC * DC / 2);
    P.S0 = P.vec + n * DVEC;
    P.U = P.S0 + n * P.D.dvp * P.D.dp;
    cudaStream_t s = (cudaStream_t)stream;
    const int dp = P.D.dp;
    static PerDeviceOnce once;
    if (once.first()) LT_CUDA(cudaFuncSetAttribute(k_delta_prep, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prep_smem(256)));
    k_delta_prep<<<dim3(chunks, P.D.H), PREP_THREADS, prep_smem(dp), s>>>(P);
    int rc = check_launch("lt_dn_delta_chunked (prepare)");
    if (rc != LT_OK) return rc;
    rc = dp <= 64 ? launch_states<4, 1, 2>(P, s) : dp <= 128 ? launch_states<8, 1, 3>(P, s) : launch_states<8, 2, 2>(P, s);
    if (rc != LT_OK) return rc;
    const bool few = P.D.dvp <= 64;
    if (dp <= 64) return few ? launch_delta_out<4, 4>(P, chunks, s) : launch_delta_out<4, 8>(P, chunks, s);
    if (dp <= 128) return few ? launch_delta_out<8, 4>(P, chunks, s) : launch_delta_out<8, 8>(P, chunks, s);
    return few ? launch_delta_out<16, 4>(P, chunks, s) : launch_delta_out<16, 8>(P, chunks, s);
}
