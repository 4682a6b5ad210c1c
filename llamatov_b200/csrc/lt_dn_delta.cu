// Gated delta rule in token order, state in fp32:
//   k^ = k / sqrt(sum k^2 + eps),  q^ = q_scale q / sqrt(sum q^2 + eps)
//   u_t = beta_t (v_t - a_t S k^_t),  S <- a_t S + u_t k^_t^T,  o_t = S q^_t
// Tokens are taken four at a time.  With g_i the product of the block's decays up to token i, everything that needs the state is a
// product with the state before the block, S k^_i and S q^_i, and the rest is numbers of the keys and queries alone:
//   u_i = beta_i (v_i - g_i S k^_i - sum_(j < i) (g_i / g_j) (k^_i . k^_j) u_j)
//   o_i = g_i S q^_i + sum_(j <= i) (g_i / g_j) (q^_i . k^_j) u_j,   S <- g_3 S + sum_j (g_3 / g_j) u_j k^_j^T
// so that the dependent chain (products, their sum over the lanes of a column, u, the update) is gone through once for four tokens.
// (The ratios are products of the decays between, no quotients.)
//
// k_delta_scan walks rows (fp32, short portions): a CTA owns 16 value columns of one head of one sequence.  Four warps hold the state,
// eight lanes a column, dp/8 key channels each in registers, and read keys and queries as they are in memory: the norms are part of
// the blocks' numbers.  Four warps make those numbers for the next batch, a warp per block, from rows that bulk copies have brought a
// batch earlier.  What bounds it is how many instructions a block is for one warp (four to five clocks each, as its scheduler has
// little else): products are of pairs (fma.rn.f32x2), and of S q^ a lane gets the one sum that it stores.
// (14 heads of 64 in fp32, 300 rows: 94 us token by token, staged without overlap; 47 in blocks with two columns a lane; 34 now.)
// k_delta_step is one token with its convolution and step size.
#include "lt_dn_delta.cuh"
#include "lt_tc.cuh"

namespace lt {
namespace dn {

using namespace tc;

struct DeltaScanP {
    const void *q, *k, *v;
    const float *la, *beta;
    float* o;
    int* status;
    int ld, ldla, ldb, ldo;
    lt_dn_delta D;
    lt_dn_seqs Q;
};

// two fp32 in a register pair, as the packed instructions take them
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float x, float y) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// a state row's share of a lane: VEC channels at a time, LN lanes side by side
template <int KPT, int VEC = 4, int LN = 8>
__device__ __forceinline__ void load_state(float (&s)[KPT], const float* row, int dp, int g) {
#pragma unroll
    for (int i = 0; i < KPT / 4; i++) {
        const int c = (i * 4 / VEC * LN + g) * VEC + i * 4 % VEC;
        float4 x = make_float4(0, 0, 0, 0);
        if (c < dp) x = *(const float4*)(row + c);
        s[4 * i] = x.x; s[4 * i + 1] = x.y; s[4 * i + 2] = x.z; s[4 * i + 3] = x.w;
    }
}
template <int KPT, int VEC = 4, int LN = 8>
__device__ __forceinline__ void store_state(const float (&s)[KPT], float* row, int dp, int g) {
#pragma unroll
    for (int i = 0; i < KPT / 4; i++) {
        const int c = (i * 4 / VEC * LN + g) * VEC + i * 4 % VEC;
        if (c < dp) *(float4*)(row + c) = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
    }
}

// The numbers of a block of four tokens, with r_i = 1 / |k_i| and rq_i = q_scale / |q_i|
struct __align__(16) DeltaBlock {
    float kk[4][4];      // beta_i (g_i / g_j) r_i r_j k_i . k_j, below the diagonal
    float qk[4][4];      // (g_i / g_j) rq_i r_j q_i . k_j, up to it
    float beta[4], bg[4], gq[4], z[4];      // beta_i; beta_i g_i r_i; g_i rq_i; (g_3 / g_i) r_i
    float end[4];        // g_3
};
constexpr int SCAN_COLS = 16;

__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// LN lanes a column, KPT channels a lane
template <typename T, int KPT, int LN>
struct DeltaScan {
    static constexpr int DP = LN * KPT, BT = DP <= 128 ? 16 : 8, NB = BT / 4;     // tokens and blocks of a batch
    static constexpr int CW = LN / 2, THREADS = (CW + 4) * 32;                    // warps that hold the state
    static constexpr int RAW = 2 * DP + SCAN_COLS;                                // elements of a row: q, k, v
    static constexpr int VEC = sizeof(T) == 2 && KPT >= 8 ? 8 : 4;                // channels of a load
    static constexpr int RAW_B = BT * RAW * (int)sizeof(T);
    static constexpr int SMEM = 3 * RAW_B + 2 * NB * (int)sizeof(DeltaBlock);
    static_assert(SMEM <= 227 * 1024 && RAW_B % 16 == 0, "shared memory");
};
template <typename T, int VEC>
__device__ __forceinline__ void load_pairs(f2 (&f)[VEC / 2], const T* p) {
    if (sizeof(T) == 4) {
        const float4 x = *(const float4*)p;
        f[0] = pack2(x.x, x.y);
        f[1] = pack2(x.z, x.w);
    } else {
        unsigned w[4];
        if (VEC == 8) *(uint4*)w = *(const uint4*)p;
        else *(uint2*)w = *(const uint2*)p;
#pragma unroll
        for (int i = 0; i < VEC / 2; i++) f[i] = pack2(lo_f(w[i]), hi_f(w[i]));
    }
}

template <typename T, int KPT, int LN>
__global__ void __launch_bounds__(DeltaScan<T, KPT, LN>::THREADS) k_delta_scan(const __grid_constant__ DeltaScanP P) {
    using L = DeltaScan<T, KPT, LN>;
    constexpr int DP = L::DP, BT = L::BT, NB = L::NB, VEC = L::VEC, ES = (int)sizeof(T);
    extern __shared__ __align__(128) unsigned char dsm[];
    __shared__ unsigned long long full[3];
    __shared__ int abort_word;
    const lt_dn_delta& D = P.D;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.y, b = blockIdx.z, hq = h / (D.H / D.G), v0 = blockIdx.x * SCAN_COLS;
    const int rows = P.Q.rows[b], batches = (rows + BT - 1) / BT;
    const long first = P.Q.start[b];
    if (rows == 0) return;
    volatile int* abort_flag = &abort_word;
    auto raw = [&](int n) { return (T*)(dsm + (n % 3) * L::RAW_B); };
    auto ready = [&](int n) { return (DeltaBlock*)(dsm + 3 * L::RAW_B) + (n & 1) * NB; };
    auto wait = [&](int n) {
        const unsigned bar = smem_u32(&full[n % 3]);
        bar_wait(bar_test(bar, (n / 3) & 1), bar, (n / 3) & 1, abort_flag, P.status);
    };
    // what no copy writes is zero: channels behind dp, columns behind dvp, tokens behind the last (or an earlier token's, whose beta is
    // taken for 0)
    for (int e = tid; e < 3 * L::RAW_B / 16; e += L::THREADS) ((uint4*)dsm)[e] = make_uint4(0, 0, 0, 0);
    if (tid == 0) {
        abort_word = 0;
        for (int i = 0; i < 3; i++) mbar_init(&full[i], NB);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();

    if (warp >= L::CW) {
        const int blk = warp - L::CW;
        // rows of the block: a lane copies a token's q, k or v
        const int cols = min(SCAN_COLS, D.dvp - v0), what = lane >> 2, tok = blk * 4 + (lane & 3);
        const T* src = what == 0 ? (const T*)P.q + (long)hq * D.dp : what == 1 ? (const T*)P.k + (long)hq * D.dp : (const T*)P.v + (long)h * D.dvp + v0;
        src += (first + tok) * P.ld;
        const unsigned to_place = (unsigned)((tok * L::RAW + what * DP) * ES), bytes = (unsigned)((what < 2 ? D.dp : cols) * ES);
        auto fetch = [&](int n) {
            if (blk >= NB || n >= batches || *abort_flag) return;
            const int count = max(0, min(4, rows - n * BT - blk * 4));
            const unsigned bar = smem_u32(&full[n % 3]);
            if (lane == 0) bar_expect_tx(bar, (unsigned)(count * (2 * D.dp + cols) * ES));
            __syncwarp();
            if (what < 3 && (lane & 3) < count) bulk_load(smem_u32(raw(n)) + to_place, src + (long)n * BT * P.ld, bytes, bar);
        };
        // decay and beta of the block's tokens in lanes 0 - 3, asked for a batch ahead
        float la = 0.0f, be = 0.0f, la_next = 0.0f, be_next = 0.0f;
        auto numbers = [&](int n) {
            const int t = n * BT + blk * 4 + (lane & 3);
            const bool ok = n < batches && blk < NB && t < rows;
            la = la_next;
            be = be_next;
            la_next = ok ? P.la[(first + t) * P.ldla + h] : 0.0f;
            be_next = ok ? P.beta[(first + t) * P.ldb + h] : 0.0f;
        };
        auto make = [&](int n) {
            if (blk >= NB) return;
            const float decay = expf(la);
            const T* in = raw(n) + blk * 4 * L::RAW;
            float x[32];             // k_i . k_j (j < i), q_i . k_j (j <= i), q_i . q_i, k_i . k_i
#pragma unroll
            for (int i = 0; i < 32; i++) x[i] = 0.0f;
#pragma unroll
            for (int c = 0; c < DP / 32; c++) {
                float q[4], k[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    q[i] = to_f(in[i * L::RAW + lane + 32 * c]);
                    k[i] = to_f(in[i * L::RAW + DP + lane + 32 * c]);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
#pragma unroll
                    for (int j = 0; j <= i; j++) {
                        if (j < i) x[i * (i - 1) / 2 + j] = fmaf(k[i], k[j], x[i * (i - 1) / 2 + j]);
                        x[6 + i * (i + 1) / 2 + j] = fmaf(q[i], k[j], x[6 + i * (i + 1) / 2 + j]);
                    }
                    x[16 + i] = fmaf(q[i], q[i], x[16 + i]);
                    x[20 + i] = fmaf(k[i], k[i], x[20 + i]);
                }
            }
            // sums over the lanes: at every step a lane hands on one half of its values and keeps the other, and ends with number `lane`
#pragma unroll
            for (int s = 16; s > 0; s >>= 1)
#pragma unroll
                for (int i = 0; i < s; i++) {
                    const bool up = (lane & s) != 0;
                    const float give = up ? x[i] : x[i + s], have = up ? x[i + s] : x[i];
                    x[i] = have + __shfl_xor_sync(0xffffffffu, give, s);
                }
            const float dot = x[0];
            const float norm = (lane < 20 ? D.q_scale : 1.0f) / sqrtf(dot + D.eps);      // of lanes 16 - 23
            const int i = (lane >> 2) & 3, j = lane & 3;
            float a[4];
#pragma unroll
            for (int m = 0; m < 4; m++) a[m] = __shfl_sync(0xffffffffu, decay, m);
            float ratio = 1.0f, to = 1.0f, rest = 1.0f;      // g_i / g_j, g_j, g_3 / g_j
#pragma unroll
            for (int m = 0; m < 4; m++) {
                if (m > j && m <= i) ratio *= a[m];
                if (m <= j) to *= a[m];
                if (m > j) rest *= a[m];
            }
            const bool kk = lane < 16;
            const int at = kk ? (j < i ? i * (i - 1) / 2 + j : 0) : 6 + (j <= i ? i * (i + 1) / 2 + j : 0);
            const float d = __shfl_sync(0xffffffffu, dot, at);
            const float ni = __shfl_sync(0xffffffffu, norm, (kk ? 20 : 16) + i), rj = __shfl_sync(0xffffffffu, norm, 20 + j);
            const float qj = __shfl_sync(0xffffffffu, norm, 16 + j);
            const float bi = __shfl_sync(0xffffffffu, be, i), bj = __shfl_sync(0xffffffffu, be, j);
            float* o = (float*)(ready(n) + blk);
            o[lane] = (kk ? j < i : j <= i) ? ratio * (d * ni * rj) * (kk ? bi : 1.0f) : 0.0f;
            if (lane < 16) o[32 + lane] = i == 0 ? bj : i == 1 ? bj * to * rj : i == 2 ? to * qj : rest * rj;
            if (lane == 19) o[48] = to;
        };
        fetch(0);
        fetch(1);
        numbers(0);
        numbers(1);
        wait(0);
        make(0);
        __syncthreads();
        for (int n = 0; n < batches; n++) {      // while the others walk batch n
            fetch(n + 2);
            numbers(n + 2);
            if (n + 1 < batches) {
                wait(n + 1);
                make(n + 1);
            }
            __syncthreads();
        }
    } else {
        const int g = tid & (LN - 1), cl = tid / LN, col = v0 + cl, mine = g & 3;      // mine: the token whose output this lane has
        const bool col_ok = col < D.dvp;
        float* Srow = P.Q.S[b] + ((long)h * D.dvp + (col_ok ? col : 0)) * D.dp;
        f2 s[KPT / 2];
        {
            float t[KPT];
            load_state<KPT, VEC, LN>(t, Srow, D.dp, g);
#pragma unroll
            for (int i = 0; i < KPT / 2; i++) s[i] = pack2(t[2 * i], t[2 * i + 1]);
        }
        float* o = P.o + (first + mine) * P.ldo + (long)h * D.dvp + col;
        __syncthreads();
        for (int n = 0; n < batches; n++) {
            wait(n);
            const T* qb = raw(n) + g * VEC;
            const T* vb = raw(n) + 2 * DP + cl;
            const DeltaBlock* R = ready(n);
            int left = rows - n * BT;
#pragma unroll 1
            for (int blk = 0; blk < NB && left > 0; blk++) {
                f2 x[8];             // S k_i, then S q_i, in halves
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = 0ull;
#pragma unroll
                for (int c = 0; c < KPT / VEC; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        f2 k[VEC / 2], q[VEC / 2];
                        load_pairs<T, VEC>(k, qb + i * L::RAW + DP + c * LN * VEC);
                        load_pairs<T, VEC>(q, qb + i * L::RAW + c * LN * VEC);
#pragma unroll
                        for (int e = 0; e < VEC / 2; e++) {
                            x[i] = fma2(k[e], s[c * VEC / 2 + e], x[i]);
                            x[4 + i] = fma2(q[e], s[c * VEC / 2 + e], x[4 + i]);
                        }
                    }
                // the block's numbers, read ahead of the shuffles, which nothing is moved across
                const float4 be = *(const float4*)R->beta, bg = *(const float4*)R->bg, z = *(const float4*)R->z, qk = *(const float4*)R->qk[mine];
                const float4 k1 = *(const float4*)R->kk[1], k2 = *(const float4*)R->kk[2], k3 = *(const float4*)R->kk[3];
                const float end = R->end[0], gq = R->gq[mine];
                const float v0_ = be.x * to_f(vb[0]), v1 = be.y * to_f(vb[L::RAW]), v2 = be.z * to_f(vb[2 * L::RAW]), v3 = be.w * to_f(vb[3 * L::RAW]);
                float p[4], r[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float a, c;
                    unpack2(x[i], a, c);
                    p[i] = a + c;
                    unpack2(x[4 + i], a, c);
                    r[i] = a + c;
                }
#pragma unroll
                for (int m = LN / 2; m > 0; m >>= 1) {
#pragma unroll
                    for (int i = 0; i < 4; i++) p[i] += __shfl_xor_sync(0xffffffffu, p[i], m);
                    if (m >= 4) {
#pragma unroll
                        for (int i = 0; i < 4; i++) r[i] += __shfl_xor_sync(0xffffffffu, r[i], m);
                    } else {
#pragma unroll
                        for (int i = 0; i < m; i++) {    // a lane ends with the sum of its own number
                            const bool up = (g & m) != 0;
                            const float give = up ? r[i] : r[i + m], have = up ? r[i + m] : r[i];
                            r[i] = have + __shfl_xor_sync(0xffffffffu, give, m);
                        }
                    }
                }
                const float u0 = fmaf(-bg.x, p[0], v0_);
                const float u1 = fmaf(-k1.x, u0, fmaf(-bg.y, p[1], v1));
                const float u2 = fmaf(-k2.y, u1, fmaf(-k2.x, u0, fmaf(-bg.z, p[2], v2)));
                const float u3 = fmaf(-k3.z, u2, fmaf(-k3.y, u1, fmaf(-k3.x, u0, fmaf(-bg.w, p[3], v3))));
                // above the diagonal the numbers are zero, and a later token's u, which need not be finite, is taken for zero too
                const float y = fmaf(qk.w, mine == 3 ? u3 : 0.0f, fmaf(qk.z, mine >= 2 ? u2 : 0.0f, fmaf(qk.y, mine >= 1 ? u1 : 0.0f, fmaf(qk.x, u0, gq * r[0]))));
                if (col_ok && g < 4 && mine < left) *o = y;
                const float w0 = z.x * u0, w1 = z.y * u1, w2 = z.z * u2, w3 = z.w * u3;
                const f2 w[4] = {pack2(w0, w0), pack2(w1, w1), pack2(w2, w2), pack2(w3, w3)}, end2 = pack2(end, end);
#pragma unroll
                for (int c = 0; c < KPT / VEC; c++) {
#pragma unroll
                    for (int e = c * VEC / 2; e < (c + 1) * VEC / 2; e++) s[e] = mul2(s[e], end2);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        f2 k[VEC / 2];
                        load_pairs<T, VEC>(k, qb + i * L::RAW + DP + c * LN * VEC);
#pragma unroll
                        for (int e = 0; e < VEC / 2; e++) s[c * VEC / 2 + e] = fma2(w[i], k[e], s[c * VEC / 2 + e]);
                    }
                }
                qb += 4 * L::RAW;
                vb += 4 * L::RAW;
                o += 4L * P.ldo;
                left -= 4;
                R++;
            }
            __syncthreads();
        }
        if (col_ok) {
            float t[KPT];
#pragma unroll
            for (int i = 0; i < KPT / 2; i++) unpack2(s[i], t[2 * i], t[2 * i + 1]);
            store_state<KPT, VEC, LN>(t, Srow, D.dp, g);
        }
    }
    if (*abort_flag) {               // a wait ran out: let copies in flight land before the CTA leaves
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {
        }
    }
}

template <typename T, int KPT, int LN>
static int launch_delta_scan(const DeltaScanP& P, cudaStream_t s) {
    using L = DeltaScan<T, KPT, LN>;
    static PerDeviceOnce once;
    LT_ONCE(once, LT_CUDA(cudaFuncSetAttribute(k_delta_scan<T, KPT, LN>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM)));
    k_delta_scan<T, KPT, LN><<<dim3((P.D.dvp + SCAN_COLS - 1) / SCAN_COLS, P.D.H, P.Q.n), L::THREADS, L::SMEM, s>>>(P);
    return check_launch("lt_dn_delta_rows");
}
template <typename T>
static int delta_scan_size(const DeltaScanP& P, cudaStream_t s) {
    if (P.D.dp <= 32) return launch_delta_scan<T, 4, 8>(P, s);
    if (P.D.dp <= 64) return launch_delta_scan<T, 8, 8>(P, s);
    if (P.D.dp <= 128) return launch_delta_scan<T, 16, 8>(P, s);
    if (P.D.dp <= 256) return launch_delta_scan<T, 16, 16>(P, s);
    return launch_delta_scan<T, 32, 16>(P, s);
}

// ---------------------------------------------------------------------------- one token

struct DeltaStepP {
    const void* u;
    const float *dt, *beta;
    void* ring;
    float *state, *o;
    int *len, *ticket;
    int C;
    lt_dn_delta D;
};

// CTA (x, h): 32 value columns of head h, eight lanes per column, dp / 8 key channels each in registers.  Every lane of a column
// has the whole column's share of the norms in reach, so five sums go over the lanes at once: S k, S q, k.k, q.q, k.q.
template <typename T, int KPT>
__global__ void __launch_bounds__(256) k_delta_step(const __grid_constant__ DeltaStepP P) {
    constexpr int DP = 8 * KPT;
    __shared__ __align__(16) float sk[DP], sq[DP];
    __shared__ float sv[32];
    const lt_dn_delta& D = P.D;
    const int tid = threadIdx.x, g = tid & 7, cl = tid >> 3;
    const int h = blockIdx.y, per = D.H / D.G, grp = h / per, col = blockIdx.x * 32 + cl;
    const bool col_ok = col < D.dvp;
    float s[KPT];
    float* row = P.state + ((long)h * D.dvp + (col_ok ? col : 0)) * D.dp;
    load_state<KPT>(s, row, D.dp, g);
    const int pos = *P.len, slot = pos % D.taps;
    const float a = expf(D.A[h] * softplus_f(P.dt[h] + D.dt_bias[h])), be = P.beta[h];
    // channel c after convolution and silu; the new input goes to its slot of the ring, which no reader of this step needs
    auto channel = [&](int c, bool keep) {
        const T u = ((const T*)P.u)[c];
        float v = D.conv_b[c];
        int r = slot;
        for (int k = 0; k < D.taps - 1; k++) {       // positions pos - taps + 1 .. pos - 1
            r = r + 1 == D.taps ? 0 : r + 1;
            if (pos - (D.taps - 1) + k >= 0) v = fmaf(D.conv[(long)k * P.C + c], to_f(((const T*)P.ring)[(long)r * P.C + c]), v);
        }
        v = fmaf(D.conv[(long)(D.taps - 1) * P.C + c], to_f(u), v);
        if (keep) ((T*)P.ring)[(long)slot * P.C + c] = u;
        return v * sigmoid_f(v);
    };
    const bool first = blockIdx.x == 0 && h == grp * per;
    for (int e = tid; e < 2 * DP + 32; e += 256) {
        if (e < 2 * DP) {
            const int c = e < DP ? e : e - DP;
            const float v = c < D.dp ? channel(D.H * D.dvp + (e < DP ? 0 : D.G * D.dp) + grp * D.dp + c, first) : 0.0f;
            if (e < DP) sk[c] = v;
            else sq[c] = v;
        } else {
            const int c = blockIdx.x * 32 + e - 2 * DP;
            sv[e - 2 * DP] = c < D.dvp ? channel(h * D.dvp + c, true) : 0.0f;
        }
    }
    __syncthreads();
    float Sk = 0.0f, Sq = 0.0f, kk = 0.0f, qq = 0.0f, kq = 0.0f;
#pragma unroll
    for (int i = 0; i < KPT / 4; i++) {
        const float4 k = *(const float4*)(sk + i * 32 + g * 4), q = *(const float4*)(sq + i * 32 + g * 4);
        Sk = fmaf(k.x, s[4 * i], fmaf(k.y, s[4 * i + 1], fmaf(k.z, s[4 * i + 2], fmaf(k.w, s[4 * i + 3], Sk))));
        Sq = fmaf(q.x, s[4 * i], fmaf(q.y, s[4 * i + 1], fmaf(q.z, s[4 * i + 2], fmaf(q.w, s[4 * i + 3], Sq))));
        kk = fmaf(k.x, k.x, fmaf(k.y, k.y, fmaf(k.z, k.z, fmaf(k.w, k.w, kk))));
        qq = fmaf(q.x, q.x, fmaf(q.y, q.y, fmaf(q.z, q.z, fmaf(q.w, q.w, qq))));
        kq = fmaf(k.x, q.x, fmaf(k.y, q.y, fmaf(k.z, q.z, fmaf(k.w, q.w, kq))));
    }
#pragma unroll
    for (int x = 1; x < 8; x <<= 1) {            // over the eight lanes of a column, the five sums side by side
        Sk += __shfl_xor_sync(0xffffffffu, Sk, x);
        Sq += __shfl_xor_sync(0xffffffffu, Sq, x);
        kk += __shfl_xor_sync(0xffffffffu, kk, x);
        qq += __shfl_xor_sync(0xffffffffu, qq, x);
        kq += __shfl_xor_sync(0xffffffffu, kq, x);
    }
    const float rk = 1.0f / sqrtf(kk + D.eps), rq = D.q_scale / sqrtf(qq + D.eps);
    const float u = be * fmaf(-a, Sk * rk, sv[cl]), uk = u * rk;
#pragma unroll
    for (int i = 0; i < KPT / 4; i++) {
        const float4 k = *(const float4*)(sk + i * 32 + g * 4);
        s[4 * i] = fmaf(a, s[4 * i], uk * k.x);
        s[4 * i + 1] = fmaf(a, s[4 * i + 1], uk * k.y);
        s[4 * i + 2] = fmaf(a, s[4 * i + 2], uk * k.z);
        s[4 * i + 3] = fmaf(a, s[4 * i + 3], uk * k.w);
    }
    if (col_ok) store_state<KPT>(s, row, D.dp, g);
    if (g == 0 && col_ok) P.o[(long)h * D.dvp + col] = rq * fmaf(a, Sq, uk * kq);
    if (tid == 0) {      // past the barrier: every thread of this CTA has read the position
        if (atomicAdd(P.ticket, 1) == (int)(gridDim.x * gridDim.y) - 1) {
            *P.ticket = 0;
            *P.len = pos + 1;
        }
    }
}

template <typename T>
static int launch_delta_step(const DeltaStepP& P, cudaStream_t s) {
    const dim3 grid((P.D.dvp + 31) / 32, P.D.H);
    if (P.D.dp <= 32) k_delta_step<T, 4><<<grid, 256, 0, s>>>(P);
    else if (P.D.dp <= 64) k_delta_step<T, 8><<<grid, 256, 0, s>>>(P);
    else if (P.D.dp <= 128) k_delta_step<T, 16><<<grid, 256, 0, s>>>(P);
    else if (P.D.dp <= 256) k_delta_step<T, 32><<<grid, 256, 0, s>>>(P);
    else k_delta_step<T, 64><<<grid, 256, 0, s>>>(P);
    return check_launch("lt_dn_delta_step");
}

// ---------------------------------------------------------------------------- host checks

const char* delta_error(const lt_dn_delta* D) {
    if (D == nullptr) return "null description";
    if (D->H <= 0 || D->G <= 0 || D->H % D->G || D->dp <= 0 || D->dvp <= 0) return "sizes (heads must be a multiple of the key heads)";
    if (D->dp % 8 || D->dvp % 8) return "padded sizes must be multiples of 8";
    if (D->dp > 512) return "a key size above 512";
    if (D->H > 65535) return "more than 65535 heads";
    if (!(D->eps > 0.0f)) return "eps must be positive";
    return nullptr;
}
const char* delta_seqs_error(const lt_dn_seqs* Q, int* rows) {
    if (Q == nullptr) return "null sequences";
    if (Q->n < 1 || Q->n > LT_DN_SEQS) return "number of sequences";
    *rows = 0;
    for (int i = 0; i < Q->n; i++) {
        if (Q->S[i] == nullptr || !aligned16(Q->S[i])) return "a state is null or not 16-byte aligned";
        if (Q->start[i] < 0 || Q->rows[i] < 0 || (long)Q->start[i] + Q->rows[i] > 0x7fffffffL) return "rows of a sequence";
        for (int j = 0; j < i; j++) {
            if (Q->S[j] == Q->S[i]) return "two sequences with one state";
            if (Q->rows[i] && Q->rows[j] && Q->start[i] < Q->start[j] + Q->rows[j] && Q->start[j] < Q->start[i] + Q->rows[i])
                return "two sequences share rows";
        }
        if (Q->rows[i] > *rows) *rows = Q->rows[i];
    }
    return nullptr;
}

}  // namespace dn
}  // namespace lt

using namespace lt;
using namespace lt::dn;

extern "C" int lt_dn_delta_rows(const void* q, const void* k, const void* v, int ld, const float* la, int ldla, const float* beta, int ldb, float* o,
                                int ldo, int f32, const lt_dn_delta* h_d, const lt_dn_seqs* h_q, void* stream) {
    int rows = 0;
    const char* bad = delta_error(h_d);
    if (bad == nullptr) bad = delta_seqs_error(h_q, &rows);
    LT_REQUIRE(bad == nullptr, "lt_dn_delta_rows: %s", bad);
    LT_REQUIRE(q && k && v && la && beta && o, "lt_dn_delta_rows: null pointer");
    LT_REQUIRE(ld >= h_d->G * h_d->dp && ld >= h_d->H * h_d->dvp && ldla >= h_d->H && ldb >= h_d->H && ldo >= h_d->H * h_d->dvp,
               "lt_dn_delta_rows: ld=%d ldla=%d ldb=%d ldo=%d", ld, ldla, ldb, ldo);
    LT_REQUIRE(ld % 8 == 0 && ldo % 2 == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(o), "lt_dn_delta_rows: alignment");
    if (rows == 0) return LT_OK;
    DeltaScanP P = {q, k, v, la, beta, o, device_status_ptr(), ld, ldla, ldb, ldo, *h_d, *h_q};
    LT_REQUIRE(P.status != nullptr, "lt_dn_delta_rows: status word unavailable");
    if (f32) return delta_scan_size<float>(P, (cudaStream_t)stream);
    return delta_scan_size<bf16>(P, (cudaStream_t)stream);
}

extern "C" int lt_dn_delta_step(const void* vkq, const float* dt, const float* beta, void* ring, float* S, float* o, int f32, int* len,
                                int* ticket, const lt_dn_delta* h_d, void* stream) {
    const char* bad = delta_error(h_d);
    LT_REQUIRE(bad == nullptr, "lt_dn_delta_step: %s", bad);
    LT_REQUIRE(vkq && dt && beta && ring && S && o && len && ticket, "lt_dn_delta_step: null pointer");
    LT_REQUIRE(h_d->taps > 0 && h_d->conv && h_d->conv_b && h_d->dt_bias && h_d->A, "lt_dn_delta_step: taps=%d or null constants", h_d->taps);
    LT_REQUIRE(aligned16(S), "lt_dn_delta_step: the state must be 16-byte aligned");
    DeltaStepP P = {vkq, dt, beta, ring, S, o, len, ticket, h_d->H * h_d->dvp + 2 * h_d->G * h_d->dp, *h_d};
    if (f32) return launch_delta_step<float>(P, (cudaStream_t)stream);
    return launch_delta_step<bf16>(P, (cudaStream_t)stream);
}
