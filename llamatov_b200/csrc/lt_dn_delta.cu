// Gated delta rule in token order, state in fp32:
//   k^ = k / sqrt(sum k^2 + eps),  q^ = q_scale q / sqrt(sum q^2 + eps)
//   u_t = beta_t (v_t - a_t S k^_t),  S <- a_t S + u_t k^_t^T,  o_t = S q^_t
// The output needs no second pass over the new state: S_new q^ = a (S q^) + u (k^ . q^), so both products are taken of the old
// state together and a token is one dependent chain: products, their sum over the lanes of a column, u, the update.
//
// k_delta_scan walks rows (fp32, short portions): a CTA owns 32 value columns of one head of one sequence, eight lanes share a
// column (dp/8 key channels each, in registers); normed q and k and k^ . q^ are made 16 tokens at a time, a warp per token.
// k_delta_step is one token with its convolution and step size.
#include "lt_dn_delta.cuh"

namespace lt {
namespace dn {

struct DeltaScanP {
    const void *q, *k, *v;
    const float *la, *beta;
    float* o;
    int ld, ldh, ldo;
    lt_dn_delta D;
    lt_dn_seqs Q;
};
constexpr int DT = 16;    // tokens staged at a time

__device__ __forceinline__ float sum8(float v) {       // over the eight lanes of a column
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    v += __shfl_xor_sync(0xffffffffu, v, 2);
    return v + __shfl_xor_sync(0xffffffffu, v, 4);
}

template <int KPT>
__device__ __forceinline__ void load_state(float (&s)[KPT], const float* row, int dp, int g) {
#pragma unroll
    for (int i = 0; i < KPT / 4; i++) {
        const int c = i * 32 + g * 4;
        float4 x = make_float4(0, 0, 0, 0);
        if (c < dp) x = *(const float4*)(row + c);
        s[4 * i] = x.x; s[4 * i + 1] = x.y; s[4 * i + 2] = x.z; s[4 * i + 3] = x.w;
    }
}
template <int KPT>
__device__ __forceinline__ void store_state(const float (&s)[KPT], float* row, int dp, int g) {
#pragma unroll
    for (int i = 0; i < KPT / 4; i++) {
        const int c = i * 32 + g * 4;
        if (c < dp) *(float4*)(row + c) = make_float4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
    }
}

template <typename T, int KPT>
__global__ void __launch_bounds__(256) k_delta_scan(const __grid_constant__ DeltaScanP P) {
    constexpr int DP = 8 * KPT;
    extern __shared__ __align__(16) float dsm[];
    float* sq = dsm;                   // [DT][DP]
    float* sk = sq + DT * DP;
    float* sv = sk + DT * DP;          // [DT][32]
    float* sc = sv + DT * 32;          // [DT][4]: decay, beta, k . q
    const lt_dn_delta& D = P.D;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = tid & 7, cl = tid >> 3;
    const int h = blockIdx.y, b = blockIdx.z, hq = h / (D.H / D.G), col = blockIdx.x * 32 + cl;
    const bool col_ok = col < D.dvp;
    const int T_ = P.Q.rows[b];
    const long first = P.Q.start[b];
    if (T_ == 0) return;
    float s[KPT];
    float* Srow = P.Q.S[b] + ((long)h * D.dvp + (col_ok ? col : 0)) * D.dp;
    load_state<KPT>(s, Srow, D.dp, g);

    for (int t0 = 0; t0 < T_; t0 += DT) {
        const int nt = min(DT, T_ - t0);
        for (int t = warp; t < nt; t += 8) {
            const long r = first + t0 + t;
            const T* q = (const T*)P.q + r * P.ld + (long)hq * D.dp;
            const T* k = (const T*)P.k + r * P.ld + (long)hq * D.dp;
            float fq[DP / 32], fk[DP / 32], qq = 0.0f, kk = 0.0f, kq = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 32; i++) {
                const int c = lane + 32 * i;
                fq[i] = c < D.dp ? to_f(q[c]) : 0.0f;
                fk[i] = c < D.dp ? to_f(k[c]) : 0.0f;
                qq = fmaf(fq[i], fq[i], qq);
                kk = fmaf(fk[i], fk[i], kk);
                kq = fmaf(fk[i], fq[i], kq);
            }
            qq = warp_sum(qq);
            kk = warp_sum(kk);
            kq = warp_sum(kq);
            const float rq = D.q_scale / sqrtf(qq + D.eps), rk = 1.0f / sqrtf(kk + D.eps);
#pragma unroll
            for (int i = 0; i < DP / 32; i++) {
                sq[t * DP + lane + 32 * i] = fq[i] * rq;
                sk[t * DP + lane + 32 * i] = fk[i] * rk;
            }
            const int c = blockIdx.x * 32 + lane;
            sv[t * 32 + lane] = c < D.dvp ? to_f(((const T*)P.v)[r * P.ld + (long)h * D.dvp + c]) : 0.0f;
            if (lane == 0) {
                sc[4 * t] = expf(P.la[r * P.ldh + h]);
                sc[4 * t + 1] = P.beta[r * P.ldh + h];
                sc[4 * t + 2] = kq * rq * rk;
            }
        }
        __syncthreads();
        for (int t = 0; t < nt; t++) {
            const float a = sc[4 * t], be = sc[4 * t + 1], kq = sc[4 * t + 2], v = sv[t * 32 + cl];
            float4 k[KPT / 4];
            float p[4] = {0, 0, 0, 0}, r[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KPT / 4; i++) {
                const int c = t * DP + i * 32 + g * 4;
                k[i] = *(const float4*)(sk + c);
                const float4 q = *(const float4*)(sq + c);
                p[0] = fmaf(k[i].x, s[4 * i], p[0]); p[1] = fmaf(k[i].y, s[4 * i + 1], p[1]);
                p[2] = fmaf(k[i].z, s[4 * i + 2], p[2]); p[3] = fmaf(k[i].w, s[4 * i + 3], p[3]);
                r[0] = fmaf(q.x, s[4 * i], r[0]); r[1] = fmaf(q.y, s[4 * i + 1], r[1]);
                r[2] = fmaf(q.z, s[4 * i + 2], r[2]); r[3] = fmaf(q.w, s[4 * i + 3], r[3]);
            }
            const float Sk = sum8((p[0] + p[1]) + (p[2] + p[3])), Sq = sum8((r[0] + r[1]) + (r[2] + r[3]));
            const float u = be * fmaf(-a, Sk, v);
#pragma unroll
            for (int i = 0; i < KPT / 4; i++) {
                s[4 * i] = fmaf(a, s[4 * i], u * k[i].x);
                s[4 * i + 1] = fmaf(a, s[4 * i + 1], u * k[i].y);
                s[4 * i + 2] = fmaf(a, s[4 * i + 2], u * k[i].z);
                s[4 * i + 3] = fmaf(a, s[4 * i + 3], u * k[i].w);
            }
            if (g == 0 && col_ok) P.o[(first + t0 + t) * P.ldo + (long)h * D.dvp + col] = fmaf(a, Sq, u * kq);
        }
        __syncthreads();
    }
    if (col_ok) store_state<KPT>(s, Srow, D.dp, g);
}

template <typename T, int KPT>
static int launch_delta_scan(const DeltaScanP& P, cudaStream_t s) {
    const size_t smem = ((size_t)DT * 8 * KPT * 2 + (size_t)DT * 36) * 4;
    static PerDeviceOnce once;
    if (once.first()) LT_CUDA(cudaFuncSetAttribute(k_delta_scan<T, KPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    k_delta_scan<T, KPT><<<dim3((P.D.dvp + 31) / 32, P.D.H, P.Q.n), 256, smem, s>>>(P);
    return check_launch("lt_dn_delta");
}
template <typename T>
static int delta_scan_size(const DeltaScanP& P, cudaStream_t s) {
    if (P.D.dp <= 32) return launch_delta_scan<T, 4>(P, s);
    if (P.D.dp <= 64) return launch_delta_scan<T, 8>(P, s);
    if (P.D.dp <= 128) return launch_delta_scan<T, 16>(P, s);
    if (P.D.dp <= 256) return launch_delta_scan<T, 32>(P, s);
    return launch_delta_scan<T, 64>(P, s);
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
    Sk = sum8(Sk);
    Sq = sum8(Sq);
    kk = sum8(kk);
    qq = sum8(qq);
    kq = sum8(kq);
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

extern "C" int lt_dn_delta_rows(const void* q, const void* k, const void* v, int ld, const float* la, const float* beta, int ldh, float* o,
                                int ldo, int f32, const lt_dn_delta* h_d, const lt_dn_seqs* h_q, void* stream) {
    int rows = 0;
    const char* bad = delta_error(h_d);
    if (bad == nullptr) bad = delta_seqs_error(h_q, &rows);
    LT_REQUIRE(bad == nullptr, "lt_dn_delta_rows: %s", bad);
    LT_REQUIRE(q && k && v && la && beta && o, "lt_dn_delta_rows: null pointer");
    LT_REQUIRE(ld >= h_d->G * h_d->dp && ld >= h_d->H * h_d->dvp && ldh >= h_d->H && ldo >= h_d->H * h_d->dvp,
               "lt_dn_delta_rows: ld=%d ldh=%d ldo=%d", ld, ldh, ldo);
    if (rows == 0) return LT_OK;
    DeltaScanP P = {q, k, v, la, beta, o, ld, ldh, ldo, *h_d, *h_q};
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
