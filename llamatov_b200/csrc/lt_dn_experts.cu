// The two products of a feed-forward of experts, over the places (t, j) of T tokens with `top` experts each:
//   H[t][j]  = glu(gate and up rows of expert ids[t][j], x_t)                  (lt_dn_experts_glu)
//   Y[t]    += ls * sum_j w[t][j] (W of expert ids[t][j]) H[t][j]              (lt_dn_experts_sum)
//
// With a plan: lt_dn_experts_group.cu.  Without one (few places) each place reads its expert's rows itself, and the time is that of
// the matrices' bytes.
//   k_few_glu   a warp per gate row and its up row
//   k_few_sum   a CTA per rows of Y; its warps share the experts of the token, and their sums are added in order
#include "lt_dn_experts.cuh"

namespace lt {
namespace dn {

struct FewP {
    const void* W;
    const void* X;
    void* Y;
    const float *w, *ls;
    int* status;
    int ldw, ldx, ldy, M, K;     // M: gate rows (glu) or output rows (sum)
    lt_dn_choice c;
    lt_dn_epilogue epi;
};

// An SM has four CTAs of 64 registers a thread, each lane with two rows x 4 loads of 16 bytes under way.  (8 of 64 experts for one
// token in bf16: gate|up 2 x 1024 x 2048 14.2 us, 4.7 TB/s, down 2048 x 1024 10.0; with two CTAs that also hold their part of x
// ahead 15.1 and 13.3; twice the loads a lane 16.0 and 14.0; rows through rings of bulk copies in shared memory, 192 KB under way,
// 20.1 and 15.9.)
constexpr int FEW_THREADS = 256, FEW_U = 4, FEW_CTAS = 4;

// products of two rows with x: this lane's share
template <typename T>
__device__ __forceinline__ void two_dots(const T* a, const T* b, const T* x, int nvec, int lane, float& s0, float& s1) {
    constexpr int N = Vec<T>::N;
    for (int base = lane; base < nvec; base += 32 * FEW_U) {
        int4 va[FEW_U], vb[FEW_U];
#pragma unroll
        for (int u = 0; u < FEW_U; u++) {
            const int i = base + u * 32;
            if (i < nvec) {
                va[u] = ld_stream_v4((const uint4*)a + i);
                vb[u] = ld_stream_v4((const uint4*)b + i);
            }
        }
#pragma unroll
        for (int u = 0; u < FEW_U; u++) {
            if (base + u * 32 >= nvec) break;
            float fa[N], fb[N], fx[N];
            Vec<T>::unpack(make_uint4(va[u].x, va[u].y, va[u].z, va[u].w), fa);
            Vec<T>::unpack(make_uint4(vb[u].x, vb[u].y, vb[u].z, vb[u].w), fb);
            Vec<T>::unpack(((const uint4*)x)[base + u * 32], fx);
#pragma unroll
            for (int j = 0; j < N; j++) {
                s0 = fmaf(fa[j], fx[j], s0);
                s1 = fmaf(fb[j], fx[j], s1);
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(FEW_THREADS, FEW_CTAS) k_few_glu(const __grid_constant__ FewP P) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nvec = P.K / Vec<T>::N;
    const long tasks = (long)P.c.T * P.c.top * P.M, nw = (long)gridDim.x * (FEW_THREADS / 32);
    for (long i = (long)blockIdx.x * (FEW_THREADS / 32) + warp; i < tasks; i += nw) {
        const long p = i / P.M;
        const int f = (int)(i - p * P.M), e = P.c.ids[p];
        if (e < 0 || e >= P.c.n) {
            if (e >= P.c.n && lane == 0) atomicOr(P.status, (int)LT_STATUS_BAD_TOKEN);
            continue;
        }
        const T* a = (const T*)P.W + ((long)e * 2 * P.M + f) * P.ldw;
        float g = 0.0f, u = 0.0f;
        two_dots(a, a + (long)P.M * P.ldw, (const T*)P.X + p / P.c.top * P.ldx, nvec, lane, g, u);
        float v[2] = {g, u};
        warp_sums(v);
        if (lane == 0) glu_store<T>(P.epi, P.Y, p * P.ldy + f, v[0], v[1]);
    }
}

// wj warps share a pair of rows: warp s of them has the experts s, s + wj, ...
template <typename T>
__global__ void __launch_bounds__(FEW_THREADS, FEW_CTAS) k_few_sum(const __grid_constant__ FewP P, int wj) {
    __shared__ float part[2][FEW_THREADS / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nvec = P.K / Vec<T>::N;
    const int sub = warp & (wj - 1), pairs = FEW_THREADS / 32 / wj, t = blockIdx.y;
    const int npair = (P.M + 1) / 2;
    for (int b = blockIdx.x * pairs; b < npair; b += gridDim.x * pairs) {
        const int pr = b + warp / wj, r0 = 2 * pr, r1 = r0 + 1 < P.M ? r0 + 1 : r0;
        float s0 = 0.0f, s1 = 0.0f;
        if (pr < npair) {
            for (int j = sub; j < P.c.top; j += wj) {
                const long p = (long)t * P.c.top + j;
                const int e = P.c.ids[p];
                if (e < 0 || e >= P.c.n) {
                    if (e >= P.c.n && lane == 0) atomicOr(P.status, (int)LT_STATUS_BAD_TOKEN);
                    continue;
                }
                const T* W = (const T*)P.W + (long)e * P.M * P.ldw;
                float a = 0.0f, c = 0.0f;
                two_dots(W + (long)r0 * P.ldw, W + (long)r1 * P.ldw, (const T*)P.X + p * P.ldx, nvec, lane, a, c);
                s0 = fmaf(P.w[p], a, s0);
                s1 = fmaf(P.w[p], c, s1);
            }
            float v[2] = {s0, s1};
            warp_sums(v);
            s0 = v[0];
            s1 = v[1];
        }
        if (lane == 0) {
            part[0][warp] = s0;
            part[1][warp] = s1;
        }
        __syncthreads();
        if (threadIdx.x < 2 * pairs) {
            const int i = threadIdx.x >> 1, row = 2 * (b + i) + (threadIdx.x & 1);
            if (row < P.M) {
                float v = 0.0f;
                for (int s = 0; s < wj; s++) v += part[threadIdx.x & 1][i * wj + s];
                float* y = (float*)P.Y + (long)t * P.ldy + row;
                *y = fmaf(P.ls != nullptr ? P.ls[row] : 1.0f, v, *y);
            }
        }
        __syncthreads();
    }
}

// of the matrices together: a tile's row is an int coordinate of their tensor map
constexpr long MAX_ROWS = 0x7fffffffL;

static const char* choice_error(const lt_dn_choice* c) {
    if (c == nullptr || c->ids == nullptr) return "null choice";
    if (c->T <= 0 || c->top <= 0 || c->top > 32 || c->n <= 0 || c->n > 1024) return "tokens, top (at most 32) or experts (at most 1024)";
    if ((long)c->T * c->top >= (1L << 30)) return "too many places";
    return nullptr;
}

}  // namespace dn
}  // namespace lt

using namespace lt;
using namespace lt::dn;

extern "C" int lt_dn_experts_glu(const void* W, int ldw, const void* X, int ldx, void* H, int ldh, int f32, int F, int K,
                                 const lt_dn_choice* h_c, const lt_dn_epilogue* h_epi, void* ws, void* stream) {
    LT_REQUIRE(W && X && H, "lt_dn_experts_glu: null pointer");
    const char* bad = choice_error(h_c);
    if (bad == nullptr) bad = epi_error(h_epi);
    LT_REQUIRE(bad == nullptr, "lt_dn_experts_glu: %s", bad);
    LT_REQUIRE(h_epi->kind == LT_DN_GLU && !h_epi->out_f32, "lt_dn_experts_glu: the epilogue is LT_DN_GLU in the element type");
    LT_REQUIRE(F > 0 && K > 0 && K % 8 == 0 && ldw >= K && ldw % 8 == 0 && ldx >= K && ldx % 8 == 0 && ldh >= F,
               "lt_dn_experts_glu: F=%d K=%d ldw=%d ldx=%d ldh=%d (multiples of 8)", F, K, ldw, ldx, ldh);
    LT_REQUIRE(aligned16(W) && aligned16(X), "lt_dn_experts_glu: W and X must be 16-byte aligned");
    if (h_c->plan != nullptr) {
        LT_REQUIRE(f32 || (ws != nullptr && aligned16(ws)), "lt_dn_experts_glu: a plan needs the workspace, 16-byte aligned");
        LT_REQUIRE(f32 || 2L * F * h_c->n <= MAX_ROWS, "lt_dn_experts_glu: %ld rows of all matrices", 2L * F * h_c->n);
        GroupP G = {W, X, H, device_status_ptr(), F, K, ldw, ldx, ldh, h_c->top, 0, *h_c, *h_epi};
        LT_REQUIRE(G.status != nullptr, "lt_dn_experts_glu: status word unavailable");
        return launch_group(G, true, f32, ws, (cudaStream_t)stream);
    }
    FewP P = {W, X, H, nullptr, nullptr, device_status_ptr(), ldw, ldx, ldh, F, K, *h_c, *h_epi};
    LT_REQUIRE(P.status != nullptr, "lt_dn_experts_glu: status word unavailable");
    const long need = ((long)h_c->T * h_c->top * F + FEW_THREADS / 32 - 1) / (FEW_THREADS / 32), most = (long)FEW_CTAS * sm_count();
    const int grid = (int)(need < most ? need : most);
    if (f32) k_few_glu<float><<<grid, FEW_THREADS, 0, (cudaStream_t)stream>>>(P);
    else k_few_glu<bf16><<<grid, FEW_THREADS, 0, (cudaStream_t)stream>>>(P);
    return check_launch("lt_dn_experts_glu");
}

// the sums of the places, on a boundary of 16 bytes, then (bf16) their rows in the order of the plan
static long places_floats(int T, int top, int M) { return ((long)T * top * M + 3) / 4 * 4; }
extern "C" long lt_dn_experts_glu_ws(int T, int top, int K, int f32) { return f32 ? 0 : (long)T * top * K / 2; }
extern "C" long lt_dn_experts_sum_ws(int T, int top, int M, int K, int f32) {
    return places_floats(T, top, M) + (f32 ? 0 : (long)T * top * K / 2);
}

extern "C" int lt_dn_experts_sum(const void* W, int ldw, const void* H, int ldh, float* Y, int ldy, int f32, int M, int K,
                                 const lt_dn_choice* h_c, const float* w, const float* ls, float* ws, void* stream) {
    LT_REQUIRE(W && H && Y && w, "lt_dn_experts_sum: null pointer");
    const char* bad = choice_error(h_c);
    LT_REQUIRE(bad == nullptr, "lt_dn_experts_sum: %s", bad);
    LT_REQUIRE(M > 0 && K > 0 && K % 8 == 0 && ldw >= K && ldw % 8 == 0 && ldh >= K && ldh % 8 == 0 && ldy >= M,
               "lt_dn_experts_sum: M=%d K=%d ldw=%d ldh=%d ldy=%d (multiples of 8)", M, K, ldw, ldh, ldy);
    LT_REQUIRE(aligned16(W) && aligned16(H), "lt_dn_experts_sum: W and H must be 16-byte aligned");
    if (h_c->plan != nullptr) {
        LT_REQUIRE(ws != nullptr && aligned16(ws), "lt_dn_experts_sum: a plan needs the workspace, 16-byte aligned");
        LT_REQUIRE(f32 || (long)M * h_c->n <= MAX_ROWS, "lt_dn_experts_sum: %ld rows of all matrices", (long)M * h_c->n);
        GroupP G = {W, H, ws, device_status_ptr(), M, K, ldw, ldh, M, 1, 0, *h_c, {}};
        LT_REQUIRE(G.status != nullptr, "lt_dn_experts_sum: status word unavailable");
        const int rc = launch_group(G, false, f32, ws + places_floats(h_c->T, h_c->top, M), (cudaStream_t)stream);
        return rc != LT_OK ? rc : launch_combine(ws, w, ls, Y, ldy, M, *h_c, (cudaStream_t)stream);
    }
    LT_REQUIRE(h_c->T <= 65535, "lt_dn_experts_sum: %d tokens without an order of the places (at most 65535)", h_c->T);
    FewP P = {W, H, Y, w, ls, device_status_ptr(), ldw, ldh, ldy, M, K, *h_c, {}};
    LT_REQUIRE(P.status != nullptr, "lt_dn_experts_sum: status word unavailable");
    // As many warps on a token's experts as leave no CTA more than its first pairs of rows.  (One token, 8 of 64 experts, 2048 x 1024, by 8 /
    // 4 / 2 / 1 warps: 10.8 / 10.0 / 11.1 / 15.2 us, the rule takes 4; 4096 x 512: 14.1 / 11.5 / 10.0 / 12.5, 2; 1024 x 512: 6.6 / 6.9 / 7.9 /
    // 11.1, 8; four tokens: 13.7 / 11.4 / 9.9 / 11.8, 2.)
    const int npair = (M + 1) / 2, most = (FEW_CTAS * sm_count() + h_c->T - 1) / h_c->T;
    int wj = 1;
    while (wj < h_c->top && wj < FEW_THREADS / 32 && (long)npair * 2 * wj <= (long)most * (FEW_THREADS / 32)) wj *= 2;
    const int pairs = FEW_THREADS / 32 / wj, need = (npair + pairs - 1) / pairs;
    const dim3 grid(need < most ? need : most, h_c->T);
    if (f32) k_few_sum<float><<<grid, FEW_THREADS, 0, (cudaStream_t)stream>>>(P, wj);
    else k_few_sum<bf16><<<grid, FEW_THREADS, 0, (cudaStream_t)stream>>>(P, wj);
    return check_launch("lt_dn_experts_sum");
}
