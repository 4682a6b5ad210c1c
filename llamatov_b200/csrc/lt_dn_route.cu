// Routing of token rows to experts: which `top` of n experts a row of scores chooses and with what weights, and the order of
// the chosen places by expert that the grouped products walk.
//
//   s = softmax(l) or sigmoid(l),  c = s + bias,  the top of c inside the best groups,  w = s / sum of the chosen s * scale
//
// k_route: a warp per token, scores in registers.  Scores and choice values are doubles: whether an expert is among the top
// depends on the last bits of values that lie close together, and 64 bits make the choice the same whatever order a sum is
// taken in.  The choice is made on the bits of c, which order like the numbers, by integer reductions over the warp.
// k_plan: a CTA per expert counts the places of lower experts and lists its own in order.  Every CTA reads all ids, so no CTA
// waits for another and the order does not depend on timing.
#include "lt_dn_common.cuh"

namespace lt {
namespace dn {

struct RouteP {
    const float* logits;
    int* ids;
    float* w;
    int ld, T;
    lt_dn_router R;
};

constexpr int ROUTE_WARPS = 4;
constexpr int MAX_GROUPS = 32;

// bits of a double in an order that unsigned comparison follows; NaN is below every number
__device__ __forceinline__ unsigned long long order_key(double v) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(v);
    if (v != v) return 0x000fffffffffffffull;          // minus infinity's
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
constexpr unsigned long long KEY_DROPPED = 1ull;       // below minus infinity: chosen only when nothing else is left
__device__ __forceinline__ double warp_add(double v) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
    return v;
}
// the lane's (key, index) that is largest over the warp; equal keys: the lowest index
__device__ __forceinline__ int warp_best(unsigned long long key, int index) {
    const unsigned hi = (unsigned)(key >> 32), lo = (unsigned)key;
    const unsigned mh = __reduce_max_sync(0xffffffffu, hi);
    const unsigned ml = __reduce_max_sync(0xffffffffu, hi == mh ? lo : 0u);
    return (int)__reduce_min_sync(0xffffffffu, hi == mh && lo == ml ? (unsigned)index : 0xffffffffu);
}

// VPL: experts of a lane, lane + 32 i
template <int VPL>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) k_route(const __grid_constant__ RouteP P) {
    extern __shared__ __align__(16) unsigned char route_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * ROUTE_WARPS + warp;
    if (t >= P.T) return;
    const lt_dn_router& R = P.R;
    const float* l = P.logits + (long)t * P.ld;
    double s[VPL];
    unsigned long long key[VPL];
    float x[VPL], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int e = lane + 32 * i;
        x[i] = e < R.n ? l[e] : -INFINITY;
        if (x[i] != x[i]) x[i] = -INFINITY;
        x[i] = fminf(x[i], 3.402823466e38f);
        m = fmaxf(m, x[i]);
    }
    if (R.score == LT_DN_SCORE_SOFTMAX) {
        m = warp_max(m);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            s[i] = x[i] == -INFINITY ? 0.0 : exp((double)x[i] - (double)m);
            sum += s[i];
        }
        sum = warp_add(sum);
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
    } else {
#pragma unroll
        for (int i = 0; i < VPL; i++) s[i] = x[i] == -INFINITY ? 0.0 : 1.0 / (1.0 + exp(-(double)x[i]));
    }
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const int e = lane + 32 * i;
        double c = s[i];
        if (R.bias != nullptr && e < R.n) c += (double)R.bias[e];
        key[i] = e < R.n ? order_key(x[i] == -INFINITY ? -INFINITY : c) : 0ull;
    }
    if (R.groups > 1) {
        double* c = (double*)route_smem + warp * (R.n + R.groups);    // a word between the groups: no bank conflicts
        const int size = R.n / R.groups;
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int e = lane + 32 * i;
            if (e < R.n) {
                const unsigned long long k = key[i];
                c[e + e / size] = __longlong_as_double((long long)((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
            }
        }
        __syncwarp();
        unsigned long long gkey = 0ull;
        if (lane < R.groups) {
            double a = -INFINITY, b = -INFINITY;
            for (int i = 0; i < size; i++) {
                const double v = c[lane * (size + 1) + i];
                b = fmax(b, fmin(a, v));
                a = fmax(a, v);
            }
            gkey = order_key(size > 1 ? a + b : a);
        }
        unsigned kept = 0;
        for (int i = 0; i < R.top_groups; i++) {
            const int g = warp_best(gkey, lane);
            kept |= 1u << g;
            if (lane == g) gkey = 0ull;
        }
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const int e = lane + 32 * i;
            if (e < R.n && !((kept >> (e / size)) & 1)) key[i] = KEY_DROPPED;
        }
    }
    double total = 0.0, mine = 0.0;      // lane j keeps the score of choice j (and j + 32 is never needed: top <= 32)
    int chosen = 0;
    for (int j = 0; j < R.top; j++) {
        unsigned long long best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < VPL; i++)
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        const int e = warp_best(best, lane + 32 * at);
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (lane + 32 * i == e) {
                v = s[i];
                key[i] = 0ull;
            }
        v = __shfl_sync(0xffffffffu, v, e & 31);
        total += v;
        if (lane == j) {
            mine = v;
            chosen = e;
        }
    }
    if (lane < R.top) {
        if (R.renorm) mine = total > 0.0 ? mine / total : 0.0;
        P.ids[(long)t * R.top + lane] = chosen;
        P.w[(long)t * R.top + lane] = (float)(mine * (double)R.scale);
    }
}

template <int VPL>
static int launch_route(const RouteP& P, cudaStream_t s) {
    const size_t smem = P.R.groups > 1 ? (size_t)ROUTE_WARPS * (P.R.n + P.R.groups) * 8 : 0;
    k_route<VPL><<<(P.T + ROUTE_WARPS - 1) / ROUTE_WARPS, 32 * ROUTE_WARPS, smem, s>>>(P);
    return check_launch("lt_dn_route");
}

// ---------------------------------------------------------------------------- order of the places by expert

// A warp owns a stretch of the places and looks at 32 of them at a time, eight loads ahead: 16384 places of 64 experts take
// 3 us.  (A stretch per thread made every load of a warp touch 32 lines: 19 us.)
constexpr int PLAN_THREADS = 512, PLAN_AHEAD = 8;

__global__ void __launch_bounds__(PLAN_THREADS) k_plan(const int* __restrict__ ids, int P, int n, int* __restrict__ plan, int* status) {
    constexpr int WARPS = PLAN_THREADS / 32;
    __shared__ int sm[WARPS], sl[WARPS];
    const int e = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int seg = ((P + 31) / 32 + WARPS - 1) / WARPS * 32;
    const int from = (int)min((long)warp * seg, (long)P), to = min(from + seg, P);
    int mine = 0, less = 0;
    bool bad = false;
    for (int i = from; i < to; i += 32 * PLAN_AHEAD) {
        int id[PLAN_AHEAD];
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++) id[u] = i + u * 32 + lane < to ? ids[i + u * 32 + lane] : -1;
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++) {
            mine += id[u] == e;
            less += id[u] >= 0 && id[u] < e;
            bad |= id[u] >= n;
        }
    }
    if (e == 0 && bad) atomicOr(status, (int)LT_STATUS_BAD_TOKEN);
    mine = __reduce_add_sync(0xffffffffu, mine);
    less = __reduce_add_sync(0xffffffffu, less);
    if (lane == 0) {
        sm[warp] = mine;
        sl[warp] = less;
    }
    __syncthreads();
    int base = 0, at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
        base += sl[w];
        if (w < warp) at += sm[w];
        all += sm[w];
    }
    if (tid == 0) {
        plan[e] = base;
        if (e == n - 1) plan[n] = base + all;
    }
    if (mine == 0) return;
    int* out = plan + n + 1 + base + at;
    for (int i = from; i < to; i += 32 * PLAN_AHEAD) {
        int id[PLAN_AHEAD];
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++) id[u] = i + u * 32 + lane < to ? ids[i + u * 32 + lane] : -1;
#pragma unroll
        for (int u = 0; u < PLAN_AHEAD; u++) {
            const unsigned here = __ballot_sync(0xffffffffu, id[u] == e);
            if (id[u] == e) out[__popc(here & ((1u << lane) - 1))] = i + u * 32 + lane;
            out += __popc(here);
        }
    }
}

}  // namespace dn
}  // namespace lt

using namespace lt;
using namespace lt::dn;

extern "C" int lt_dn_route(const float* logits, int ld, int* ids, float* w, int T, const lt_dn_router* h_r, void* stream) {
    LT_REQUIRE(logits && ids && w && h_r, "lt_dn_route: null pointer");
    const lt_dn_router& R = *h_r;
    LT_REQUIRE(T > 0 && R.n > 0 && R.n <= 1024 && ld >= R.n, "lt_dn_route: T=%d n=%d (at most 1024) ld=%d", T, R.n, ld);
    LT_REQUIRE(R.score == LT_DN_SCORE_SOFTMAX || R.score == LT_DN_SCORE_SIGMOID, "lt_dn_route: unknown score %d", R.score);
    LT_REQUIRE(R.groups >= 1 && R.groups <= MAX_GROUPS && R.n % R.groups == 0 && R.top_groups >= 1 && R.top_groups <= R.groups,
               "lt_dn_route: %d of %d groups of %d experts (at most %d groups)", R.top_groups, R.groups, R.n, MAX_GROUPS);
    LT_REQUIRE(R.top >= 1 && R.top <= 32 && R.top <= R.n / R.groups * R.top_groups, "lt_dn_route: top %d of %d experts (at most 32)", R.top,
               R.n / R.groups * R.top_groups);
    RouteP P = {logits, ids, w, ld, T, R};
    cudaStream_t s = (cudaStream_t)stream;
    if (R.n <= 64) return launch_route<2>(P, s);
    if (R.n <= 128) return launch_route<4>(P, s);
    if (R.n <= 256) return launch_route<8>(P, s);
    if (R.n <= 512) return launch_route<16>(P, s);
    return launch_route<32>(P, s);
}

extern "C" long lt_dn_experts_plan_ints(int T, int top, int n) { return (long)T * top + n + 1; }

extern "C" int lt_dn_experts_plan(const int* ids, int T, int top, int n, int* plan, void* stream) {
    LT_REQUIRE(ids && plan, "lt_dn_experts_plan: null pointer");
    LT_REQUIRE(T > 0 && top > 0 && n > 0 && n <= 1024 && (long)T * top < (1L << 30), "lt_dn_experts_plan: T=%d top=%d n=%d", T, top, n);
    int* status = device_status_ptr();
    LT_REQUIRE(status != nullptr, "lt_dn_experts_plan: status word unavailable");
    k_plan<<<n, PLAN_THREADS, 0, (cudaStream_t)stream>>>(ids, T * top, n, plan, status);
    return check_launch("lt_dn_experts_plan");
}
