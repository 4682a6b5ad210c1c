// Routing of token rows to experts: which `top` of n experts a row of scores chooses and with what weights, and the order of
// the chosen places by expert that the grouped products walk.
//
//   s = softmax(l) or sigmoid(l),  c = s + bias,  the top of c inside the best groups,  w = s / sum of the chosen s * scale
//
// k_route: a warp per token.  Scores and choice values are doubles: whether an expert is among the top depends on the last bits of
// values that lie close together, and 64 bits make the choice the same whatever order a sum is taken in.  The choice is made on the
// bits of c, which order like the numbers, by integer reductions over the warp; the scores of the chosen are made once more at the
// end, a lane each, instead of being carried along.  A group's experts are shared by consecutive lanes, so that a lane is kept or
// dropped as a whole.  (2048 tokens, top 8 of 256 in 4 of 8 groups: instructions bound it, half of them in the picks.)
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

__device__ __forceinline__ float clean_logit(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f); }
__device__ __forceinline__ double key_value(unsigned long long k) {
    return __longlong_as_double((long long)((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
}

// VPL: experts of a lane at most; `each` lanes share a group, `own` experts a lane
template <int VPL>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) k_route(const __grid_constant__ RouteP P, int each, int own) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * ROUTE_WARPS + warp;
    if (t >= P.T) return;
    const lt_dn_router& R = P.R;
    const float* l = P.logits + (long)t * P.ld;
    const int group = lane / each, size = R.n / R.groups, in = (lane - group * each) * own;      // first expert, inside the group
    const int first = group * size + in, mine = group < R.groups ? max(0, min(own, size - in)) : 0;
    unsigned long long key[VPL];
    float x[VPL], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        x[i] = i < mine ? clean_logit(l[first + i]) : -INFINITY;
        m = fmaxf(m, x[i]);
    }
    double sum = 0.0;
    const bool softmax = R.score == LT_DN_SCORE_SOFTMAX;
    if (softmax) m = warp_max(m);
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        double e = 0.0;
        if (x[i] != -INFINITY) e = exp(softmax ? (double)x[i] - (double)m : -(double)x[i]);
        sum += e;
        key[i] = (unsigned long long)__double_as_longlong(e);
    }
    if (softmax) sum = warp_add(sum);
    const double inv = sum > 0.0 ? 1.0 / sum : 0.0;
#pragma unroll
    for (int i = 0; i < VPL; i++) {
        const double e = __longlong_as_double((long long)key[i]);
        double c = softmax ? e * inv : 1.0 / (1.0 + e);
        if (R.bias != nullptr && i < mine) c += (double)R.bias[first + i];
        key[i] = i < mine ? order_key(x[i] == -INFINITY ? -INFINITY : c) : 0ull;
    }
    if (R.groups > 1) {
        unsigned long long a = 0ull, b = 0ull;           // the two best of the lane, then of the group
#pragma unroll
        for (int i = 0; i < VPL; i++) {
            const unsigned long long low = min(a, key[i]);
            a = max(a, key[i]);
            b = max(b, low);
        }
        for (int s = 1; s < each; s <<= 1) {
            const unsigned long long oa = __shfl_xor_sync(0xffffffffu, a, s), ob = __shfl_xor_sync(0xffffffffu, b, s);
            b = max(min(a, oa), max(b, ob));
            a = max(a, oa);
        }
        unsigned long long gkey = 0ull;
        if (lane - group * each == 0 && group < R.groups) gkey = order_key(size > 1 ? key_value(a) + key_value(b) : key_value(a));
        unsigned kept = 0;
        for (int i = 0; i < R.top_groups; i++) {
            const int g = warp_best(gkey, group);
            kept |= 1u << g;
            if (group == g) gkey = 0ull;
        }
        if (!((kept >> group) & 1)) {
#pragma unroll
            for (int i = 0; i < VPL; i++)
                if (i < mine) key[i] = KEY_DROPPED;
        }
    }
    int chosen = 0;                      // of place `lane`
    for (int j = 0; j < R.top; j++) {
        unsigned long long best = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < VPL; i++)
            if (key[i] > best) {
                best = key[i];
                at = i;
            }
        const int e = warp_best(best, first + at);
        if (lane == j) chosen = e;
        const bool here = e >= first && e < first + mine;
#pragma unroll
        for (int i = 0; i < VPL; i++)
            if (here && i == at) key[i] = 0ull;
    }
    double s = 0.0;
    if (lane < R.top) {
        const float v = clean_logit(l[chosen]);
        if (v != -INFINITY) {
            const double e = exp(softmax ? (double)v - (double)m : -(double)v);
            s = softmax ? e * inv : 1.0 / (1.0 + e);
        }
    }
    if (R.renorm) {
        const double total = warp_add(s);
        s = total > 0.0 ? s / total : 0.0;
    }
    if (lane < R.top) {
        P.ids[(long)t * R.top + lane] = chosen;
        P.w[(long)t * R.top + lane] = (float)(s * (double)R.scale);
    }
}

template <int VPL>
static int launch_route(const RouteP& P, int each, int own, cudaStream_t s) {
    k_route<VPL><<<(P.T + ROUTE_WARPS - 1) / ROUTE_WARPS, 32 * ROUTE_WARPS, 0, s>>>(P, each, own);
    return check_launch("lt_dn_route");
}

// ---------------------------------------------------------------------------- order of the places by expert

// A warp owns a stretch of the places and looks at 32 of them at a time, eight loads ahead: 16000 places of 64 experts take
// 5 us.  (A stretch per thread made every load of a warp touch 32 lines: 19 us.)
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
    int each = 32;
    while (each * R.groups > 32) each /= 2;
    const int size = R.n / R.groups, own = (size + each - 1) / each;
    if (own <= 2) return launch_route<2>(P, each, own, s);
    if (own <= 4) return launch_route<4>(P, each, own, s);
    if (own <= 8) return launch_route<8>(P, each, own, s);
    if (own <= 16) return launch_route<16>(P, each, own, s);
    if (own <= 32) return launch_route<32>(P, each, own, s);
    return launch_route<64>(P, each, own, s);       // more than 16 groups that are no power of two
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
