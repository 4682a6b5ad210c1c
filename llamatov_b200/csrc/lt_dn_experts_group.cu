// The experts' products for many places: every expert's matrix is read once for all of its places, which the plan lists by
// expert (lt_dn_route.cu).
//
// bf16 (k_group_tc): tcgen05.mma kind::f16, fp32 accumulators in tensor memory.  A tile is 128 gate rows with their 128 up rows (or
// 256 output rows) of one expert, two MMAs of M = 128, by N places of it.  An expert's places are shared out evenly over as few tiles
// as hold them, and N is the share rounded up to 16: rows of no place cost at most 15 columns of a tile, whatever the shares are.
// The rows of X are first put in the order of the plan (k_gather), so that tiled TMA fetches them.  (Fetched from where they are by
// gathering TMA, four rows an instruction: 83 clocks each, 425 us for gate|up 2 x 1024 x 2048 of 8 of 64 experts, 2000 tokens; by
// asynchronous copies of 16 bytes: 203; in order 162, 13 of it for putting them there.)
//   warp 16 : producer, TMA
//   warp 17 : MMAs (a warp's loop with one thread picked at the instructions: 2 % less than that thread's own loop)
//   warps 0-15 : epilogue, a thread per weight row and a quarter of the places
// What bounds it is the matrices' bytes with what shares the way: of 141 us (gate|up, 537 MB in 620 MB of reads) the copies of W alone take
// 109, 5.6 TB/s; the sums' fp32 outputs are 23 us of 91.  (Two SMs on a tile, cta_group::2 with M = 256, halve X's bytes: 137 and 92 us for as
// much code again.  An L2 prefetch four stages ahead: 4 % more; one accumulator of the sums kept in registers over its release: nothing.)
// All of K adds up in one accumulator, and the tensor cores cut sums off toward zero instead of rounding them: over K = 2048 a product is
// 2e-6 of its size from 64 bits (fp32 matrix products of the plain form 4e-7), 1.8e-6 of it one-sided.  Of gated outputs 0.2 % round to the
// next bf16 for it; their distance from 64 bits, 1.7e-3, is that of the rounding with or without.
// fp32 (k_group_f32): register-blocked tiles on the CUDA cores.
#include "lt_dn_experts.cuh"
#include "lt_tc.cuh"

namespace lt {
namespace dn {

using namespace tc;

constexpr int GK = 64;           // k elements of a stage (128 bytes)
constexpr int XBOX = 64;         // places of a TMA box
constexpr int MAX_EXPERTS = 1024;

template <int NT>
struct GroupCfg {
    static constexpr int W_STAGE = 2 * 128 * 128, X_STAGE = NT * 128, STAGE = W_STAGE + X_STAGE;
    static constexpr int NSTAGE = (206 * 1024) / STAGE > 8 ? 8 : (206 * 1024) / STAGE;
    static constexpr int BUFS = NT <= 128 ? 2 : 1;          // sets of accumulators
    static constexpr int TMEM = BUFS * 2 * NT;
    static constexpr int EW = 16, THREADS = (EW + 2) * 32;
    static constexpr int SMEM = 1024 + NSTAGE * STAGE + 512 + (MAX_EXPERTS + 1) * 4 + MAX_EXPERTS * 4;
    static_assert(TMEM <= 512 && (TMEM & (TMEM - 1)) == 0, "tensor memory columns");
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct GroupBars {
    unsigned long long full[8], empty[8], tfull[2], tempty[2];
    unsigned tmem_base;
    int abort_flag;
    int sums[18];
};

// D[tmem] (+)= A[smem] * B[smem], bf16 x bf16 -> fp32
__device__ __forceinline__ void group_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((int)acc)
        : "memory");
}
// gelu(z) u = z u / (1 + 2^(-z (a + b z^2))) with the constants of the tanh form times log2 e
__device__ __forceinline__ float gelu_up(float z, float u) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * fmaf(z * z, -0.10294324f, -2.3022082f)));
    return __fdividef(z * u, 1.0f + e);
}

// Experts in order of their tiles' columns, the widest first: cum[i] tiles lie before the i-th's, which is expert order[i].  CTAs take
// tiles in turn, there and back, so that the wide and the last narrow ones are shared out evenly, as well as by handing them out one by
// one.  (Gate|up of 2000 tokens 143 us, with experts as they are numbered 149.)  Every role walks them with a cursor of its own.
struct Cursor {
    int i, e;
    int from, count, n, rt;      // places of the tile in the plan's list, columns, row tile
    __device__ __forceinline__ void seek(const GroupP& P, const int* cum, const int* order, int tile) {
        const int g = tile / P.row_tiles;
        rt = tile - g * P.row_tiles;
        while (cum[i + 1] <= g) i++;
        e = order[i];
        const int at = P.c.plan[e], c = P.c.plan[e + 1] - at, tiles = cum[i + 1] - cum[i];
        n = ((c + tiles - 1) / tiles + 15) & ~15;
        from = at + (g - cum[i]) * n;
        count = min(n, at + c - from);       // at least 1: the tiles before hold (tiles - 1) n <= (tiles - 1) NT < c places
    }
};
__device__ __forceinline__ int tile_of(int round) {
    return round * gridDim.x + ((round & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}
// makes cum and order; all threads, 16 warps and more
template <int NT>
__device__ __forceinline__ void sort_tiles(const lt_dn_choice& c, int* cum, int* order, int* sums) {
    static_assert(NT / 16 <= 16, "a warp per number of columns");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int* columns = cum;                    // in units of 16, until the order is known
    for (int e = tid; e < c.n; e += blockDim.x) {
        const int all = c.plan[e + 1] - c.plan[e], tiles = (all + NT - 1) / NT;
        columns[e] = tiles > 0 ? ((all + tiles - 1) / tiles + 15) / 16 : 0;
    }
    __syncthreads();
    const int mine = NT / 16 - warp;       // this warp's number of columns
    int at = 0;
    if (mine > 0)
        for (int e0 = 0; e0 < c.n; e0 += 32) at += __popc(__ballot_sync(0xffffffffu, e0 + lane < c.n && columns[e0 + lane] == mine));
    if (lane == 0) sums[warp] = at;
    __syncthreads();
    at = 0;
    for (int w = 0; w < warp; w++) at += sums[w];
    int used = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) used += sums[w];
    if (mine > 0)
        for (int e0 = 0; e0 < c.n; e0 += 32) {
            const bool ok = e0 + lane < c.n && columns[e0 + lane] == mine;
            const unsigned here = __ballot_sync(0xffffffffu, ok);
            if (ok) order[at + __popc(here & ((1u << lane) - 1))] = e0 + lane;
            at += __popc(here);
        }
    __syncthreads();
    int t[4], sum = 0;                     // sums of tiles: four experts a thread
#pragma unroll
    for (int k = 0; k < 4; k++) {
        t[k] = 0;
        if (tid * 4 + k < used) {
            const int e = order[tid * 4 + k];
            t[k] = (c.plan[e + 1] - c.plan[e] + NT - 1) / NT;
        }
        sum += t[k];
    }
    int before = sum;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, before, s);
        if (lane >= s) before += o;
    }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    before -= sum;
    for (int w = 0; w < warp; w++) before += sums[w];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (tid * 4 + k <= c.n) cum[tid * 4 + k] = before;
        before += t[k];
    }
}

template <int NT, bool GLU>
__global__ void __launch_bounds__(GroupCfg<NT>::THREADS, 1)
k_group_tc(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const __grid_constant__ GroupP P) {
    using C = GroupCfg<NT>;
    constexpr int NS = C::NSTAGE;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    GroupBars* B = (GroupBars*)(base + NS * C::STAGE);
    int* cum = (int*)(base + NS * C::STAGE + 512);
    int* order = cum + MAX_EXPERTS + 1;
    static_assert(sizeof(GroupBars) <= 512, "barriers");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nk = (P.K + GK - 1) / GK;
    volatile int* abort_flag = &B->abort_flag;
    const int* places = P.c.plan + P.c.n + 1;

    if (tid == 0) {
        for (int s = 0; s < NS; s++) {
            mbar_init(&B->full[s], 1);
            mbar_init(&B->empty[s], 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(&B->tfull[s], 1);
            mbar_init(&B->tempty[s], C::EW);
        }
        B->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == C::EW + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&B->tmem_base)),
                     "r"((unsigned)C::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    sort_tiles<NT>(P.c, cum, order, B->sums);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = B->tmem_base;
    const int tiles = cum[P.c.n] * P.row_tiles;
    Cursor cur;
    cur.i = 0;

    if (warp == C::EW) {
        unsigned it = 0;
        bool go = true;
        const bool one = elect_one();
        for (int round = 0, tile; go && (tile = tile_of(round)) < tiles; round++) {
            cur.seek(P, cum, order, tile);
            const int row = GLU ? cur.e * 2 * P.M + cur.rt * 128 : cur.e * P.M + cur.rt * 256;
            const int row2 = GLU ? row + P.M : row + 128;
            for (int kb = 0; kb < nk; kb++, it++) {
                const int s = it % NS;
                const unsigned st = smem_u32(base) + s * C::STAGE, full = smem_u32(&B->full[s]);
                if (!acquire(smem_u32(&B->empty[s]), ((it / NS) & 1) ^ 1, abort_flag, P.status)) {
                    go = false;
                    break;
                }
                if (one) {
                    bar_expect_tx(full, C::W_STAGE + ((cur.n + XBOX - 1) & ~(XBOX - 1)) * 128);
                    tma_load_2d(st, &tmW, kb * GK, row, full);
                    tma_load_2d(st + 128 * 128, &tmW, kb * GK, row2, full);
                    for (int x = 0; x < cur.n; x += XBOX) tma_load_2d(st + C::W_STAGE + x * 128, &tmX, kb * GK, cur.from + x, full);
                }
                __syncwarp();
            }
        }
    } else if (warp == C::EW + 1) {
        {
            const bool one = elect_one();
            const unsigned long long w0 = smem_desc<4>(smem_u32(base));
            const unsigned long long x0 = smem_desc<4>(smem_u32(base) + C::W_STAGE);
            unsigned it = 0, n = 0;
            for (int round = 0, tile; (tile = tile_of(round)) < tiles; round++) {
                cur.seek(P, cum, order, tile);
                // D fp32, A and B bf16, both K-major, M = 128
                const unsigned idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(cur.n >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
                const unsigned slot = n % C::BUFS;
                bar_wait(false, smem_u32(&B->tempty[slot]), ((n / C::BUFS) & 1) ^ 1, abort_flag, P.status);
                tc_fence_after();
                const unsigned d = tmem + slot * 2 * NT;
                for (int kb = 0; kb < nk; kb++, it++) {
                    const unsigned s = it % NS;
                    bar_wait(false, smem_u32(&B->full[s]), (it / NS) & 1, abort_flag, P.status);
                    tc_fence_after();
                    const unsigned long long wd = w0 + (unsigned long long)(s * (C::STAGE >> 4));
                    const unsigned long long xd = x0 + (unsigned long long)(s * (C::STAGE >> 4));
#pragma unroll
                    for (int j = 0; j < GK / 16; j++)
#pragma unroll
                        for (int a = 0; a < 2; a++)
                            if (one) group_mma(d + a * NT, wd + a * (128 * 128 >> 4) + 2 * j, xd + 2 * j, idesc, kb > 0 || j > 0);
                    if (one) mma_commit(&B->empty[s]);
                }
                if (one) mma_commit(&B->tfull[slot]);
                n++;
            }
        }
    } else {
        const int q = warp & 3, cg = warp >> 2;
        unsigned n = 0;
        for (int round = 0, tile; (tile = tile_of(round)) < tiles; round++) {
            cur.seek(P, cum, order, tile);
            const int row = cur.rt * (GLU ? 128 : 256) + q * 32 + lane;
            const unsigned slot = n % C::BUFS;
            int mine[NT / 64];                // places of this warp's columns, fetched under the products
#pragma unroll
            for (int i = 0; i < NT / 64; i++) mine[i] = places[cur.from + min(64 * i + cg * 16 + (lane & 15), cur.count - 1)];
            bar_wait(false, smem_u32(&B->tfull[slot]), (n / C::BUFS) & 1, abort_flag, P.status);
            tc_fence_after();
            const unsigned ta = tmem + ((unsigned)(q * 32) << 16) + slot * 2 * NT;
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&B->tempty[slot]);
            };
            unsigned out[GLU ? NT / 64 : 1][8];      // gated outputs, so that the accumulators are free before the stores
#pragma unroll
            for (int i = 0; i < NT / 64; i++) {
                const int c0 = 64 * i + cg * 16, left = cur.count - c0;
                if (left <= 0) break;
                int v[2][16];
#pragma unroll
                for (int a = 0; a < 2; a++) tmem_ld<16>(ta + a * NT + c0, v[a]);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int a = 0; a < 2; a++)
#pragma unroll
                    for (int c = 0; c < 16; c += 4) reg_fence4(&v[a][c]);
                if (GLU) {
                    float f[16];
                    if (P.epi.glu_act == LT_DN_GLU_GELU) {
#pragma unroll
                        for (int c = 0; c < 16; c++) f[c] = gelu_up(__int_as_float(v[0][c]), __int_as_float(v[1][c]));
                    } else {
                        glu_bf16(P.epi, v[0], v[1], f);
                    }
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * c], f[2 * c + 1]);
                        out[GLU ? i : 0][c] = *(const unsigned*)&h;
                    }
                } else {
                    float* y = (float*)P.Y + row;
#pragma unroll
                    for (int c = 0; c < 16; c++) {
                        const long p = (long)__shfl_sync(0xffffffffu, mine[i], c) * P.ldy;
                        if (c < left) {
                            if (row < P.M) y[p] = __int_as_float(v[0][c]);
                            if (row + 128 < P.M) y[p + 128] = __int_as_float(v[1][c]);
                        }
                    }
                }
            }
            release();
            if (GLU) {
#pragma unroll
                for (int i = 0; i < NT / 64; i++) {
                    const int left = cur.count - 64 * i - cg * 16;
                    if (left <= 0) break;
                    unsigned short* y = (unsigned short*)P.Y + row;
#pragma unroll
                    for (int c = 0; c < 16; c++) {
                        const int p = __shfl_sync(0xffffffffu, mine[i], c);
                        if (row < P.M && c < left) y[(long)p * P.ldy] = (unsigned short)(out[GLU ? i : 0][c >> 1] >> (16 * (c & 1)));
                    }
                }
            }
            n++;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag && tid == 0) {     // a wait ran out: let copies in flight land before the CTA leaves
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {
        }
    }
    __syncthreads();
    if (warp == C::EW + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((unsigned)C::TMEM) : "memory");
    }
}

static int group_map(CUtensorMap* m, const void* ptr, long rows, int K, int ld, int box_rows) {
    encode_fn_t fn = encode_fn();
    LT_REQUIRE(fn != nullptr, "experts' products: cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)GK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    // 256 bytes into L2 at a time: a row's next 128 are the next stage's (gate|up of 2000 tokens 159 -> 153 us)
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("experts' products: cuTensorMapEncodeTiled failed (%d) for rows=%ld K=%d ld=%d", (int)r, rows, K, ld);
        return LT_ERR_CUDA;
    }
    return LT_OK;
}

// rows of X in the order of the plan: a warp per place, 16 bytes a lane
__global__ void __launch_bounds__(256) k_gather(const __grid_constant__ GroupP P, uint4* out) {
    const int s = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, units = P.K / 8;
    if (s >= P.c.plan[P.c.n]) return;
    const int place = P.c.plan[P.c.n + 1 + s];
    const uint4* in = (const uint4*)((const bf16*)P.X + (long)(place / P.per) * P.ldx);
    uint4* o = out + (long)s * units;
    for (int x = lane; x < units; x += 128) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (x + 32 * u < units) v[u] = in[x + 32 * u];
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (x + 32 * u < units) o[x + 32 * u] = v[u];
    }
}

template <int NT, bool GLU>
static int launch_group_tc(GroupP P, void* rows, cudaStream_t s) {
    using C = GroupCfg<NT>;
    const long places = (long)P.c.T * P.c.top;
    CUtensorMap tmW, tmX;
    int rc = group_map(&tmW, P.W, (long)P.c.n * P.M * (GLU ? 2 : 1), P.K, P.ldw, 128);
    if (rc != LT_OK) return rc;
    rc = group_map(&tmX, rows, places, P.K, P.K, XBOX);
    if (rc != LT_OK) return rc;
    static PerDeviceOnce once;
    LT_ONCE(once, LT_CUDA(cudaFuncSetAttribute(k_group_tc<NT, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)));
    k_gather<<<(unsigned)((places + 7) / 8), 256, 0, s>>>(P, (uint4*)rows);
    rc = check_launch("experts' products (rows in order)");
    if (rc != LT_OK) return rc;
    P.row_tiles = (P.M + (GLU ? 127 : 255)) / (GLU ? 128 : 256);
    k_group_tc<NT, GLU><<<sm_count(), C::THREADS, C::SMEM, s>>>(tmW, tmX, P);
    return check_launch("experts' products");
}
// By the mean share, though shares differ: a larger expert has more than one tile.  The fewer columns, the deeper the ring (5, 4 and 3 stages)
// and, up to 128, two sets of accumulators; the more, the fewer times a matrix is read from L2.  (us of the product alone with 64 / 128 /
// 256 columns at so many places an expert.  64 experts of 2 x 1024 x 2048: 16 85.6 / 87.5 / 89.3, 24 85.7 / 88.8 / 91.1, 32 86.9 / 89.4 / 92.7,
// 48 91.8 / 90.4 / 93.8, 64 98.1 / 92.2 / 95.8, 80 102.9 / 96.5 / 96.3, 128 122 / 109 / 103, 250 197 / 149 / 139; of 2048 x 1024: 24 47.2 / 48.3 /
// 49.4, 32 48.6 / 50.8 / 52.3, 48 51.1 / 50.4 / 53.3, 64 56.4 / 53.0 / 55.9, 80 61.3 / 59.3 / 57.2, 250 113 / 94.0 / 90.8; 128 experts of 1024 x 512:
// 24 27.1 / 27.3 / 29.1, 32 29.5 / 28.6 / 30.2, 64 35.7 / 33.1 / 34.0, 96 41.3 / 37.1 / 37.2, 250 73.4 / 61.5 / 62.2.)
template <bool GLU>
static int pick_group_tc(const GroupP& P, void* rows, cudaStream_t s) {
    const long each = (long)P.c.T * P.c.top / P.c.n;        // places of an expert
    if (each <= 24) return launch_group_tc<64, GLU>(P, rows, s);
    if (each <= 64) return launch_group_tc<128, GLU>(P, rows, s);
    return launch_group_tc<256, GLU>(P, rows, s);
}

// ---------------------------------------------------------------------------- fp32

// By one warp: the expert whose tiles of BN places hold number g, 32 experts at a time.  found: expert, places (none past the last
// tile); place: the tile's places, the last repeated.
template <int BN>
__device__ __forceinline__ void find_tile(const lt_dn_choice& c, int g, int lane, int* found, int* place) {
    int before = 0, from = 0, count = 0;
    for (int e0 = 0; e0 < c.n && before <= g; e0 += 32) {
        const int e = e0 + lane, at = e < c.n ? c.plan[e] : 0, all = e < c.n ? c.plan[e + 1] - at : 0;
        const int tiles = (all + BN - 1) / BN;
        int up = tiles;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, up, s);
            if (lane >= s) up += o;
        }
        const int first = before + up - tiles;
        const unsigned here = __ballot_sync(0xffffffffu, g >= first && g < first + tiles);
        if (here != 0) {
            const int l = __ffs(here) - 1, skip = (g - __shfl_sync(0xffffffffu, first, l)) * BN;
            from = __shfl_sync(0xffffffffu, at, l) + skip;
            count = min(BN, __shfl_sync(0xffffffffu, all, l) - skip);
            if (lane == 0) found[0] = e0 + l;
        }
        before += __shfl_sync(0xffffffffu, up, 31);
    }
    if (lane == 0) found[1] = count;
    if (count > 0 && lane < BN) place[lane] = c.plan[c.n + 1 + from + min(lane, count - 1)];
}

// 64 weight rows (with GLU: and their 64 up rows) x 8 MQ places of one expert per CTA of 128 threads; a thread owns 4 rows x MQ
// places, 16-byte reads of shared memory, three stages of 32 k filled by asynchronous copies.  k is added up 256 at a time, so that
// chains of roundings stay short.  Instructions bound it, and places that a tile has no use for cost as many as the others.
constexpr int GF_THREADS = 128, GF_BM = 64, GF_BK = 32, GF_ST = GF_BK + 4, GF_STAGES = 3, GF_PART = 8;

template <bool GLU, int MQ>
__global__ void __launch_bounds__(GF_THREADS) k_group_f32(const __grid_constant__ GroupP P) {
    constexpr int GF_BN = 8 * MQ, NG = GLU ? 2 : 1, ROWS = NG * GF_BM + GF_BN;
    extern __shared__ __align__(16) float gf_smem[];
    __shared__ int place[GF_BN];
    __shared__ int found[2];
    const int tid = threadIdx.x, n = tid & 15, m = tid >> 4;
    const int n0 = blockIdx.x * GF_BM;
    if (tid < 32) find_tile<GF_BN>(P.c, blockIdx.y, tid, found, place);
    __syncthreads();
    const int count = found[1];
    if (count == 0) return;
    const float* W = (const float*)P.W + (long)found[0] * NG * P.M * P.ldw;
    const int nk = (P.K + GF_BK - 1) / GF_BK;
    auto copy = [&](int c, int stage) {
        float* dst = gf_smem + stage * ROWS * GF_ST;
        if (c < nk) {
#pragma unroll
            for (int e = tid; e < ROWS * (GF_BK / 4); e += GF_THREADS) {
                const int r = e >> 3, k = c * GF_BK + (e & 7) * 4;          // K is a multiple of 8
                const float* src;
                bool ok = k < P.K;
                if (r < NG * GF_BM) {
                    const int row = n0 + (r & (GF_BM - 1));
                    ok = ok && row < P.M;
                    src = W + (long)((r / GF_BM) * P.M + row) * P.ldw + k;
                } else {
                    src = (const float*)P.X + (long)(place[r - NG * GF_BM] / P.per) * P.ldx + k;
                }
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + r * GF_ST + (e & 7) * 4)),
                             "l"(ok ? src : (const float*)P.W), "r"(ok ? 16 : 0)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float acc[NG][MQ][4], all[NG][MQ][4];
#pragma unroll
    for (int a = 0; a < NG; a++)
#pragma unroll
        for (int i = 0; i < MQ; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[a][i][j] = all[a][i][j] = 0.0f;
#pragma unroll
    for (int s = 0; s < GF_STAGES - 1; s++) copy(s, s);
    int stage = 0;
    for (int c = 0; c < nk; c++) {
        asm volatile("cp.async.wait_group %0;" ::"n"(GF_STAGES - 2) : "memory");
        __syncthreads();                                   // chunk c is there, chunk c - 1 is used up
        copy(c + GF_STAGES - 1, stage == 0 ? GF_STAGES - 1 : stage - 1);
        const float4* w4 = (const float4*)(gf_smem + (stage * ROWS + n) * GF_ST);
        const float4* x4 = (const float4*)(gf_smem + (stage * ROWS + NG * GF_BM + m * MQ) * GF_ST);
#pragma unroll 4
        for (int k = 0; k < GF_BK / 4; k++) {
            float4 x[MQ];
#pragma unroll
            for (int i = 0; i < MQ; i++) x[i] = x4[i * (GF_ST / 4) + k];
#pragma unroll
            for (int a = 0; a < NG; a++) {
                float4 w[4];
#pragma unroll
                for (int j = 0; j < 4; j++) w[j] = w4[(a * GF_BM + 16 * j) * (GF_ST / 4) + k];
#pragma unroll
                for (int i = 0; i < MQ; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        acc[a][i][j] = fmaf(w[j].w, x[i].w, fmaf(w[j].z, x[i].z, fmaf(w[j].y, x[i].y, fmaf(w[j].x, x[i].x, acc[a][i][j]))));
            }
        }
        stage = stage == GF_STAGES - 1 ? 0 : stage + 1;
        if (c % GF_PART == GF_PART - 1 || c + 1 == nk) {
#pragma unroll
            for (int a = 0; a < NG; a++)
#pragma unroll
                for (int i = 0; i < MQ; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        all[a][i][j] += acc[a][i][j];
                        acc[a][i][j] = 0.0f;
                    }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
    for (int i = 0; i < MQ; i++) {
        if (m * MQ + i >= count) break;
        const long y = (long)place[m * MQ + i] * P.ldy;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = n0 + n + 16 * j;
            if (row >= P.M) break;
            if (GLU) glu_store<float>(P.epi, P.Y, y + row, all[0][i][j], all[NG - 1][i][j]);
            else ((float*)P.Y)[y + row] = all[0][i][j];
        }
    }
}

// Few places an expert: up to 16 of them per CTA of four warps.  A warp owns four weight rows (two gate rows and their up rows),
// streams them through registers once, 16 bytes a lane and a chunk of 256 k ahead, and multiplies them with the places' rows from
// shared memory; the 64 sums go over the lanes at the end.  Bound by the matrices' bytes until reads of shared memory, one for 16
// multiply-adds, take as long.  (16 experts of 616 x 896 gated, 148 places: 34 us; register-blocked tiles of 64 rows x 16 places 50,
// x 32 places 63.)
constexpr int FM_PLACES = 16, FM_K = 256;

template <bool GLU>
__global__ void __launch_bounds__(128, 3) k_group_f32_few(const __grid_constant__ GroupP P) {
    __shared__ __align__(16) float4 sx[2][FM_PLACES][FM_K / 4];
    __shared__ int place[FM_PLACES], found[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nq = P.K / 4, nk = (P.K + FM_K - 1) / FM_K;
    if (tid < 32) find_tile<FM_PLACES>(P.c, blockIdx.y, tid, found, place);
    __syncthreads();
    const int count = found[1];
    if (count == 0) return;
    const int r0 = (blockIdx.x * 4 + warp) * (GLU ? 2 : 4);      // first pair or row
    const float4* w[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int row = GLU ? min(r0 + (r & 1), P.M - 1) + (r >> 1) * P.M : min(r0 + r, P.M - 1);
        w[r] = (const float4*)((const float*)P.W + ((long)found[0] * (GLU ? 2 : 1) * P.M + row) * P.ldw);
    }
    auto copy = [&](int c) {
        if (c < nk) {
#pragma unroll
            for (int e = tid; e < FM_PLACES * (FM_K / 4); e += 128) {
                const int p = e / (FM_K / 4), x = e % (FM_K / 4), q = c * (FM_K / 4) + x;
                const bool ok = p < count && q < nq;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(&sx[c & 1][p][x])),
                             "l"(ok ? (const float4*)((const float*)P.X + (long)(place[p] / P.per) * P.ldx) + q : (const float4*)P.W), "r"(ok ? 16 : 0)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int4 next[4][2];
    auto fetch = [&](int c) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int q = c * (FM_K / 4) + lane + 32 * u;
                next[r][u] = q < nq ? ld_stream_v4(w[r] + q) : make_int4(0, 0, 0, 0);
            }
    };
    float acc[4 * FM_PLACES];
#pragma unroll
    for (int i = 0; i < 4 * FM_PLACES; i++) acc[i] = 0.0f;
    copy(0);
    fetch(0);
    for (int c = 0; c < nk; c++) {
        float4 v[4][2];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                v[r][u] = make_float4(__int_as_float(next[r][u].x), __int_as_float(next[r][u].y), __int_as_float(next[r][u].z), __int_as_float(next[r][u].w));
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();             // chunk c is there, and nobody reads the one before
        copy(c + 1);
        if (c + 1 < nk) fetch(c + 1);
#pragma unroll
        for (int g = 0; g < FM_PLACES; g += 4) {
            if (g >= count) break;
#pragma unroll
            for (int p = g; p < g + 4; p++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float4 x = sx[c & 1][p][lane + 32 * u];
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        acc[r * FM_PLACES + p] = fmaf(v[r][u].w, x.w, fmaf(v[r][u].z, x.z, fmaf(v[r][u].y, x.y, fmaf(v[r][u].x, x.x, acc[r * FM_PLACES + p]))));
                }
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // at every step a lane hands on one half of its sums and keeps the other: it ends with numbers 2 lane and 2 lane + 1
#pragma unroll
    for (int s = 16; s > 0; s >>= 1)
#pragma unroll
        for (int i = 0; i < 2 * s; i++) {
            const bool up = (lane & s) != 0;
            const float give = up ? acc[i] : acc[i + 2 * s], have = up ? acc[i + 2 * s] : acc[i];
            acc[i] = have + __shfl_xor_sync(0xffffffffu, give, s);
        }
    const int r = lane >> 3, p = (lane & 7) * 2;
    float u[2];
#pragma unroll
    for (int i = 0; i < 2; i++) u[i] = __shfl_down_sync(0xffffffffu, acc[i], 16);      // the up rows' sums to the gate rows' lanes
    const int row = r0 + r;
    if (row >= P.M || (GLU && r >= 2)) return;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        if (p + i >= count) break;
        const long y = (long)place[p + i] * P.ldy + row;
        if (GLU) glu_store<float>(P.epi, P.Y, y, acc[i], u[i]);
        else ((float*)P.Y)[y] = acc[i];
    }
}

static int f32_tiles(const GroupP& P, int BN, long* tiles) {         // at most: one begun by every expert
    const long places = (long)P.c.T * P.c.top;
    *tiles = places < P.c.n ? places : P.c.n + (places - P.c.n) / BN;
    LT_REQUIRE(*tiles <= 65535, "experts' products: %ld places in fp32", places);
    return LT_OK;
}
template <bool GLU, int MQ>
static int launch_group_f32(const GroupP& P, cudaStream_t s) {
    constexpr int BN = 8 * MQ, SMEM = GF_STAGES * ((GLU ? 2 : 1) * GF_BM + BN) * GF_ST * 4;
    static PerDeviceOnce once;
    LT_ONCE(once, LT_CUDA(cudaFuncSetAttribute(k_group_f32<GLU, MQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM)));
    long tiles;
    const int rc = f32_tiles(P, BN, &tiles);
    if (rc != LT_OK) return rc;
    k_group_f32<GLU, MQ><<<dim3((P.M + GF_BM - 1) / GF_BM, (unsigned)tiles), GF_THREADS, SMEM, s>>>(P);
    return check_launch("experts' products");
}
template <bool GLU>
static int launch_group_f32_few(const GroupP& P, cudaStream_t s) {
    long tiles;
    const int rc = f32_tiles(P, FM_PLACES, &tiles);
    if (rc != LT_OK) return rc;
    const int rows = GLU ? 8 : 16;
    k_group_f32_few<GLU><<<dim3((P.M + rows - 1) / rows, (unsigned)tiles), 128, 0, s>>>(P);
    return check_launch("experts' products");
}
// By places of an expert.  Gated, 64 experts of 512 x 2048, us in registers / tiles of 32 places: 8 180 / 294, 16 275 / 321, 24 375 / 322.
// Sums, 2048 x 512, in registers / tiles of 16 / of 32: 4 91 / 92 / 125, 8 122 / 114 / 137, 16 180 / 147 / 156, 24 242 / 187 / 180.
// Gated tiles that leave SMs idle are in registers too, in many more CTAs.  (About so many tiles, us in registers /
// tiles: 82 of 2048 x 512 64 / 93, 92 of 4096 x 1024 127 / 174, 109 of 1616 x 264 66 / 76, 107 of 512 x 256 30 / 29, 208 of 896 x 616
// 90 / 69.)
template <bool GLU>
static int pick_group_f32(const GroupP& P, cudaStream_t s) {
    const long each = (long)P.c.T * P.c.top / P.c.n;
    const long tiles = (P.M + GF_BM - 1) / GF_BM * ((long)P.c.T * P.c.top / 32 + P.c.n / 2);
    if (each <= (GLU ? 18 : 5) || (GLU && tiles <= 3 * sm_count() / 4)) return launch_group_f32_few<GLU>(P, s);
    if (!GLU && each <= 20) return launch_group_f32<false, 2>(P, s);
    return launch_group_f32<GLU, 4>(P, s);
}

int launch_group(GroupP P, bool glu, bool f32, void* rows, cudaStream_t s) {
    if (f32) return glu ? pick_group_f32<true>(P, s) : pick_group_f32<false>(P, s);
    return glu ? pick_group_tc<true>(P, rows, s) : pick_group_tc<false>(P, rows, s);
}

// ---------------------------------------------------------------------------- sum over a token's places

// V columns a thread, four places' loads in flight
template <int V>
__global__ void __launch_bounds__(256) k_combine(const float* __restrict__ ws, const float* __restrict__ w, const float* __restrict__ ls, float* Y,
                                                 int ldy, int M, const __grid_constant__ lt_dn_choice c) {
    __shared__ float sw[32];
    __shared__ int from[32];             // the places that count, in order
    __shared__ int used;
    const int t = blockIdx.x, m = (blockIdx.y * 256 + threadIdx.x) * V;
    if (threadIdx.x < 32) {
        const int j = threadIdx.x, e = j < c.top ? c.ids[(long)t * c.top + j] : -1;
        const bool on = e >= 0 && e < c.n;
        const unsigned all = __ballot_sync(0xffffffffu, on);
        if (on) {
            const int at = __popc(all & ((1u << j) - 1));
            from[at] = j;
            sw[at] = w[(long)t * c.top + j];
        }
        if (j == 0) used = __popc(all);
    }
    __syncthreads();
    if (m >= M || used == 0) return;
    const float* in = ws + (long)t * c.top * M + m;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = 0.0f;
    for (int j = 0; j < used; j += 4) {
        float x[4][V];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (j + u >= used) break;
            const float* p = in + (long)from[j + u] * M;
            if (V == 4) *(float4*)x[u] = __ldcs((const float4*)p);
            else x[u][0] = __ldcs(p);
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (j + u >= used) break;
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = fmaf(sw[j + u], x[u][i], v[i]);
        }
    }
    float* y = Y + (long)t * ldy + m;
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = ls != nullptr ? ls[m + i] * v[i] : v[i];
    if (V == 4) {
        const float4 o = *(const float4*)y;
        *(float4*)y = make_float4(o.x + v[0], o.y + v[V > 1 ? 1 : 0], o.z + v[V > 1 ? 2 : 0], o.w + v[V > 1 ? 3 : 0]);
    } else {
        y[0] += v[0];
    }
}

int launch_combine(const float* ws, const float* w, const float* ls, float* Y, int ldy, int M, const lt_dn_choice& c, cudaStream_t s) {
    if (M % 4 == 0 && ldy % 4 == 0 && aligned16(ws) && aligned16(Y))
        k_combine<4><<<dim3(c.T, (M + 1023) / 1024), 256, 0, s>>>(ws, w, ls, Y, ldy, M, c);
    else
        k_combine<1><<<dim3(c.T, (M + 255) / 256), 256, 0, s>>>(ws, w, ls, Y, ldy, M, c);
    return check_launch("lt_dn_experts_sum");
}

}  // namespace dn
}  // namespace lt
