// The experts' products: what the forms for few places (lt_dn_experts.cu) and for many (lt_dn_experts_group.cu) share.
#pragma once
#include "lt_dn_common.cuh"

namespace lt {
namespace dn {

struct GroupP {
    const void* W;
    const void* X;
    void* Y;
    int* status;
    int M, K, ldw, ldx, ldy;     // M: gate rows (glu) or output rows
    int per;                     // places that share a row of X: top (glu) or 1
    int row_tiles;
    lt_dn_choice c;
    lt_dn_epilogue epi;
};
// Y[p] = products of place p, with the plan of P.c: gated outputs in the element type, or fp32 sums.  rows: bf16, K elements a place
int launch_group(GroupP P, bool glu, bool f32, void* rows, cudaStream_t s);

// Y[t] += ls * sum_j w[t][j] ws[t * top + j]
int launch_combine(const float* ws, const float* w, const float* ls, float* Y, int ldy, int M, const lt_dn_choice& c, cudaStream_t s);

}  // namespace dn
}  // namespace lt
