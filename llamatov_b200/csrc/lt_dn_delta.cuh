// The gated delta rule: what its token-order form (lt_dn_delta.cu) and its chunked form (lt_dn_delta_chunk.cu) share.
#pragma once
#include "lt_dn_common.cuh"

namespace lt {
namespace dn {

// Logarithms of decays below this are taken for it: e^x is 0 in fp32 long before, and differences of sums stay numbers.
constexpr float DELTA_LOG_MIN = -1e4f;

__device__ __forceinline__ float delta_log(float la) { return fmaxf(la, DELTA_LOG_MIN) + (la != la ? la : 0.0f); }

const char* delta_error(const lt_dn_delta* D);
const char* delta_seqs_error(const lt_dn_seqs* Q, int* rows);

}  // namespace dn
}  // namespace lt
