// What the two attention kernels over the 4-bit cache share.
#pragma once

#include "kernels.h"
#include "kv_cache.cuh"

namespace sage3 {

// The running maximum of a row need not be its maximum: weights are 2^(s - m + kTop), and m is brought up to date only where a score
// passes it by more than kSlack.  Weights stay below 2^15, within fp16, and those of 2^-20 of the largest keep all their bits.
constexpr float kTop = 6.f, kSlack = 9.f;
constexpr float kLowest = -1e38f;         // the maximum of a row that has seen no key

// Where a sequence's rows and keys lie; every bound that memory accesses rely on is taken here.  What a bound leaves out - rows beyond max_q
// or the tensor, keys beyond the table or max_k - moves nothing else: the causal diagonal goes by the lengths as they are.
struct KvSeq {
  int q0, q_len, kv_len;
  int ahead;                              // keys in front of the first row's own; within 32 bits, as a difference of two lengths
  __device__ __forceinline__ KvSeq(const KvAttnArgs& A, int b) {
    q0 = b; q_len = 1;
    if (A.cu_q != nullptr) { q0 = __ldg(A.cu_q + b); q_len = __ldg(A.cu_q + b + 1) - q0; }
    if (q0 < 0 || q_len < 0 || q0 > A.tokens) { q0 = 0; q_len = 0; }
    kv_len = max(__ldg(A.kv_lens + b), 0);
    ahead = kv_len - q_len;
    q_len = min(min(q_len, A.max_q), A.tokens - q0);
    kv_len = (int)min((int64_t)min(kv_len, A.max_k), (int64_t)A.cols * A.page_size);
  }
  // keys that token t (below q_len) of the sequence sees
  __device__ __forceinline__ int seen(const KvAttnArgs& A, int t) const { return A.causal ? max(0, min(kv_len, ahead + t + 1)) : kv_len; }
};

// A query's scale: 2^(14 - exponent) of its largest channel, so that bf16 values become fp16 values exactly (down to 2^-31 of the
// largest), within the normal numbers; and what undoes it.
struct RowScale {
  float up, undo;
  __device__ __forceinline__ explicit RowScale(float largest) {
    const int field = min(268 - (int)(__float_as_uint(largest) >> 23), 253);
    up = __uint_as_float((uint32_t)field << 23);
    undo = __uint_as_float((uint32_t)(254 - field) << 23);
  }
};

// LSE of a row from its maximum and sum (of weights as above)
__device__ __forceinline__ float lse_of(float m, float l, float add) {
  return l == 0.f ? -INFINITY : (m - kTop + log2f(l)) * 0.6931471805599453f + add;
}

}  // namespace sage3
