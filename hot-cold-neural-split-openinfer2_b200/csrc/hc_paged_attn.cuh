// Shared parts of the paged-attention kernels: arguments, element types, requests.
#pragma once

#include <type_traits>

#include "hc_common.cuh"

namespace hca8 {
using namespace hc;

constexpr int MAX_REQ = 2048;
constexpr uint32_t NONE = 0xffffffffu; // no page
constexpr int KEPT_REQ = 256;          // requests whose lengths stay in shared memory
constexpr float M_NONE = -1e30f;       // softmax reference before the first key
// Weights are 2^(t - m), rounded to f16 for the product, and f16's step is 2^-24 at the bottom: the larger the
// greatest weight, the smaller a weight may be beside it.  A row's reference m is put W_REF below its largest
// exponent and moves when a weight would pass 2^W_MAX (65504 is the largest f16).  A weight of 2^-d of the largest
// is then rounded by at most max(2^-11, 2^(d - 36)) of itself.  A window of 2^4 keeps moves rare: scores with a
// deviation of 1 never leave it after the first keys.
constexpr float W_REF = 11.0f, W_MAX = 15.0f;
constexpr float VS_MIN = 0x1p-80f;     // value scales below count as this: 2^W_MAX / VS_MIN times 2^31 keys stays in fp32
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct AttnParams {
  const void* q;
  void* out;
  float* lse;
  int64_t q_row, q_head, o_row, o_head;
  const int32_t* tables;
  int64_t t_stride;
  int width;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  int n_req, n_rows, nq, nkv, g;
  float scale2;                        // scale * log2(e)
  const uint8_t* kp;
  const uint8_t* vp;
  const float* ks;
  const float* vs;
  int n_pages, page_log2;
  int rows_from, rows_to;              // requests of rows_from <= q_len * g < rows_to are served
  float* part;                         // [grid][2][RT (D + 2)]: partials of a share's first and last item
  int4* cuts;                          // [grid][2]: the divided item that begins in a share
  // tiles of 256 rows: pieces of cut tiles
  int sms;
  int4* pf_cuts;                       // slots in use; then tile and number of pieces of each slot
  float* pf_part;                      // [slot][256 (D + 2)]
  int32_t* status;
};

template <typename T>
__device__ __forceinline__ float load_f(const T* p);
template <>
__device__ __forceinline__ float load_f(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// new tokens and cached length of request r; q_len 0 when the step leaves it out
struct Req {
  int q0, q_len, kv;
};
__device__ __forceinline__ Req request(const AttnParams& p, int r, bool flag) {
  Req x;
  x.q0 = p.cu_q[r];
  const int q1 = p.cu_q[r + 1];
  x.kv = p.kv_lens[r];
  x.q_len = q1 - x.q0;
  if (x.q0 < 0 || q1 < x.q0 || q1 > p.n_rows || x.kv < 0 || x.kv > ((int64_t)p.width << p.page_log2)) {
    if (flag && p.status) atomicOr(p.status, HC_ERR_RANGE);
    x.q_len = 0;
  }
  if (x.q_len * p.g < p.rows_from || x.q_len * p.g >= p.rows_to) x.q_len = 0;
  return x;
}

// tiles of 256 rows on tcgen05 -- hc_paged_prefill.cu
int64_t prefill_workspace(int head_dim);
int launch_prefill(const AttnParams& p, int dtype, int head_dim, void* workspace, int sms, cudaStream_t stream);

}  // namespace hca8
