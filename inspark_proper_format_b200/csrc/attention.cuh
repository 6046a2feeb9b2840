// Softmax attention, streaming form: a warp walks over the keys of one (query, head) 32 at a
// time with the running maximum m and sum l of the softmax, all in FP32.
#pragma once

#include "kv_cache.cuh"

namespace isp {
namespace attn {

struct PromptParams {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  uint8_t* out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;   // strides, elements
  int64_t q_tokens, k_tokens;
  const int* cu_q;
  const int* cu_k;
  int batch, heads, kv_heads;
  float scale;
  int causal;
};

// acc[i] belongs to dim lane * (kD / 32) + i.
template <int kD>
struct RowState {
  float m = -INFINITY, l = 0.f;
  float acc[kD / 32] = {};
};

// One step over 32 keys: lane j holds the score s of key j (-inf: not visible); value(j, i)
// gives element i of this lane's dims of key j.
template <int kD, class Value>
ISP_D void softmax_step(RowState<kD>& st, float s, unsigned visible, Value value) {
  float top = s;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float m = fmaxf(st.m, top);
  const float base = m == -INFINITY ? 0.f : m;
  const float keep = __expf(st.m - base), p = __expf(s - base);
  st.m = m;
  float sum = p;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  st.l = st.l * keep + sum;
#pragma unroll
  for (int i = 0; i < kD / 32; ++i) st.acc[i] *= keep;
  for (int j = 0; j < 32; ++j) {
    if (!((visible >> j) & 1u)) continue;
    const float pj = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
    for (int i = 0; i < kD / 32; ++i) st.acc[i] += pj * value(j, i);
  }
}

template <int kType>
ISP_D float load1(const void* p) {
  if constexpr (kType == ISP_F32) return *reinterpret_cast<const float*>(p);
  else if constexpr (kType == ISP_BF16) return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
  else if constexpr (kType == ISP_F16) return __half2float(*reinterpret_cast<const __half*>(p));
  else if constexpr (kType == ISP_E4M3) return e4m3_to_f32(*reinterpret_cast<const uint8_t*>(p));
  else return static_cast<float>(*reinterpret_cast<const int8_t*>(p));
}
template <int kType>
ISP_D void store1(void* p, float x) {
  if constexpr (kType == ISP_BF16) *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(x);
  else *reinterpret_cast<__half*>(p) = __float2half_rn(x);
}

template <int kD, int kType>
ISP_D float dot(const void* row, const float* q) {
  float s = 0.f;
#pragma unroll 4
  for (int c = 0; c < kD / 8; ++c) {
    float x[8];
    kv::load8<kType>(static_cast<const uint8_t*>(row) + c * 8 * kv::type_bytes(kType), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += x[j] * q[c * 8 + j];
  }
  return s;
}

constexpr int kWarps = 4;

// grid (query tokens / kWarps, heads)
template <int kD, int kType>
__global__ void __launch_bounds__(kWarps * 32) prompt_kernel(const PromptParams p) {
  constexpr int kB = 2;
  __shared__ float qs[kWarps][kD];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int h = blockIdx.y, hk = h / (p.heads / p.kv_heads);
  if (i >= p.q_tokens) return;
  for (int d = lane; d < kD; d += 32) qs[warp][d] = load1<kType>(p.q + (i * p.q_token + h * p.q_head + d) * kB) * p.scale;
  __syncwarp();
  const int b = kv::sequence_of(p.cu_q, p.batch, i);
  const int64_t q0 = p.cu_q[b], q1 = p.cu_q[b + 1], k0 = p.cu_k[b], k1 = p.cu_k[b + 1];
  int64_t visible = 0;
  if (i >= q0 && i < q1) {
    if (k0 < 0 || k1 < k0 || k1 > p.k_tokens) kv::record_bad_index();
    else visible = p.causal ? (i - q0) + 1 + (k1 - k0) - (q1 - q0) : k1 - k0;
  }
  RowState<kD> st;
  for (int64_t j0 = 0; j0 < visible; j0 += 32) {
    const int n = static_cast<int>(min(static_cast<int64_t>(32), visible - j0));
    const unsigned mask = n == 32 ? 0xffffffffu : (1u << n) - 1u;
    float s = -INFINITY;
    if (lane < n) s = dot<kD, kType>(p.k + ((k0 + j0 + lane) * p.k_token + hk * p.k_head) * kB, qs[warp]);
    softmax_step<kD>(st, s, mask, [&](int j, int d) {
      return load1<kType>(p.v + ((k0 + j0 + j) * p.v_token + hk * p.v_head + lane * (kD / 32) + d) * kB);
    });
  }
  const float inv = st.l == 0.f ? 0.f : 1.f / st.l;
#pragma unroll
  for (int d = 0; d < kD / 32; ++d)
    store1<kType>(p.out + (i * p.o_token + h * p.o_head + lane * (kD / 32) + d) * kB, st.acc[d] * inv);
}

}  // namespace attn
}  // namespace isp
