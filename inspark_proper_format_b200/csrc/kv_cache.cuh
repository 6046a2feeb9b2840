// Paged key-value cache: rows quantised as they are written, and read back.
//
// A cache holds K and V as [pages, kv_heads, page_size, head_dim] in BF16, FP16, E4M3 or
// INT8.  For the 8-bit formats every (token, head) row carries one FP32 scale,
//   s = max(amax / Q, 1e-12),  code = RNE(x / s),   Q = 448 (E4M3) or 127 (INT8),
// amax and both quotients in FP32, correctly rounded (the per-row E4M3 rule that the
// activation quantiser uses).  A row with a non-finite element gets scale NaN and codes 0,
// so it reads back as NaN whatever the format does with infinities.
//
// Token i of sequence b's n_b = cu[b + 1] - cu[b] tokens has position lengths[b] - n_b + i
// (lengths counts the tokens of this call), found in page table[b][position / page_size].
// A negative position means "no such token": nothing is written, zeros are read.  A
// position past the page table or a page id outside the pool is recorded in the device
// error word and treated the same way.
#pragma once

#include "common.cuh"

namespace isp {
namespace kv {

struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;        // [pages, heads, page_size], 8-bit formats only
  float* v_scale;
  int64_t pages;
  int page_size;
  int heads;
  // n / page_size = (n * page_mul) >> page_shift for 0 <= n < 2^31: page_shift = 31 + s,
  // 2^s >= page_size, page_mul = ceil(2^page_shift / page_size), whose excess times n stays
  // below 2^page_shift
  uint32_t page_mul;
  int page_shift;
};

ISP_HD int page_of(const Cache& c, int pos) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(pos)) * c.page_mul) >> c.page_shift);
}

struct Table {
  const int* pages;      // [batch, stride]
  int64_t stride;
  int width;
  const int* lengths;    // [batch]
  int batch;
};

// An index read from device memory (page id, length, sequence bound) is out of its range.
ISP_D void record_bad_index() { atomicExch(&g_device_error, (int)ISP_ERR_ARG); }

// Row of position `pos` of head 0 of sequence b: (page * heads) * page_size + offset, or
// -1.  Head h lies h * page_size rows further on.
ISP_D int64_t row_of(const Cache& c, const Table& t, int b, int pos) {
  if (pos < 0) return -1;
  const int slot = page_of(c, pos);
  if (slot >= t.width) {
    record_bad_index();
    return -1;
  }
  const int page = t.pages[b * t.stride + slot];
  if (page < 0 || page >= c.pages) {
    record_bad_index();
    return -1;
  }
  return static_cast<int64_t>(page) * c.heads * c.page_size + (pos - slot * c.page_size);
}

// Sequence of packed token i: the last b with cu[b] <= i (cu ascending).
ISP_D int sequence_of(const int* cu, int batch, int64_t i) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Row (head 0) of packed token i, or -1.
ISP_D int64_t row_of_token(const Cache& c, const Table& t, const int* cu, int64_t i) {
  int b = static_cast<int>(i);
  int64_t first = i, end = i + 1;
  if (cu != nullptr) {
    b = sequence_of(cu, t.batch, i);
    first = cu[b];
    end = cu[b + 1];
    if (i < first || i >= end) return -1;      // a token that no sequence claims
  }
  return row_of(c, t, b, static_cast<int>(t.lengths[b] - (end - first) + (i - first)));
}

// ---- eight elements of a row -------------------------------------------------------------
template <int kType>
ISP_D void load8(const void* p, float (&x)[8]) {
  if constexpr (kType == ISP_F32) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else if constexpr (kType == ISP_BF16) {
    bf16x8_to_f32(*reinterpret_cast<const uint4*>(p), x);
  } else if constexpr (kType == ISP_F16) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint8_t c = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
      if constexpr (kType == ISP_E4M3) x[i] = e4m3_to_f32(c);
      else x[i] = static_cast<float>(static_cast<int8_t>(c));
    }
  }
}

template <int kType>
ISP_D void store8(void* p, const float (&x)[8]) {
  if constexpr (kType == ISP_F32) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *(reinterpret_cast<float4*>(p) + 1) = make_float4(x[4], x[5], x[6], x[7]);
  } else if constexpr (kType == ISP_BF16) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16_rn(x[0], x[1]), pack_bf16_rn(x[2], x[3]),
                                              pack_bf16_rn(x[4], x[5]), pack_bf16_rn(x[6], x[7]));
  } else if constexpr (kType == ISP_F16) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    uint32_t u[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t c;
      if constexpr (kType == ISP_E4M3) c = e4m3x2(x[i], 0.f) & 0xFFu;
      else c = static_cast<uint8_t>(int8_rne_sat(x[i]));
      u[i / 4] |= c << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
  }
}

ISP_HD constexpr int type_bytes(int t) { return t == ISP_F32 ? 4 : (t == ISP_BF16 || t == ISP_F16 ? 2 : 1); }
ISP_HD constexpr bool is_code(int t) { return t == ISP_E4M3 || t == ISP_I8; }

struct RowParams {
  Cache cache;
  Table table;
  const int* cu;          // [batch + 1], or nullptr: one token per sequence
  int64_t tokens;
  uint8_t* x[2];          // K, V rows: [tokens, heads, head_dim] by strides (append reads, gather writes)
  int64_t token_stride[2], head_stride[2];   // elements
  int tokens_per_block;
};

constexpr int kRowThreads = 256;
constexpr int kMaxTokensPerBlock = 64;

// kD / 8 lanes hold one row; a block covers tokens_per_block tokens x all heads x {K, V}.
template <int kD, int kIn, int kCode>
__global__ void __launch_bounds__(kRowThreads) append_kernel(const RowParams p) {
  constexpr int kLanes = kD / 8;
  __shared__ int64_t rows[kMaxTokensPerBlock];
  pdl_wait();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.tokens_per_block), p.tokens - first));
  if (threadIdx.x < n) rows[threadIdx.x] = row_of_token(p.cache, p.table, p.cu, first + threadIdx.x);
  __syncthreads();
  const int lane = threadIdx.x % kLanes;
  const int per_token = 2 * p.cache.heads;
  for (int i = threadIdx.x / kLanes; i < n * per_token; i += kRowThreads / kLanes) {
    const int tok = i / per_token;
    const int kv = (i % per_token) / p.cache.heads, h = i % p.cache.heads;
    const int64_t row0 = rows[tok];
    if (row0 < 0) continue;                     // uniform over the row's lanes
    float x[8];
    load8<kIn>(p.x[kv] + ((first + tok) * p.token_stride[kv] + h * p.head_stride[kv] + lane * 8) * type_bytes(kIn), x);
    const int64_t row = row0 + static_cast<int64_t>(h) * p.cache.page_size;
    uint8_t* dst = (kv ? p.cache.v : p.cache.k) + (row * kD + lane * 8) * type_bytes(kCode);
    if constexpr (is_code(kCode)) {
      float amax = 0.f;
      bool finite = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        amax = fmaxf(amax, fabsf(x[j]));
        finite = finite && (fabsf(x[j]) < __int_as_float(0x7f800000));
      }
      if (!finite) amax = __int_as_float(0x7f800000);
      const unsigned mask = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u)) << ((threadIdx.x & 31) / kLanes * kLanes);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
      const bool ok = amax < __int_as_float(0x7f800000);
      const float s = fmaxf(__fdiv_rn(amax, kCode == ISP_E4M3 ? 448.f : 127.f), 1e-12f);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = ok ? __fdiv_rn(x[j], s) : 0.f;
      store8<kCode>(dst, x);
      if (lane == 0) (kv ? p.cache.v_scale : p.cache.k_scale)[row] = ok ? s : __int_as_float(0x7fc00000);
    } else {
      store8<kCode>(dst, x);
    }
  }
}

template <int kD, int kCode, int kOut>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(const RowParams p) {
  constexpr int kLanes = kD / 8;
  __shared__ int64_t rows[kMaxTokensPerBlock];
  pdl_wait();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int n = static_cast<int>(min(static_cast<int64_t>(p.tokens_per_block), p.tokens - first));
  if (threadIdx.x < n) rows[threadIdx.x] = row_of_token(p.cache, p.table, p.cu, first + threadIdx.x);
  __syncthreads();
  const int lane = threadIdx.x % kLanes;
  const int per_token = 2 * p.cache.heads;
  for (int i = threadIdx.x / kLanes; i < n * per_token; i += kRowThreads / kLanes) {
    const int tok = i / per_token;
    const int kv = (i % per_token) / p.cache.heads, h = i % p.cache.heads;
    const int64_t row0 = rows[tok];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row0 >= 0) {
      const int64_t row = row0 + static_cast<int64_t>(h) * p.cache.page_size;
      load8<kCode>((kv ? p.cache.v : p.cache.k) + (row * kD + lane * 8) * type_bytes(kCode), x);
      if constexpr (is_code(kCode)) {
        const float s = (kv ? p.cache.v_scale : p.cache.k_scale)[row];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(x[j], s);
      }
    }
    store8<kOut>(p.x[kv] + ((first + tok) * p.token_stride[kv] + h * p.head_stride[kv] + lane * 8) * type_bytes(kOut), x);
  }
}

}  // namespace kv
}  // namespace isp
