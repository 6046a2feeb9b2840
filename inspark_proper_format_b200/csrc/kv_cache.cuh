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
// position past the page table, a page id outside the pool or counts outside the call's rows
// are recorded in the device error word and treated the same way.
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

// Whether [first, end) are rows of a call with `tokens` rows.
ISP_D bool bounds_ok(int64_t first, int64_t end, int64_t tokens) { return first >= 0 && first <= end && end <= tokens; }

// Row (head 0) of packed token i of `tokens`, or -1.
ISP_D int64_t row_of_token(const Cache& c, const Table& t, const int* cu, int64_t i, int64_t tokens) {
  if (t.batch == 0) return -1;
  int b = static_cast<int>(i);
  int64_t first = i, end = i + 1;
  if (cu != nullptr) {
    b = sequence_of(cu, t.batch, i);
    first = cu[b];
    end = cu[b + 1];
    if (i < first || i >= end || !bounds_ok(first, end, tokens)) return -1;   // a token that no sequence claims
  }
  return row_of(c, t, b, static_cast<int>(t.lengths[b] - (end - first) + (i - first)));
}

// ---- eight elements of a row -------------------------------------------------------------
template <int kType>
ISP_D void load8(const void* p, float* x) {
  if constexpr (kType == ISP_F32) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    const float4 b = *(reinterpret_cast<const float4*>(p) + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else if constexpr (kType == ISP_BF16) {
    bf16x8_to_f32(*reinterpret_cast<const uint4*>(p), x);
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <int kType>
ISP_D void store8(void* p, const float* x) {
  if constexpr (kType == ISP_F32) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *(reinterpret_cast<float4*>(p) + 1) = make_float4(x[4], x[5], x[6], x[7]);
  } else if constexpr (kType == ISP_BF16) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16_rn(x[0], x[1]), pack_bf16_rn(x[2], x[3]),
                                              pack_bf16_rn(x[4], x[5]), pack_bf16_rn(x[6], x[7]));
  } else {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// Sixteen codes.
template <int kType>
ISP_D void codes16_to_f32(const uint4& w, float (&x)[16]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kType == ISP_E4M3) {
      uint32_t a, b;
      asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
          : "=r"(a), "=r"(b)
          : "r"(u[i]));
      const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&a)), hi = __half22float2(*reinterpret_cast<const __half2*>(&b));
      x[4 * i] = lo.x; x[4 * i + 1] = lo.y; x[4 * i + 2] = hi.x; x[4 * i + 3] = hi.y;
    } else {
      // 2^23 + (code + 128) as a float, minus 2^23 + 128: exact, and no conversion unit
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[4 * i + j] = __uint_as_float(__byte_perm(u[i] ^ 0x80808080u, 0x4B000000u, 0x7440u + j)) - 8388736.f;
    }
  }
}
template <int kType>
ISP_D uint4 f32_to_codes16(const float (&x)[16]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kType == ISP_E4M3) {
      u[i] = static_cast<uint32_t>(e4m3x2(x[4 * i], x[4 * i + 1])) | (static_cast<uint32_t>(e4m3x2(x[4 * i + 2], x[4 * i + 3])) << 16);
    } else {
      // |x| <= 127 after rounding: adding 1.5 * 2^23 rounds to the nearest even integer, whose low
      // byte is the code
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(__fadd_rn(x[4 * i + j], 12582912.f));
      u[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

ISP_HD constexpr int type_bytes(int t) { return t == ISP_F32 ? 4 : (t == ISP_BF16 || t == ISP_F16 ? 2 : 1); }
ISP_HD constexpr bool is_code(int t) { return t == ISP_E4M3 || t == ISP_I8; }

// Blocks of a multiprocessor: append in one wave, gather in four of eight.
ISP_HD constexpr int append_blocks(int code) { return is_code(code) ? 6 : 8; }
constexpr int kGatherBlocks = 32;

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
constexpr int kBoundsAtOnce = 1024;            // sequences whose bounds a block keeps in shared memory

// Rows (head 0) of the block's tokens into `rows`; returns their number.  A search in global
// memory is a chain of dependent loads, so the bounds are copied first where they fit.
ISP_D int find_rows(const RowParams& p, int64_t first, int64_t (&rows)[kMaxTokensPerBlock], int (&bounds)[kBoundsAtOnce + 1]) {
  const int n = static_cast<int>(min(static_cast<int64_t>(p.tokens_per_block), p.tokens - first));
  const int* cu = p.cu;
  if (cu != nullptr && blockIdx.x == 0) {
    for (int i = threadIdx.x; i < p.table.batch; i += kRowThreads)
      if (!bounds_ok(cu[i], cu[i + 1], p.tokens)) record_bad_index();
  }
  if (cu != nullptr && p.table.batch <= kBoundsAtOnce) {
    for (int i = threadIdx.x; i <= p.table.batch; i += kRowThreads) bounds[i] = p.cu[i];
    __syncthreads();
    cu = bounds;
  }
  if (threadIdx.x < n) rows[threadIdx.x] = row_of_token(p.cache, p.table, cu, first + threadIdx.x, p.tokens);
  __syncthreads();
  return n;
}

// The rows of a block, a group's every `by`-th: number i is token i % n of head i / n % heads of
// K or V, so neighbouring groups read and write neighbouring rows of a page.
struct RowWalk {
  int token, head, kv, n, heads, d_token, d_head, d_kv;
  ISP_D RowWalk(int first, int by, int n_, int heads_) : n(n_), heads(heads_) {
    token = first % n;
    head = first / n % heads;
    kv = first / n / heads;
    d_token = by % n;
    d_head = by / n % heads;
    d_kv = by / n / heads;
  }
  ISP_D bool inside() const { return kv < 2; }
  ISP_D void advance() {
    token += d_token;
    head += d_head;
    kv += d_kv;
    if (token >= n) {
      token -= n;
      ++head;
    }
    if (head >= heads) {
      head -= heads;
      ++kv;
    }
  }
};

// Both kernels are bound by the bytes they move: 16 elements a lane (8 for 16-bit caches) and
// kD / 16 lanes a row.  A block starts with the look-up of its tokens, three dependent loads.
// Append takes one wave of equal blocks, as many as its registers leave room for (16384 tokens,
// 20 heads of 64: INT8 32.7 us, in blocks of 256 rows 36.4, in more than one wave 36 to 43;
// BF16 rows 33.3 us, 37.5 in such blocks); gather, with less work a row, four waves, so that
// some blocks look up while others move (2% faster than blocks of 256 rows, 7% than one
// wave).  One row a lane at a time: two or four in flight cost registers, and with them more
// than they hid (10 and 45%).  Measured, append then gather on one B200, launches of a captured
// graph over changing inputs: INT8, 64 x 256 tokens, 20 heads of 64, 58.7 us (4.4 TB/s of 257
// MB); E4M3, 44246 tokens, 8 heads of 128, 109 us (5.0 TB/s of 549 MB), as calls 115 us.
template <int kD, int kIn, int kCode>
__global__ void __launch_bounds__(kRowThreads, append_blocks(kCode)) append_kernel(const RowParams p) {
  constexpr int kElems = is_code(kCode) ? 16 : 8, kLanes = kD / kElems;
  __shared__ int64_t rows[kMaxTokensPerBlock];
  __shared__ int bounds[kBoundsAtOnce + 1];
  pdl_wait();
  pdl_trigger();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int n = find_rows(p, first, rows, bounds);
  const int lane = threadIdx.x % kLanes;
  RowWalk at(threadIdx.x / kLanes, kRowThreads / kLanes, n, p.cache.heads);
  for (; __any_sync(0xffffffffu, at.inside()); at.advance()) {
    float x[kElems];
    int64_t row = at.inside() ? rows[at.token] : -1;
    if (row >= 0) {
      row += static_cast<int64_t>(at.head) * p.cache.page_size;
      const uint8_t* src = p.x[at.kv] + ((first + at.token) * p.token_stride[at.kv] + at.head * p.head_stride[at.kv] + lane * kElems) * type_bytes(kIn);
#pragma unroll
      for (int e = 0; e < kElems; e += 8) load8<kIn>(src + e * type_bytes(kIn), &x[e]);
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) x[e] = 0.f;
    }
    uint8_t* dst = (at.kv == 0 ? p.cache.k : p.cache.v) + (row * kD + lane * kElems) * type_bytes(kCode);
    if constexpr (is_code(kCode)) {
      // the largest magnitude as bits, which also order infinities and NaN above the rest
      uint32_t top = 0u;
#pragma unroll
      for (int e = 0; e < kElems; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      const bool ok = top < 0x7F800000u;
      const float s = fmaxf(__fdiv_rn(__uint_as_float(top), kCode == ISP_E4M3 ? 448.f : 127.f), 1e-12f);
      const float y = __fdiv_rn(1.f, s);
      // RN(x / s) as in div_rn_recip; |x / s| <= 448 (1 + 2^-22) and 1e-12 <= s < 2^122, so its
      // range checks never apply
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        const float q = __fmul_rn(x[e], y);
        x[e] = ok ? __fmaf_rn(__fmaf_rn(-q, s, x[e]), y, q) : 0.f;
      }
      if (row >= 0) {
        *reinterpret_cast<uint4*>(dst) = f32_to_codes16<kCode>(x);
        if (lane == 0) (at.kv == 0 ? p.cache.k_scale : p.cache.v_scale)[row] = ok ? s : __int_as_float(0x7fc00000);
      }
    } else if (row >= 0) {
      store8<kCode>(dst, x);
    }
  }
}

template <int kD, int kCode, int kOut>
__global__ void __launch_bounds__(kRowThreads) gather_kernel(const RowParams p) {
  constexpr int kElems = is_code(kCode) ? 16 : 8, kLanes = kD / kElems;
  __shared__ int64_t rows[kMaxTokensPerBlock];
  __shared__ int bounds[kBoundsAtOnce + 1];
  pdl_wait();
  pdl_trigger();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tokens_per_block;
  const int n = find_rows(p, first, rows, bounds);
  const int lane = threadIdx.x % kLanes;
  RowWalk at(threadIdx.x / kLanes, kRowThreads / kLanes, n, p.cache.heads);
  for (; at.inside(); at.advance()) {
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    float scale = 0.f;
    int64_t row = rows[at.token];
    if (row >= 0) {
      row += static_cast<int64_t>(at.head) * p.cache.page_size;
      w = *reinterpret_cast<const uint4*>((at.kv == 0 ? p.cache.k : p.cache.v) + (row * kD + lane * kElems) * type_bytes(kCode));
      if constexpr (is_code(kCode)) scale = (at.kv == 0 ? p.cache.k_scale : p.cache.v_scale)[row];
    }
    float x[kElems];
    if constexpr (is_code(kCode)) {
      codes16_to_f32<kCode>(w, x);
#pragma unroll
      for (int e = 0; e < kElems; ++e) x[e] = __fmul_rn(x[e], scale);
    } else {
      load8<kCode>(&w, x);
    }
    uint8_t* dst = p.x[at.kv] + ((first + at.token) * p.token_stride[at.kv] + at.head * p.head_stride[at.kv] + lane * kElems) * type_bytes(kOut);
#pragma unroll
    for (int e = 0; e < kElems; e += 8) store8<kOut>(dst + e * type_bytes(kOut), x + e);
  }
}

}  // namespace kv
}  // namespace isp
