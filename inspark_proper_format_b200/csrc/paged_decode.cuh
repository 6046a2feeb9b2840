// Attention of one token per sequence over the paged cache, split over the cache's length.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = scale log2(e) q.k_j: one pass
// over K and V with the running maximum m, sum and weighted sum in FP32.  Bound by the
// bytes of the cache: every code and scale is read once per block of 8 query heads that
// share a key head.
//
// Split.  The unit of work is a step of kWarps * kT positions of one (sequence, key head,
// block of 8 query heads); all units in that order form one line, and every block of the
// grid takes an equal run of it, whatever the lengths are (they are read on the device).  A
// run that covers an item whole writes its result; pieces of an item go to the workspace,
// and the block that finishes an item's last piece joins them in piece order, so results do
// not depend on timing and no block waits for another.
//
// Each warp streams its own kT-row tiles of K and V through a ring in shared memory
// (cp.async, kStages deep, running on across items), 16 bytes a lane, rows found through
// the page table one tile ahead.  Rows past the length are zero-filled and masked, so
// stale rows never enter a product.
//
// Products run on mma.m16n8k16 in 16-bit types, keys (for K) and head dimensions (for V) on
// its 16 rows and the 8 query heads on its columns: S^T = K Q^T, O^T = V^T P^T.  With one
// query head per key head 7 of 8 columns are empty; the tensor pipe is far from the bound
// either way.  P^T's fragment is S^T's after one 8 x 8 transpose per 8 keys.  16-bit rows
// come as fragments by ldmatrix.  8-bit codes become FP16 in registers, which holds them
// exactly; the order of a row's elements inside a product is free, so each lane takes the
// 16 bytes it loads as its fragment, with keys in the order of key_row() that makes K's
// rows V's columns and keeps both reads free of bank conflicts.  Their scales go to the
// FP32 scores (K) and to p (V): p * v_scale carries a power of two that follows its largest
// value so far and keeps that between 2^6 and 2^15.  BF16 queries over 8-bit rows are brought
// into FP16's range by a power of two per head and keep all their bits down to 2^-31 of the
// head's largest element; below 2^-39 of it they are lost.  p is rounded to 16 bits: FP16 over
// 8-bit and FP16 rows (over the latter p times 2^7), BF16 over BF16 rows.  What FP16 cannot hold
// of a small weight goes into a second product, so weights keep the result's bits down to 2^-60
// of the largest.  (It costs 3% on the E4M3 case below, where few blocks of 16 keys have such
// weights, and 7% on the INT8 case, where a third have.)  Sums are FP32.
//
// Measured on one B200, launches of a captured graph over changing inputs: INT8, head_dim 128,
// 32 over 8 heads, 238651 cached tokens 106 us (4.8 TB/s; as calls 115 us); FP16, the same heads,
// 37 sequences of up to 6000 tokens 29.2 us (3.24 TB/s); E4M3, head_dim 64, 20 heads, 64
// sequences of 256 to 2048 tokens 46.4 us (3.27 TB/s), bound by latency in the warps' unpacking
// rather than by the copies, which alone take 29 us.
#pragma once

#include "kv_cache.cuh"

namespace isp {
namespace attn {

struct DecodeParams {
  kv::Cache cache;
  kv::Table table;
  const uint8_t* q;
  uint8_t* out;
  int64_t q_seq, q_head, o_seq, o_head;   // strides, elements
  int heads;
  int group;              // query heads per key head
  int gblocks;            // blocks of 8 query heads per key head
  int gb;                 // query heads of a full block: min(group, 8)
  float scale;            // softmax scale * log2(e)
  unsigned* counters;     // [kMaxBlocks], zero between calls
  float* partials;        // [2 * kMaxBlocks] pieces: [8][head_dim] weighted sums, [8] Refs
};

constexpr int kDecWarps = 4;
constexpr int kMaxBlocks = 1024;
constexpr int kSlotFloats = 8 * (128 + 4);
constexpr int64_t kDecWorkspace = kMaxBlocks * 4ll + 2ll * kMaxBlocks * kSlotFloats * 4;

// log2 of what a weighted sum and a sum of weights are in units of, and the sum of weights
struct __align__(16) Refs {
  float o, m, l, unused;
};

ISP_D void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
ISP_D void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// zeros where !valid (src is not read, but is a valid address)
ISP_D void cp_async16_or_zero(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
ISP_D void cp_async4_or_zero(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
ISP_D void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
ISP_D void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory"); }

ISP_D float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// D += A (16 x 16) B (16 x 8), FP32 accumulators.
struct Frag {
  uint32_t v[4];
  ISP_D uint32_t& operator[](int i) { return v[i]; }
  ISP_D const uint32_t& operator[](int i) const { return v[i]; }
};
template <bool kBf16>
ISP_D void mma16816(float (&c)[4], const Frag& a, uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <bool kBf16>
ISP_D uint32_t pack16(float lo, float hi) {
  if constexpr (kBf16) return pack_bf16_rn(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool kBf16>
ISP_D float2 unpack16(uint32_t w) {
  if constexpr (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
ISP_D uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}

// 8 x 8 matrix of 16-bit elements, transposed within the warp: lane (g, t) gives row g,
// elements 2t and 2t + 1, and takes the same of the transpose.
ISP_D uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <bool kTrans>
ISP_D Frag ldmatrix4(uint32_t addr) {
  Frag f;
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(f.v[0]), "=r"(f.v[1]), "=r"(f.v[2]), "=r"(f.v[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(f.v[0]), "=r"(f.v[1]), "=r"(f.v[2]), "=r"(f.v[3]) : "r"(addr) : "memory");
  return f;
}

// Codes as FP16, exactly: bytes 0 and 1 of `w` (lo) and bytes 2 and 3 (hi), each a pair in order.
template <int kCode>
ISP_D void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kCode == ISP_E4M3) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;                // code + 128
    const uint32_t a = prmt(u, 0x64646464u, 0x4140u), b = prmt(u, 0x64646464u, 0x4342u);   // 1024 + (code + 128)
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));                 // - 1152
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  }
}

template <int kD, int kCode>
struct Tile {
  static constexpr int kBytes = kv::type_bytes(kCode);
  static constexpr int kRow = kD * kBytes;                 // 64, 128 or 256 bytes
  static constexpr int kT = kRow == 256 ? 16 : 32;   // rows of a warp's tile
  static constexpr int kChunks = kRow / 16;
  static constexpr int kStep = kDecWarps * kT;             // positions of one unit of work
  // Ring depth and blocks per SM: 16 warps with two 4 KB tiles each in flight, or 12 with one
  // of 8 KB (three stages for two blocks, or 16-row tiles, are 2 to 10% slower).  The joins leave
  // room for a block less from 4 query heads to a key head on (codes), 5 (16-bit rows, head_dim
  // 128) or 8 (head_dim 64).
  static constexpr int kStages = kRow == 64 ? 3 : 2;
  static constexpr int kBlocks = kRow == 64 ? 4 : 3;
  // stage: K rows, V rows, per row {K scale, V scale}, the valid mask
  static constexpr int kV = kT * kRow, kScales = 2 * kV, kMask = kScales + 8 * kT, kBytesPerStage = kMask + 16;
  static constexpr int kRing = kDecWarps * kStages * kBytesPerStage;
  static constexpr int smem_bytes(int gb) { return kRing + kDecWarps * gb * (kD + 4) * 4; }
};

// 16-byte chunk c of row r lies at chunk c ^ swizzle(r), so that the 8 lanes of a 16-byte
// read phase hit all banks once: for codes two rows x four chunks (K) and four rows x two
// chunks (V) in the order of key_row(), for 16-bit rows the eight rows of an ldmatrix.
// swizzle(a ^ b) = swizzle(a) ^ swizzle(b), and it depends on r's low three bits alone.
template <int kRow, bool kIsCode>
ISP_HD constexpr int swizzle(int r) {
  return !kIsCode ? r & 7 : (kRow == 64 ? ((r >> 1) & 1) * 2 : (2 * (r & 3)) ^ (r & 4));
}

// Tile row of key n of a block of 8 keys, for codes.
ISP_D int key_row(int n) { return (n & 1) ? 4 + ((n >> 1) ^ 1) : n >> 1; }

// Position on the line of work units.
struct Cursor {
  int b, hg, step, steps, len;
};

ISP_D int clamp_length(int len, const DecodeParams& p) {
  const int64_t most = static_cast<int64_t>(p.table.width) * p.cache.page_size;
  if (len > most) {
    kv::record_bad_index();
    len = static_cast<int>(most);
  }
  return max(len, 0);
}

template <int kStep>
ISP_D void advance(Cursor& c, const DecodeParams& p) {
  if (++c.step < c.steps) return;
  c.step = 0;
  if (++c.hg < p.cache.heads * p.gblocks) return;
  c.hg = 0;
  do {
    ++c.b;
    c.len = c.b < p.table.batch ? clamp_length(p.table.lengths[c.b], p) : 0;
    c.steps = (c.len + kStep - 1) / kStep;
  } while (c.steps == 0 && c.b < p.table.batch);
}

template <int kD, int kCode, int kType>
__global__ void __launch_bounds__(kDecWarps * 32, Tile<kD, kCode>::kBlocks) decode_kernel(const DecodeParams p) {
  using T = Tile<kD, kCode>;
  constexpr bool kIsCode = kv::is_code(kCode);
  constexpr bool kMmaBf16 = kCode == ISP_BF16;
  constexpr bool kQBf16 = kType == ISP_BF16;
  constexpr int kT = T::kT, kRow = T::kRow, kStep = T::kStep, kStages = T::kStages;
  constexpr int kKSteps = kD / 16;
  constexpr int kKeyBlocks = kT / 16;
  constexpr int kOBlocks = kD / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kAtOnce = 8;                           // 32-sequence groups whose lengths are read together
  __shared__ int64_t line[2];                          // units in all, units before the first sequence
  __shared__ int first[2];                             // the first sequence and its length
  __shared__ unsigned arrived;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + warp * kStages * T::kBytesPerStage;
  float* joins = reinterpret_cast<float*>(smem + T::kRing);   // [warp][gb][kD] weighted sums, [warp][gb] Refs
  Refs* joins_refs = reinterpret_cast<Refs*>(joins + kDecWarps * p.gb * kD);
  const int hgs = p.cache.heads * p.gblocks;
  pdl_wait();
  pdl_trigger();

  // ---- this block's run of the line: [u0, u0 + count) ----
  if (warp == 0) {
    int len[kAtOnce];
    const auto read = [&](int b0) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int b = b0 + 32 * i + lane;
        len[i] = b < p.table.batch ? p.table.lengths[b] : 0;
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) len[i] = clamp_length(len[i], p);
    };
    int64_t total = 0;
    for (int b0 = 0; b0 < p.table.batch; b0 += 32 * kAtOnce) {
      read(b0);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (b0 + 32 * i < p.table.batch) total += __reduce_add_sync(0xffffffffu, (len[i] + kStep - 1) / kStep);
    }
    const int64_t per = (total * hgs + gridDim.x - 1) / gridDim.x;
    const int64_t u0 = per * blockIdx.x;
    int64_t before = 0;
    bool found = u0 >= total * hgs;
    for (int b0 = 0; b0 < p.table.batch && !found; b0 += 32 * kAtOnce) {
      if (p.table.batch > 32 * kAtOnce) read(b0);      // else still held
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (found || b0 + 32 * i >= p.table.batch) continue;
        const int steps = (len[i] + kStep - 1) / kStep;
        int sum = steps;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, (before + sum) * hgs > u0);
        if (hit != 0) {
          const int l = __ffs(hit) - 1;
          if (lane == l) {
            line[1] = (before + sum - steps) * hgs;
            first[0] = b0 + 32 * i + l;
            first[1] = len[i];
          }
          found = true;
        } else {
          before += __shfl_sync(0xffffffffu, sum, 31);
        }
      }
    }
    if (lane == 0) line[0] = total * hgs;
  } else if (warp == 1) {
    // sequences without a position give zeros (the grid's blocks share them)
    for (int b = blockIdx.x; b < p.table.batch; b += gridDim.x) {
      if (p.table.lengths[b] > 0) continue;
      for (int i = lane; i < p.heads * (kD / 2); i += 32)
        *reinterpret_cast<uint32_t*>(p.out + (b * p.o_seq + (i / (kD / 2)) * p.o_head + 2 * (i % (kD / 2))) * 2) = 0u;
    }
  }
  __syncthreads();
  const int64_t total = line[0];
  const int64_t per = (total + gridDim.x - 1) / gridDim.x;
  const int64_t u0 = per * blockIdx.x;
  if (u0 >= total) return;
  const int count = static_cast<int>(min(per, total - u0));   // units of this run

  Cursor at;                                           // the unit computed next
  at.b = first[0];
  at.len = first[1];
  at.steps = (at.len + kStep - 1) / kStep;
  at.hg = static_cast<int>((u0 - line[1]) / at.steps);
  at.step = static_cast<int>((u0 - line[1]) % at.steps);
  Cursor ahead = at;                                   // the unit whose copies start next
  int issued = 0;

  // Row of this lane's position of unit `ahead` (head 0 rows + head offset).
  uint32_t row = 0;
  bool row_ok = false;
  auto find_row = [&]() {
    row_ok = false;
    const int pos = ahead.step * kStep + warp * kT + lane;
    if (lane < kT && pos < ahead.len) {
      const int slot = kv::page_of(p.cache, pos);      // inside the table: lengths are clamped to it
      const int page = p.table.pages[ahead.b * p.table.stride + slot];
      row_ok = static_cast<unsigned>(page) < static_cast<uint64_t>(p.cache.pages);
      if (!row_ok) kv::record_bad_index();
      const int hk = p.gblocks == 1 ? ahead.hg : ahead.hg / p.gblocks;
      row = (static_cast<uint32_t>(page) * p.cache.heads + hk) * p.cache.page_size + (pos - slot * p.cache.page_size);
    }
  };
  const uint32_t ring_u32 = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  constexpr int kRowsPer = 32 / T::kChunks;            // rows that one 16-byte-a-lane access covers
  const int chunk = lane % T::kChunks, sub = lane / T::kChunks;
  const uint8_t* const k_base = p.cache.k + chunk * 16;
  const uint8_t* const v_base = p.cache.v + chunk * 16;
  // where this lane's chunk of its row of a group goes
  const uint32_t copy_to = static_cast<uint32_t>(sub * kRow);
  const int copy_chunk = chunk ^ swizzle<kRow, kIsCode>(sub);
  // Start the copies of unit `ahead` into its stage (rows found before), and find the next unit's rows.
  int stage_in = 0, stage_out = 0;
  constexpr unsigned kAll = kT == 32 ? 0xffffffffu : (1u << kT) - 1u;
  auto issue = [&]() {
    if (issued < count) {
      const uint32_t base = ring_u32 + stage_in * T::kBytesPerStage;
      const unsigned mask = __ballot_sync(0xffffffffu, row_ok);
      if (lane == 0) *reinterpret_cast<unsigned*>(ring + stage_in * T::kBytesPerStage + T::kMask) = mask;
      if (mask == kAll) {
#pragma unroll
        for (int i = 0; i < kT / kRowsPer; ++i) {
          const uint64_t src = static_cast<uint64_t>(__shfl_sync(0xffffffffu, row, i * kRowsPer + sub)) * kRow;
          const uint32_t dst = base + copy_to + ((copy_chunk ^ swizzle<kRow, kIsCode>(i * kRowsPer)) << 4) + i * kRowsPer * kRow;
          cp_async16(dst, k_base + src);
          cp_async16(dst + T::kV, v_base + src);
        }
        if (kIsCode && lane < kT) {
          cp_async4(base + T::kScales + lane * 8, p.cache.k_scale + row);
          cp_async4(base + T::kScales + lane * 8 + 4, p.cache.v_scale + row);
        }
      } else {                                         // the sequence's end, or a bad page: zeros
        if (!row_ok) row = 0u;
        for (int i = 0; i < kT / kRowsPer; ++i) {
          const uint64_t src = static_cast<uint64_t>(__shfl_sync(0xffffffffu, row, i * kRowsPer + sub)) * kRow;
          const uint32_t dst = base + copy_to + ((copy_chunk ^ swizzle<kRow, kIsCode>(i * kRowsPer)) << 4) + i * kRowsPer * kRow;
          const bool ok = (mask >> (i * kRowsPer + sub)) & 1u;
          cp_async16_or_zero(dst, k_base + src, ok);
          cp_async16_or_zero(dst + T::kV, v_base + src, ok);
        }
        if (kIsCode && lane < kT) {
          cp_async4_or_zero(base + T::kScales + lane * 8, p.cache.k_scale + row, row_ok);
          cp_async4_or_zero(base + T::kScales + lane * 8 + 4, p.cache.v_scale + row, row_ok);
        }
      }
      if (++issued < count) {
        advance<kStep>(ahead, p);
        find_row();
      }
      if (++stage_in == kStages) stage_in = 0;
    }
    cp_commit();
  };
  find_row();
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue();

  // This lane's places in a stage.  Codes: its 16-byte chunks of K's row key_row(g) of 8
  // keys, its elements of V's rows of keys 2t and 2t + 1 of 8.  16-bit rows: its row and
  // chunk for ldmatrix.  Its keys' scales: rows kr and kr + 8 of each 16.
  const int kr = kIsCode ? key_row(g) : g;
  const int v0 = key_row(2 * t), v1 = key_row(2 * t + 1);
  const int v_chunk = kRow == 64 ? g >> 1 : g, v_byte = kRow == 64 ? (g & 1) * 8 : 0;
  int k_at[kIsCode ? T::kChunks / 4 : 1];
  if constexpr (kIsCode) {
#pragma unroll
    for (int i = 0; i < T::kChunks / 4; ++i) k_at[i] = kr * kRow + (((t + 4 * i) ^ swizzle<kRow, true>(kr)) << 4);
  } else {
    k_at[0] = 0;
  }
  const int v_at0 = T::kV + v0 * kRow + ((v_chunk ^ swizzle<kRow, true>(v0)) << 4) + v_byte;
  const int v_at1 = T::kV + v1 * kRow + ((v_chunk ^ swizzle<kRow, true>(v1)) << 4) + v_byte;
  // ldmatrix: lanes 0-7, 8-15, 16-23, 24-31 name the rows of the four 8 x 8 matrices
  const int lm_row = (lane & 7) + (lane & 8), lm_chunk = lane >> 4;              // K: keys 0-7, 8-15, then the next 8 dims
  const int lv_row = (lane & 7) + (lane >> 4) * 8, lv_chunk = (lane >> 3) & 1;   // V: dims 0-7, 8-15, then the next 8 keys

  uint32_t qb[kKSteps][2];
  float q_unit[2] = {p.scale, p.scale};                // heads 2t, 2t + 1: softmax scale over the power of two in qb
  // Heads 2t and 2t + 1.  l = sum of p = 2^(s - m) over this lane's keys, m following the maximum
  // of s.  Over 8-bit rows p * v_scale enters the product with V as p * v_scale * c, c = 2^(m - r +
  // kUp), where r follows the largest s + log2(v_scale): the largest weight in use lies in (2^(kUp
  // - 1), 2^15], whatever the scales of rows are whose own weight is small.  Either reference may
  // stay up to kSlack behind, so that most tiles rescale nothing.
  constexpr float kSlack = 8.f, kUp = 15.f - kSlack;
  // Below 2^-17 (2^-14) FP16 has fewer bits than the result's 8 (11): the bits of that limit
  constexpr unsigned kSmall = kQBf16 ? 0x37000000u : 0x38800000u;
  constexpr float kRestUnits = 0x1p40f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, r[2] = {-INFINITY, -INFINITY}, c[2] = {0.f, 0.f};
  // log2 of |v_scale|, rounded up; scales under 2^-64 are not brought up
  const auto log2_above = [](float v) { return fmaxf(static_cast<float>(static_cast<int>((__float_as_uint(v) >> 23) & 255u) - 126), -64.f); };
  float o[kOBlocks][4];

  for (int u = 0; u < count; ++u) {
    if (u == 0 || at.step == 0) {                      // a new item
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      r[0] = r[1] = -INFINITY;
      c[0] = c[1] = 0.f;
#pragma unroll
      for (int i = 0; i < kOBlocks; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
      const int hk = at.hg / p.gblocks, gq = (at.hg % p.gblocks) * 8 + g;
      const bool mine = g < p.gb && gq < p.group;
      const uint8_t* qr = p.q + (at.b * p.q_seq + (hk * p.group + (mine ? gq : 0)) * p.q_head) * 2;
#pragma unroll
      for (int ks = 0; ks < kKSteps; ++ks) {
        qb[ks][0] = qb[ks][1] = 0u;
        if (!mine) continue;
        if constexpr (kIsCode) {                       // the order of a lane's chunks as they lie in K's rows
          const uint2 w = *reinterpret_cast<const uint2*>(qr + (16 * (t + 4 * (ks / 4)) + 4 * (ks % 4)) * 2);
          qb[ks][0] = w.x;
          qb[ks][1] = w.y;
        } else {
          qb[ks][0] = *reinterpret_cast<const uint32_t*>(qr + (16 * ks + 2 * t) * 2);
          qb[ks][1] = *reinterpret_cast<const uint32_t*>(qr + (16 * ks + 8 + 2 * t) * 2);
        }
      }
      if constexpr (kIsCode && kQBf16) {
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < kKSteps; ++ks) {
          const float2 a = unpack16<true>(qb[ks][0]), b = unpack16<true>(qb[ks][1]);
          top = fmaxf(fmaxf(top, fmaxf(fabsf(a.x), fabsf(a.y))), fmaxf(fabsf(b.x), fabsf(b.y)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // top * unit in [2^14, 2^15); the exponent of unit kept inside FP32
        const int e = max(1, min(254, 127 + 14 + 127 - static_cast<int>(__float_as_uint(top) >> 23)));
        const float unit = __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
        for (int ks = 0; ks < kKSteps; ++ks) {
          const float2 a = unpack16<true>(qb[ks][0]), b = unpack16<true>(qb[ks][1]);
          qb[ks][0] = pack16<false>(a.x * unit, a.y * unit);
          qb[ks][1] = pack16<false>(b.x * unit, b.y * unit);
        }
        q_unit[0] = p.scale / __shfl_sync(0xffffffffu, unit, 8 * t);
        q_unit[1] = p.scale / __shfl_sync(0xffffffffu, unit, 8 * t + 4);
      }
    }
    cp_wait<kStages - 2>();
    __syncwarp();                                      // unit u has landed, unit u - 1's stage is free
    issue();
    const uint8_t* st = ring + stage_out * T::kBytesPerStage;
    const uint32_t st_u32 = ring_u32 + stage_out * T::kBytesPerStage;
    if (++stage_out == kStages) stage_out = 0;
    const unsigned mask = *reinterpret_cast<const unsigned*>(st + T::kMask);

    // ---- scores of keys kr and kr + 8 of each 16, heads 2t and 2t + 1 ----
    float s[kKeyBlocks][4];                            // {key kr: two heads, key kr + 8: two heads}
    float2 f[kKeyBlocks][2];                           // {K scale, V scale} of the two keys
#pragma unroll
    for (int kb = 0; kb < kKeyBlocks; ++kb) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[kb][j] = 0.f;
      if constexpr (kIsCode) {
        f[kb][0] = *reinterpret_cast<const float2*>(st + T::kScales + kr * 8 + kb * 128);
        f[kb][1] = *reinterpret_cast<const float2*>(st + T::kScales + kr * 8 + kb * 128 + 64);
#pragma unroll
        for (int i = 0; i < T::kChunks / 4; ++i) {
          const uint4 wa = *reinterpret_cast<const uint4*>(st + k_at[i] + kb * 16 * kRow);
          const uint4 wb = *reinterpret_cast<const uint4*>(st + k_at[i] + kb * 16 * kRow + 8 * kRow);
          const uint32_t a[4] = {wa.x, wa.y, wa.z, wa.w}, b[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            Frag k;
            codes_to_f16<kCode>(a[j], k[0], k[2]);
            codes_to_f16<kCode>(b[j], k[1], k[3]);
            mma16816<false>(s[kb], k, qb[i * 4 + j][0], qb[i * 4 + j][1]);
          }
        }
        const float a = f[kb][0].x, b = f[kb][1].x;
        s[kb][0] *= a * q_unit[0];
        s[kb][1] *= a * q_unit[1];
        s[kb][2] *= b * q_unit[0];
        s[kb][3] *= b * q_unit[1];
      } else {
#pragma unroll
        for (int ks = 0; ks < kKSteps; ++ks) {
          const int r = kb * 16 + lm_row;
          const Frag k = ldmatrix4<false>(st_u32 + r * kRow + (((2 * ks + lm_chunk) ^ (lane & 7)) << 4));
          mma16816<kMmaBf16>(s[kb], k, qb[ks][0], qb[ks][1]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s[kb][j] *= p.scale;
      }
    }
    if (mask != kAll) {
#pragma unroll
      for (int kb = 0; kb < kKeyBlocks; ++kb) {
        if (!((mask >> (kb * 16 + kr)) & 1u)) s[kb][0] = s[kb][1] = -INFINITY;
        if (!((mask >> (kb * 16 + kr + 8)) & 1u)) s[kb][2] = s[kb][3] = -INFINITY;
      }
    }

    // ---- references: move them when a score or a product passes them ----
    float top[2] = {s[0][0], s[0][1]};
#pragma unroll
    for (int kb = 0; kb < kKeyBlocks; ++kb) {
      top[0] = fmaxf(top[0], fmaxf(s[kb][0], s[kb][2]));
      top[1] = fmaxf(top[1], fmaxf(s[kb][1], s[kb][3]));
    }
    bool past = top[0] > m[0] + kSlack || top[1] > m[1] + kSlack;
    if constexpr (kIsCode) {
      float v_top = 0.f;                               // a NaN scale is dropped: its row's weight is NaN anyway
#pragma unroll
      for (int kb = 0; kb < kKeyBlocks; ++kb) v_top = fmaxf(v_top, fmaxf(fabsf(f[kb][0].y), fabsf(f[kb][1].y)));
      const float above = log2_above(v_top);           // top + above: no product of this lane lies higher
      past = past || top[0] + above > r[0] + kSlack || top[1] + above > r[1] + kSlack;
    }
    if (__any_sync(0xffffffffu, past)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float product = -INFINITY;                     // the largest s + log2(v_scale)
        if constexpr (kIsCode) {
#pragma unroll
          for (int kb = 0; kb < kKeyBlocks; ++kb)
            product = fmaxf(product, fmaxf(s[kb][h] + log2_above(f[kb][0].y), s[kb][2 + h] + log2_above(f[kb][1].y)));
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], d));
          if constexpr (kIsCode) product = fmaxf(product, __shfl_xor_sync(0xffffffffu, product, d));
        }
        const float m_old = m[h], r_old = r[h];
        if (top[h] > m[h] + kSlack) m[h] = top[h];
        const float keep_l = m_old == -INFINITY ? 0.f : exp2_approx(m_old - m[h]);
        float keep_o = keep_l;
        l[h] *= keep_l;
        if constexpr (kIsCode) {
          if (product > r[h] + kSlack) r[h] = product;
          keep_o = r_old == -INFINITY ? 0.f : exp2_approx(r_old - r[h]);
          c[h] = r[h] == -INFINITY ? 0.f : exp2_approx(m[h] - r[h] + kUp);
        }
#pragma unroll
        for (int i = 0; i < kOBlocks; ++i) {
          o[i][h] *= keep_o;
          o[i][2 + h] *= keep_o;
        }
      }
    }
    // over FP16 rows the weights are placed as high as FP16 allows, sums and weighted sums alike
    constexpr float kPlace = kCode == ISP_F16 ? kUp : 0.f;
    const float base[2] = {(m[0] == -INFINITY ? 0.f : m[0]) - kPlace, (m[1] == -INFINITY ? 0.f : m[1]) - kPlace};

    // ---- weights and their product with V, 16 keys at a time ----
    // V's fragments of key block kb, one for every 16 head dimensions, to `use`
    const auto each_v = [&](int kb, const auto& use) {
      if constexpr (kIsCode) {
        // this lane's kD / 8 elements of each row: kD / 8 * g ..; row g of output block j takes
        // element 2j, row g + 8 element 2j + 1
        constexpr int kWords = kD / 32;
        uint32_t x[4][kWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* from = st + ((i & 1) ? v_at1 : v_at0) + (16 * kb + 8 * (i >> 1)) * kRow;
          if constexpr (kD == 64) {
            const uint2 y = *reinterpret_cast<const uint2*>(from);
            x[i][0] = y.x; x[i][1] = y.y;
          } else {
            const uint4 y = *reinterpret_cast<const uint4*>(from);
            x[i][0] = y.x; x[i][1] = y.y; x[i][2] = y.z; x[i][3] = y.w;
          }
        }
#pragma unroll
        for (int j = 0; j < kOBlocks; ++j) {
          const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;     // {key a e, key b e, key a e + 1, key b e + 1}
          Frag v;
          codes_to_f16<kCode>(prmt(x[0][j / 2], x[1][j / 2], sel), v[0], v[1]);
          codes_to_f16<kCode>(prmt(x[2][j / 2], x[3][j / 2], sel), v[2], v[3]);
          use(j, v);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kOBlocks; ++j) {
          const int r = kb * 16 + lv_row;
          use(j, ldmatrix4<true>(st_u32 + T::kV + r * kRow + (((2 * j + lv_chunk) ^ (lane & 7)) << 4)));
        }
      }
    };
#pragma unroll
    for (int kb = 0; kb < kKeyBlocks; ++kb) {
      float w[4];
      unsigned least = 0xFFFFFFFFu;                    // of the weights' bits, minus 1, so that 0 counts as large
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = exp2_approx(s[kb][j] - base[j & 1]);
        l[j & 1] += w[j];
        if constexpr (kIsCode) w[j] = w[j] * c[j & 1] * f[kb][j >> 1].y;
        least = min(least, __float_as_uint(w[j]) - 1u);
      }
      const uint32_t p01 = pack16<kMmaBf16>(w[0], w[1]), p23 = pack16<kMmaBf16>(w[2], w[3]);
      const uint32_t b0 = transpose8x8(p01), b1 = transpose8x8(p23);
      each_v(kb, [&](int j, const Frag& v) { mma16816<kMmaBf16>(o[j], v, b0, b1); });
      if constexpr (!kMmaBf16) {
        if (__any_sync(0xffffffffu, least < kSmall - 1u)) {
          // The rounding left at most 2^-25 of a small weight.  It counts where the rows with the
          // larger products are 0, so it is added in a second product, in units of 2^-40.
          const auto left = [&](float x, float rounded) { return __float_as_uint(x) < kSmall ? (x - rounded) * kRestUnits : 0.f; };
          const float2 r01 = unpack16<false>(p01), r23 = unpack16<false>(p23);
          const uint32_t c0 = transpose8x8(pack16<false>(left(w[0], r01.x), left(w[1], r01.y)));
          const uint32_t c1 = transpose8x8(pack16<false>(left(w[2], r23.x), left(w[3], r23.y)));
          each_v(kb, [&](int j, const Frag& v) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816<false>(x, v, c0, c1);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = fmaf(x[i], 1.f / kRestUnits, o[j][i]);
          });
        }
      }
    }

    // ---- end of the item, or of this run ----
    if (at.step + 1 == at.steps || u + 1 == count) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
        if (2 * t + h < p.gb) {
          const int mine = warp * p.gb + 2 * t + h;
#pragma unroll
          for (int j = 0; j < kOBlocks; ++j) {
            const int d0 = kIsCode ? g * (kD / 8) + 2 * j : 16 * j + g;
            joins[mine * kD + d0] = o[j][h];
            joins[mine * kD + d0 + (kIsCode ? 1 : 8)] = o[j][2 + h];
          }
          if (g == 0) joins_refs[mine] = {kIsCode ? r[h] - kUp : m[h], m[h], l[h], 0.f};
        }
      }
      __syncthreads();
      const int hk = at.hg / p.gblocks, head0 = hk * p.group + (at.hg % p.gblocks) * 8;
      const int n = min(8, p.group - (at.hg % p.gblocks) * 8);
      const int64_t begin = u0 + u - at.step, end = begin + at.steps;   // the item's units
      // the four sums in shared memory as one: the result, or this run's piece of it.  Weighted sums and
      // sums of weights are added in units of their own, which meet in the quotient.
      const auto or_zero = [](float x) { return x == -INFINITY ? 0.f : x; };
      const auto join = [&](float* slot) {
        for (int i = threadIdx.x; i < n * (kD / 4); i += kDecWarps * 32) {
          const int h = i / (kD / 4), d = i % (kD / 4) * 4;
          Refs refs[kDecWarps];
          Refs top = {-INFINITY, -INFINITY, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) {
            refs[w] = joins_refs[w * p.gb + h];
            top.o = fmaxf(top.o, refs[w].o);
            top.m = fmaxf(top.m, refs[w].m);
          }
          const float ref_o = or_zero(top.o), ref_m = or_zero(top.m);
          float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) {
            const float f = exp2_approx(refs[w].o - ref_o);
            const float4 x = *reinterpret_cast<const float4*>(joins + (w * p.gb + h) * kD + d);
            top.l += (kIsCode ? exp2_approx(refs[w].m - ref_m) : f) * refs[w].l;
            r.x += f * x.x;
            r.y += f * x.y;
            r.z += f * x.z;
            r.w += f * x.w;
          }
          if (slot != nullptr) {
            __stcg(reinterpret_cast<float4*>(slot + h * kD + d), r);
            if (d == 0) __stcg(reinterpret_cast<float4*>(slot + 8 * kD) + h, make_float4(top.o, top.m, top.l, 0.f));
          } else {
            const float inv = top.l == 0.f ? 0.f : 1.f / top.l, unit = kIsCode ? exp2_approx(ref_o - ref_m) : 1.f;
            uint8_t* dst = p.out + (at.b * p.o_seq + (head0 + h) * p.o_head + d) * 2;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<kQBf16>(r.x * inv * unit, r.y * inv * unit),
                                                        pack16<kQBf16>(r.z * inv * unit, r.w * inv * unit));
          }
        }
      };
      if (begin >= u0 && end <= u0 + count) {
        join(nullptr);
      } else {
        join(p.partials + static_cast<int64_t>(2 * blockIdx.x + (begin >= u0 ? 1 : 0)) * kSlotFloats);
        const int64_t b0 = begin / per, b1 = (end - 1) / per;           // the blocks that hold its pieces
        __syncthreads();
        if (threadIdx.x == 0) {
          __threadfence();
          arrived = atomicAdd(p.counters + b0, 1u);
          __threadfence();
        }
        __syncthreads();
        if (arrived == static_cast<unsigned>(b1 - b0)) {
          // the last piece: groups of kD / 4 lanes take every kGroups-th piece, four at a time
          constexpr int kLanes = kD / 4, kGroups = kDecWarps * 32 / kLanes;
          const int group = threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4;
          for (int h = 0; h < n; ++h) {
            Refs top = {-INFINITY, -INFINITY, 0.f, 0.f};
            float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
            const auto scale = [&](float f, float f_l) {
              top.l *= f_l;
              r.x *= f;
              r.y *= f;
              r.z *= f;
              r.w *= f;
            };
            for (int64_t b = b0 + group; b <= b1; b += 4 * kGroups) {
              float4 refs[4], x[4];                    // Refs
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int64_t bi = b + i * kGroups;
                refs[i] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
                x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (bi <= b1) {
                  const float* src = p.partials + (2 * bi + (bi == b0 ? 1 : 0)) * kSlotFloats;
                  refs[i] = __ldcg(reinterpret_cast<const float4*>(src + 8 * kD) + h);
                  x[i] = __ldcg(reinterpret_cast<const float4*>(src + h * kD + d));
                }
              }
              const float now_o = fmaxf(fmaxf(fmaxf(refs[0].x, refs[1].x), fmaxf(refs[2].x, refs[3].x)), top.o);
              const float now_m = kIsCode ? fmaxf(fmaxf(fmaxf(refs[0].y, refs[1].y), fmaxf(refs[2].y, refs[3].y)), top.m) : now_o;
              const float ref_o = or_zero(now_o), ref_m = or_zero(now_m), keep = exp2_approx(top.o - ref_o);
              scale(keep, kIsCode ? exp2_approx(top.m - ref_m) : keep);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float f = exp2_approx(refs[i].x - ref_o);
                top.l += (kIsCode ? exp2_approx(refs[i].y - ref_m) : f) * refs[i].z;
                r.x += f * x[i].x;
                r.y += f * x[i].y;
                r.z += f * x[i].z;
                r.w += f * x[i].w;
              }
              top.o = now_o;
              top.m = now_m;
            }
            if constexpr (kLanes == 16) {              // the warp's two groups
              const float now_o = fmaxf(top.o, __shfl_xor_sync(0xffffffffu, top.o, 16));
              const float now_m = kIsCode ? fmaxf(top.m, __shfl_xor_sync(0xffffffffu, top.m, 16)) : now_o;
              const float f = exp2_approx(top.o - or_zero(now_o));
              scale(f, kIsCode ? exp2_approx(top.m - or_zero(now_m)) : f);
              top.l += __shfl_xor_sync(0xffffffffu, top.l, 16);
              r.x += __shfl_xor_sync(0xffffffffu, r.x, 16);
              r.y += __shfl_xor_sync(0xffffffffu, r.y, 16);
              r.z += __shfl_xor_sync(0xffffffffu, r.z, 16);
              r.w += __shfl_xor_sync(0xffffffffu, r.w, 16);
              top.o = now_o;
              top.m = now_m;
            }
            if (lane < kLanes) {
              *reinterpret_cast<float4*>(joins + (warp * p.gb + h) * kD + d) = r;
              if (lane == 0) joins_refs[warp * p.gb + h] = top;
            }
          }
          __syncthreads();
          join(nullptr);
          if (threadIdx.x == 0) p.counters[b0] = 0u;
        }
      }
      __syncthreads();                                 // joins is free
    }
    advance<kStep>(at, p);
  }
  cp_wait<0>();
}

}  // namespace attn
}  // namespace isp
