// Attention of packed sequences on the tensor cores (tcgen05), sm_100a.
//
// o_i = sum_j p_ij v_j / sum_j p_ij over the keys j that query i sees, p_ij =
// 2^(scale log2(e) q_i.k_j - m_i), with the running maximum m and sum of each row in FP32,
// one pass over K and V.
//
// A work item is a block of 256 queries of one (sequence, head): two tiles of 128 that share
// every K and V tile of 128 keys.  Blocks of the grid are persistent and take items in an
// order of falling block index, back and forth (static, so results and order are fixed).
// Roles of the 12 warps:
//   warps 0-3, 4-7  softmax of tile 0 and 1: a thread owns a row.  It takes the row's 128
//                   scores from TMEM, writes p in 16 bits over them, and at the end scales
//                   and stores the row's output.  m stays up to kSlack behind the maximum,
//                   so that most steps leave the accumulated output alone.
//   warp 8          issues the MMAs: S = Q K^T (both operands in shared memory) and
//                   O += P V (P in TMEM, V's tile read with its keys along K).  For each
//                   tile PV(j - 1) then S(j), the two tiles in turn, so one tile's softmax
//                   runs beside the other's MMAs.
//   warp 9          finds the items and loads Q and the ring of K and V tiles by TMA.
//   warps 10, 11    check the V tiles that hold keys some row must not see.  A product with
//                   p = 0 would turn an infinity or NaN there into NaN, so they are set to
//                   zero in shared memory; values that other rows do see are added to those
//                   rows at the end.
// Every wait is bounded; on expiry the block unwinds as the GEMMs do.
#pragma once

#include "gemm_sm100.cuh"
#include "kv_cache.cuh"

namespace isp {
namespace prompt {

struct Params {
  uint8_t* out;
  const uint8_t* v;             // the slow path of the V check reads single elements
  int64_t v_token, v_head, o_token, o_head;   // strides, elements
  int64_t q_tokens, k_tokens;
  const int* cu_q;
  const int* cu_k;
  int batch, heads, group;
  float scale;                  // softmax scale * log2(e)
  int causal;
  int out32;                    // 32-byte stores: rows of the output are 32-byte aligned
};

constexpr int kTile = 128;                  // queries of a tile, keys of a step
constexpr int kThreads = 384;
constexpr int kItemSlots = 4;
constexpr int kTmemColumns = 512;           // S0, S1, then O0, O1
constexpr float kSlack = 8.f;
#ifndef POLY
#define POLY 4
#endif
constexpr int kPolyEvery = POLY;            // one pair of exponentials in this many goes by polynomial
// registers of a softmax thread and of the other warps' threads (a sum over the launch's 384 x 168 would wait for ever)
constexpr int kSoftmaxRegs = 208, kOtherRegs = 80;
static_assert(2 * 128 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168, "");

template <int kD>
struct Layout {
  static constexpr int kTileBytes = kTile * kD * 2;            // a tile of Q, K or V: kD / 64 boxes of 128 rows x 128 bytes
  static constexpr int kStages = kD == 64 ? 8 : 5;             // K and V tiles in flight
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kTileBytes;
  static constexpr int kBars = kRing + kStages * kTileBytes;
  static constexpr int kBytes = kBars + 1024;
  static_assert(kStages <= 8, "at most four V tiles in the ring");
};

struct Item {
  int stop;              // no more items
  int head;
  int q0, rows;          // first query row, queries of the block
  int k0, keys;          // first key row, keys of the sequence
  int off;               // row r of the block sees the first min(keys, r + off + 1) keys
  int steps[2];          // key tiles of each query tile
  int edge;              // first key tile that some row does not see whole
  int flagged;           // the V check found non-finite values in view
  int pad[5];
};

struct Bars {
  uint64_t full[8], empty[8];                        // K and V ring
  uint64_t q_full, q_free;
  uint64_t s_full[2], p_full[2][2], o_full[2], o_free[2];   // p: keys 0-63, then 64-127
  // V tiles through the check, in order: their loads complete on v_in instead of the ring's
  // barrier (which the producer completes by hand), the check answers on v_ok.  The ring
  // holds at most four V tiles, so neither side is more than these ahead.
  uint64_t v_in[4], v_ok[4];
  uint64_t item_full[kItemSlots], item_free[kItemSlots];
  uint64_t drained;
  Item items[kItemSlots];
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Bars) <= 1024, "");

ISP_D uint32_t idesc(bool bf16, int n, bool b_mn_major) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

// V tile as B with its N (head dimension) contiguous: boxes of 64 elements x 128 keys, 128-byte
// swizzle; 8 keys are 1024 bytes apart (stride offset), 64 head dimensions a box (leading offset).
ISP_D uint64_t v_desc(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((kTile * 128) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

ISP_D void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n " ISP_ELECT_PRED
               " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
               "l"(a), "l"(b), "r"(desc), "r"(accumulate));
}
ISP_D void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n " ISP_ELECT_PRED
               " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
               "r"(a), "l"(b), "r"(desc), "r"(accumulate));
}
ISP_D void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
ISP_D void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
ISP_D void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

ISP_D float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The larger of three; NaN if one is.
ISP_D float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x for x <= 2^7 without the special function unit: x = n + f with n whole and |f| <= 1/2
// (adding 1.5 * 2^23 rounds to n), 2^f by the polynomial of least largest relative error on
// [-1/2, 1/2] (Remez; 2^-13.7 in degree 3, 2^-18.5 in degree 4, below the rounding to BF16
// and FP16), n added to the exponent.  x below -126 counts as -126.
template <bool kBf16>
ISP_D float2 ex2_poly(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f);
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 r = __fadd2_rn(x, magic);
  const float2 f = __fadd2_rn(x, __ffma2_rn(r, make_float2(-1.f, -1.f), magic));
  const auto two = [](float c) { return make_float2(c, c); };
  float2 y;
  if constexpr (kBf16) {
    y = __ffma2_rn(f, two(0.05517167f), two(0.24261113f));
    y = __ffma2_rn(f, y, two(0.69326097f));
    y = __ffma2_rn(f, y, two(0.99992806f));
  } else {
    y = __ffma2_rn(f, two(0.009570102f), two(0.05591786f));
    y = __ffma2_rn(f, y, two(0.24024744f));
    y = __ffma2_rn(f, y, two(0.6931218f));
    y = __ffma2_rn(f, y, two(0.9999993f));
  }
  return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(r.x) << 23)),
                     __int_as_float(__float_as_int(y.y) + (__float_as_int(r.y) << 23)));
}

template <bool kBf16>
ISP_D uint32_t pack(float a, float b) {
  return kBf16 ? gemm::pack_bf16(a, b) : gemm::pack_f16(a, b);
}

// Number of 256-query blocks of sequence b (0 where its bounds are bad).
ISP_D int blocks_of(const Params& p, int b) {
  if (b >= p.batch) return 0;
  const int64_t a = p.cu_q[b], e = p.cu_q[b + 1];
  if (a < 0 || e < a || e > p.q_tokens) {
    kv::record_bad_index();
    return 0;
  }
  return static_cast<int>((e - a + 2 * kTile - 1) / (2 * kTile));
}

// Blocks with index >= i in all sequences (whole warp).
ISP_D int64_t blocks_from(const Params& p, int i, int lane) {
  int64_t n = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) n += __reduce_add_sync(0xffffffffu, max(0, blocks_of(p, b0 + lane) - i));
  return n;
}

// Item number x in the order of falling block index (whole warp; `top`: blocks of the longest sequence).
ISP_D void find_item(const Params& p, int64_t x, int top, int lane, Item& it) {
  const int64_t block = x / p.heads;
  int lo = 0, hi = top - 1;                             // the largest i with blocks_from(i) > block
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (blocks_from(p, mid, lane) > block) lo = mid;
    else hi = mid - 1;
  }
  int rank = static_cast<int>(block - (lo + 1 < top ? blocks_from(p, lo + 1, lane) : 0));
  int seq = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {            // the rank-th sequence with more than lo blocks
    unsigned has = __ballot_sync(0xffffffffu, blocks_of(p, b0 + lane) > lo);
    const int n = __popc(has);
    if (rank < n) {
      for (; rank > 0; --rank) has &= has - 1;
      seq = b0 + __ffs(has) - 1;
      break;
    }
    rank -= n;
  }
  const int q_first = p.cu_q[seq], q_end = p.cu_q[seq + 1];
  int64_t k_first = p.cu_k[seq], k_end = p.cu_k[seq + 1];
  if (k_first < 0 || k_end < k_first || k_end > p.k_tokens) {
    kv::record_bad_index();
    k_first = k_end = 0;
  }
  it.stop = 0;
  it.head = static_cast<int>(x % p.heads);
  it.q0 = q_first + lo * 2 * kTile;
  it.rows = min(2 * kTile, q_end - it.q0);
  it.k0 = static_cast<int>(k_first);
  it.keys = static_cast<int>(k_end - k_first);
  it.off = p.causal ? (it.q0 - q_first) + it.keys - (q_end - q_first) : it.keys;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int last = min(it.rows, (t + 1) * kTile) - 1;
    const int seen = it.rows > t * kTile ? min(static_cast<int64_t>(it.keys), static_cast<int64_t>(last) + it.off + 1) : 0;
    it.steps[t] = max(0, (seen + kTile - 1) / kTile);
  }
  it.edge = max(0, min(it.keys, it.off < it.keys ? it.off + 1 : it.keys)) / kTile;
  it.flagged = 0;
}

// Whether one of two 16-bit values is infinite or NaN (exponent all ones).
template <bool kBf16>
ISP_D bool not_finite(uint32_t w) {
  const uint32_t mask = kBf16 ? 0x7F807F80u : 0x7C007C00u, one = kBf16 ? 0x00800080u : 0x04000400u;
  return (((w & mask) + one) & 0x80008000u) != 0;
}

template <int kD, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(const __grid_constant__ CUtensorMap q_map,
                                                             const __grid_constant__ CUtensorMap k_map,
                                                             const __grid_constant__ CUtensorMap v_map, const Params p) {
  using L = Layout<kD>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars& bars = *reinterpret_cast<Bars*>(smem + L::kBars);
  volatile int* const abort = &bars.abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      gemm::mbar_init(&bars.full[i], 1);
      gemm::mbar_init(&bars.empty[i], 1);
    }
    gemm::mbar_init(&bars.q_full, 1);
    gemm::mbar_init(&bars.q_free, 1);
    for (int t = 0; t < 2; ++t) {
      gemm::mbar_init(&bars.s_full[t], 1);
      gemm::mbar_init(&bars.p_full[t][0], 4);
      gemm::mbar_init(&bars.p_full[t][1], 4);
      gemm::mbar_init(&bars.o_full[t], 1);
      gemm::mbar_init(&bars.o_free[t], 4);
    }
    for (int i = 0; i < 4; ++i) {
      gemm::mbar_init(&bars.v_in[i], 1);
      gemm::mbar_init(&bars.v_ok[i], 2);
    }
    for (int i = 0; i < kItemSlots; ++i) {
      gemm::mbar_init(&bars.item_full[i], 1);
      gemm::mbar_init(&bars.item_free[i], 11);
    }
    gemm::mbar_init(&bars.drained, 1);
    bars.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gemm::smem_u32(&bars.tmem)),
                 "r"(kTmemColumns));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (warp == 9 && lane == 0) {
    gemm::prefetch_tmap(&q_map);
    gemm::prefetch_tmap(&k_map);
    gemm::prefetch_tmap(&v_map);
  }
  gemm::tc_fence_before();
  __syncthreads();
  gemm::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars.tmem);
  pdl_wait();
  pdl_trigger();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 9) {
      // ---- items and loads ----
      int top = 0;
      for (int b0 = 0; b0 < p.batch; b0 += 32) top = max(top, __reduce_max_sync(0xffffffffu, blocks_of(p, b0 + lane)));
      const int64_t total = blocks_from(p, 0, lane) * p.heads;
      uint32_t kv = 0, edges = 0;                        // tiles loaded into the ring, checked tiles among them
      int loaded = 0;                                    // items with loads
      bool ok = true;
      for (int64_t n = 0; ok; ++n) {
        const int slot = static_cast<int>(n % kItemSlots);
        const int64_t x = n * gridDim.x + ((n & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        Item it = {};
        it.stop = 1;
        if (x < total) find_item(p, x, top, lane, it);
        if (n >= kItemSlots && !gemm::wait_warp(&bars.item_free[slot], static_cast<uint32_t>((n / kItemSlots - 1) & 1), abort)) break;
        if (lane == 0) {
          bars.items[slot] = it;
          gemm::mbar_arrive(&bars.item_full[slot]);
        }
        __syncwarp();
        if (it.stop) break;
        const int steps = max(it.steps[0], it.steps[1]);
        if (steps == 0) continue;
        if (loaded > 0 && !(ok = gemm::wait_warp(&bars.q_free, (loaded - 1) & 1, abort))) break;
        ++loaded;
        if (lane == 0) {
          const int tiles = (it.steps[0] > 0) + (it.steps[1] > 0);
          gemm::mbar_expect_tx(&bars.q_full, tiles * L::kTileBytes);
          for (int t = 0; t < 2; ++t) {
            if (it.steps[t] == 0) continue;
            for (int c = 0; c < kD / 64; ++c)
              gemm::tma_load_3d(smem + L::kQ + t * L::kTileBytes + c * kTile * 128, &q_map, &bars.q_full, c * 64, it.head,
                                it.q0 + t * kTile);
          }
        }
        __syncwarp();
        for (int j = 0; j < 2 * steps; ++j, ++kv) {      // K0, V0, K1, V1, ...
          const uint32_t s = kv % L::kStages;
          if (kv >= L::kStages && !(ok = gemm::wait_warp(&bars.empty[s], (kv / L::kStages - 1) & 1, abort))) break;
          const bool check = (j & 1) && (j >> 1) >= it.edge;
          if (lane == 0) {
            uint64_t* const bar = check ? &bars.v_in[edges & 3] : &bars.full[s];
            gemm::mbar_expect_tx(bar, L::kTileBytes);
            for (int c = 0; c < kD / 64; ++c)
              gemm::tma_load_3d(smem + L::kRing + s * L::kTileBytes + c * kTile * 128, (j & 1) ? &v_map : &k_map, bar, c * 64,
                                it.head / p.group, it.k0 + (j >> 1) * kTile);
            if (check) gemm::mbar_arrive(&bars.full[s]);
          }
          edges += check;
          __syncwarp();
        }
      }
      // loads in flight land before the block ends
      if (*abort) {
        if (loaded > 0) gemm::wait_warp_drain(&bars.q_full, (loaded - 1) & 1);
        for (int i = 0; i < L::kStages; ++i)
          if (kv > static_cast<uint32_t>(i))               // (kv - 1 - i) / kStages: fills of stage i so far, minus one
            gemm::wait_warp_drain(&bars.full[i], ((kv - 1 - i) / L::kStages) & 1);
        for (int i = 0; i < 4; ++i)
          if (edges > static_cast<uint32_t>(i)) gemm::wait_warp_drain(&bars.v_in[i], ((edges - 1 - i) / 4) & 1);
      }
    } else if (warp == 8) {
      // ---- MMAs ----
      const uint32_t s_desc = idesc(kBf16, kTile, false), o_desc = idesc(kBf16, kD, true);
      const uint32_t q_addr = gemm::smem_u32(smem + L::kQ), ring = gemm::smem_u32(smem + L::kRing);
      uint32_t kv = 0;
      int loaded = 0, edges = 0;
      int s_count[2] = {0, 0}, o_count[2] = {0, 0};
      bool ok = true;
      for (int64_t n = 0; ok; ++n) {
        const int slot = static_cast<int>(n % kItemSlots);
        if (!gemm::wait_warp(&bars.item_full[slot], static_cast<uint32_t>((n / kItemSlots) & 1), abort)) break;
        const int stop = bars.items[slot].stop, edge = bars.items[slot].edge;
        const int steps0 = bars.items[slot].steps[0], steps1 = bars.items[slot].steps[1];
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&bars.item_free[slot]);
        if (stop) break;
        const int steps = max(steps0, steps1);
        if (steps == 0) continue;
        if (!(ok = gemm::wait_warp(&bars.q_full, loaded & 1, abort))) break;
        ++loaded;
        for (int j = 0; j <= steps && ok; ++j) {
          const uint32_t ik = kv + 2 * j, iv = kv + 2 * j - (j > 0);    // K_j and V_(j - 1) in the ring
          const uint32_t sk = ik % L::kStages, sv = iv % L::kStages;
          if (j < steps && !(ok = gemm::wait_warp(&bars.full[sk], (ik / L::kStages) & 1, abort))) break;
          if (j > 0) {
            if (j - 1 >= edge) {                                        // checked tiles
              if (!(ok = gemm::wait_warp(&bars.v_ok[edges & 3], (edges >> 2) & 1, abort))) break;
              ++edges;
            } else if (!(ok = gemm::wait_warp(&bars.full[sv], (iv / L::kStages) & 1, abort))) {
              break;
            }
          }
          gemm::tc_fence_after();
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int mine = t == 0 ? steps0 : steps1;
            const uint32_t s_tmem = tmem + t * kTile, o_tmem = tmem + 2 * kTile + t * kD;
            if (j > 0 && j - 1 < mine) {
              if (j == 1) {
                if (o_count[t] > 0 && !(ok = gemm::wait_warp(&bars.o_free[t], (o_count[t] - 1) & 1, abort))) break;
                ++o_count[t];
              }
              const uint64_t b = v_desc(ring + sv * L::kTileBytes);
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (!(ok = gemm::wait_warp(&bars.p_full[t][half], (s_count[t] - 1) & 1, abort))) break;
                gemm::tc_fence_after();
#pragma unroll
                for (int i = 0; i < kTile / 32; ++i) {                  // 16 keys: 8 columns of P, 2048 bytes of V
                  const int k = half * (kTile / 32) + i;
                  mma_ts(o_tmem, s_tmem + k * 8, b + ((k * 2048) >> 4), o_desc, j > 1 || k > 0);
                }
              }
              if (!ok) break;
              if (j == mine) gemm::mma_commit_elect<false>(&bars.o_full[t]);
            }
            if (j < mine) {
              const uint64_t a = gemm::smem_desc_sw128(q_addr + t * L::kTileBytes);
              const uint64_t b = gemm::smem_desc_sw128(ring + sk * L::kTileBytes);
#pragma unroll
              for (int k = 0; k < kD / 16; ++k) {                       // 16 head dimensions: 32 bytes of a row
                const int o = ((k / 4) * kTile * 128 + (k % 4) * 32) >> 4;
                mma_ss(s_tmem, a + o, b + o, s_desc, k > 0);
              }
              gemm::mma_commit_elect<false>(&bars.s_full[t]);
              ++s_count[t];
            }
          }
          if (!ok) break;
          if (j > 0) gemm::mma_commit_elect<false>(&bars.empty[sv]);
          if (j < steps) gemm::mma_commit_elect<false>(&bars.empty[sk]);
          if (j == steps - 1) gemm::mma_commit_elect<false>(&bars.q_free);
        }
        kv += 2 * steps;
      }
      // the MMAs issued end before TMEM is freed
      gemm::mma_commit_elect<false>(&bars.drained);
      gemm::wait_warp_drain(&bars.drained, 0);
    } else {
      // ---- V check: warps 10 and 11 take 64 keys of a tile each ----
      uint32_t kv = 0, edges = 0;
      for (int64_t n = 0;; ++n) {
        const int slot = static_cast<int>(n % kItemSlots);
        if (!gemm::wait_warp(&bars.item_full[slot], static_cast<uint32_t>((n / kItemSlots) & 1), abort)) break;
        const Item it = bars.items[slot];
        bool ok = true;
        const int steps = max(it.steps[0], it.steps[1]);
        for (int j = it.edge; j < steps && !it.stop; ++j) {
          const uint32_t i = kv + 2 * j + 1, s = i % L::kStages;
          if (!(ok = gemm::wait_warp(&bars.v_in[edges & 3], (edges >> 2) & 1, abort))) break;
          uint8_t* tile = smem + L::kRing + s * L::kTileBytes;
          const int first = (warp - 10) * 64;
          uint32_t bad = 0;
#pragma unroll 4
          for (int c = 0; c < 64 * kD * 2 / 512; ++c) {                 // 4 rows of 128 bytes a step
            const uint4 w = *reinterpret_cast<const uint4*>(tile + (c / 16) * kTile * 128 + (first + (c % 16) * 4) * 128 + lane * 16);
            bad |= not_finite<kBf16>(w.x) | not_finite<kBf16>(w.y) | not_finite<kBf16>(w.z) | not_finite<kBf16>(w.w);
          }
          if (__any_sync(0xffffffffu, bad)) {
            for (int c = 0; c < 64 * kD * 2 / 512; ++c) {
              const int row = first + (c % 16) * 4 + lane / 8;
              uint32_t* w = reinterpret_cast<uint32_t*>(tile + (c / 16) * kTile * 128 + (first + (c % 16) * 4) * 128 + lane * 16);
              for (int e = 0; e < 4; ++e) {
                if (!not_finite<kBf16>(w[e])) continue;
                if (j * kTile + row < it.keys) *reinterpret_cast<volatile int*>(&bars.items[slot].flagged) = 1;
                if (not_finite<kBf16>(w[e] & 0xFFFFu)) w[e] &= 0xFFFF0000u;
                if (not_finite<kBf16>(w[e] & 0xFFFF0000u)) w[e] &= 0xFFFFu;
              }
            }
            gemm::fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) gemm::mbar_arrive(&bars.v_ok[edges & 3]);
          ++edges;
        }
        if (!ok) break;
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&bars.item_free[slot]);
        if (it.stop) break;
        kv += 2 * steps;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ---- softmax ----
    const int t = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;        // TMEM lane quarter
    const uint32_t s_tmem = tmem + t * kTile + lanes, o_tmem = tmem + 2 * kTile + t * kD + lanes;
    const int row = t * kTile + (warp & 3) * 32 + lane;                  // row of the block
    const float slack = kSlack / p.scale;
    int s_count = 0, o_count = 0;
    bool ok = true;
    for (int64_t n = 0; ok; ++n) {
      const int slot = static_cast<int>(n % kItemSlots);
      if (!gemm::wait_warp(&bars.item_full[slot], static_cast<uint32_t>((n / kItemSlots) & 1), abort)) break;
      const Item it = bars.items[slot];
      if (it.stop) break;
      const int steps = t == 0 ? it.steps[0] : it.steps[1];
      const int whole = min(it.keys, max(0, it.off + t * kTile + 1));    // keys that the tile's first row sees
      const int64_t sees64 = min(static_cast<int64_t>(it.keys), static_cast<int64_t>(it.off) + row + 1);
      const int sees = static_cast<int>(sees64);                         // keys that this row sees (<= 0: none)
      float m = -INFINITY;                                               // in units of q.k
      float2 l[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      for (int j = 0; j < steps; ++j) {
        if (!(ok = gemm::wait_warp(&bars.s_full[t], s_count & 1, abort))) break;
        ++s_count;
        gemm::tc_fence_after();
        uint32_t raw[kTile / 32][32];
        float s[kTile];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const bool masked = (j + 1) * kTile > whole;
        const int left = sees - j * kTile;                               // keys of this tile that the row sees
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 0) {
            gemm::tmem_ld32(s_tmem, raw[0]);
            gemm::tmem_ld32(s_tmem + 32, raw[1]);
            gemm::tmem_ld_wait(raw[0], raw[1]);
            gemm::tmem_ld32(s_tmem + 64, raw[2]);
            gemm::tmem_ld32(s_tmem + 96, raw[3]);
          } else {
            gemm::tmem_ld_wait(raw[2], raw[3]);
          }
#pragma unroll
          for (int i = h * 64; i < h * 64 + 64; ++i) s[i] = __uint_as_float(raw[i / 32][i % 32]);
          if (masked) {
#pragma unroll
            for (int i = h * 64; i < h * 64 + 64; ++i) s[i] = i < left ? s[i] : -INFINITY;
          }
#pragma unroll
          for (int i = h * 64; i < h * 64 + 64; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) tops[e] = max3_nan(tops[e], s[i + 2 * e], s[i + 2 * e + 1]);
        }
        const float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
        if (__any_sync(0xffffffffu, top > m + slack)) {
          const float now = top > m + slack ? top : m;
          const float keep = m == -INFINITY ? 0.f : ex2((m - now) * p.scale);
          m = now;
          l[0] = __fmul2_rn(l[0], make_float2(keep, keep));
          l[1] = __fmul2_rn(l[1], make_float2(keep, keep));
          if (j > 0) {
#pragma unroll
            for (int c = 0; c < kD / 32; ++c) {
              uint32_t o[32];
              gemm::tmem_ld32(o_tmem + c * 32, o);
              gemm::tmem_ld_wait(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st32(o_tmem + c * 32, o);
            }
          }
        }
        // a NaN or an infinite score makes the row NaN (the polynomial below would lose it)
        if (!(top < INFINITY)) l[0].x = __int_as_float(0x7fc00000);
        // s * scale - m * scale in one rounding; where the second product's own rounding would
        // count (scores beyond 2^16), the difference is taken first
        float base = m == -INFINITY ? 0.f : m * p.scale;
        if (__any_sync(0xffffffffu, fabsf(base) > 65536.f)) {
          const float shift = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int i = 0; i < kTile; ++i) s[i] -= shift;
          base = 0.f;
        }
        const float2 scale2 = make_float2(p.scale, p.scale), base2 = make_float2(-base, -base);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int c = 2 * h; c < 2 * h + 2; ++c) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float2 x = __ffma2_rn(make_float2(s[c * 32 + 2 * i], s[c * 32 + 2 * i + 1]), scale2, base2);
              const float2 e = (i % kPolyEvery) == kPolyEvery - 1 ? ex2_poly<kBf16>(x) : make_float2(ex2(x.x), ex2(x.y));
              l[i & 1] = __fadd2_rn(l[i & 1], e);
              w[i] = pack<kBf16>(e.x, e.y);
            }
            tmem_st16(s_tmem + c * 16, w);
          }
          tmem_st_wait();
          gemm::tc_fence_before();
          __syncwarp();
          if (lane == 0) gemm::mbar_arrive(&bars.p_full[t][h]);
        }
      }
      if (!ok) break;
      // ---- the row's output ----
      const bool mine = row < it.rows;
      uint8_t* dst = p.out + ((static_cast<int64_t>(it.q0) + row) * p.o_token + it.head * p.o_head) * 2;
      const float sum = (l[0].x + l[0].y) + (l[1].x + l[1].y);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (steps > 0) {
        if (!(ok = gemm::wait_warp(&bars.o_full[t], o_count & 1, abort))) break;
        ++o_count;
        gemm::tc_fence_after();
      }
      const bool flagged = steps > 0 && *reinterpret_cast<volatile int*>(&bars.items[slot].flagged) != 0;
#pragma unroll
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t o[32];
        if (steps > 0) {
          gemm::tmem_ld32(o_tmem + c * 32, o);
          gemm::tmem_ld_wait(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (c == kD / 32 - 1 && steps > 0) {
          gemm::tc_fence_before();
          __syncwarp();
          if (lane == 0) gemm::mbar_arrive(&bars.o_free[t]);
        }
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(o[i]) * inv;
        if (flagged && mine) {                           // what the V check set to zero and this row sees
          for (int k = it.edge * kTile; k < sees; ++k) {
            const uint8_t* v = p.v + ((static_cast<int64_t>(it.k0) + k) * p.v_token + (it.head / p.group) * p.v_head + c * 32) * 2;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const uint32_t bits = *reinterpret_cast<const uint16_t*>(v + i * 2);
              if (not_finite<kBf16>(bits))
                f[i] += kBf16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(bits)));
            }
          }
        }
        if (mine) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack<kBf16>(f[2 * i], f[2 * i + 1]);
          if (p.out32) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c * 64 + i * 32),
                           "r"(w[8 * i]), "r"(w[8 * i + 1]), "r"(w[8 * i + 2]), "r"(w[8 * i + 3]), "r"(w[8 * i + 4]),
                           "r"(w[8 * i + 5]), "r"(w[8 * i + 6]), "r"(w[8 * i + 7])
                           : "memory");
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              *reinterpret_cast<uint4*>(dst + c * 64 + i * 16) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) gemm::mbar_arrive(&bars.item_free[slot]);
    }
  }
  gemm::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    gemm::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
  }
}

}  // namespace prompt
}  // namespace isp
