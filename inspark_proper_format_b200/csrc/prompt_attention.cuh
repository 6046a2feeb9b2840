// Attention of packed sequences on the tensor cores (tcgen05), sm_100a.
//
// o_i = sum_j p_ij v_j / sum_j p_ij over the keys j that query i sees, p_ij =
// 2^(scale log2(e) q_i.k_j - m_i), with the running maximum m and sum of each row in FP32,
// one pass over K and V.  p enters the product with V in the operands' type: BF16, or FP16 times
// 2^7, which keeps all its bits down to 2^-21 of a row's largest weight and loses what lies below
// 2^-32 of it (FP16 rows reach from 2^-24 to 2^16).
//
// A work item is a block of 256 queries of one (sequence, head): two tiles of 128 that share
// every K and V tile of 128 keys.  Blocks of the grid are persistent and take items in an
// order of falling block index, back and forth (static, so results and order are fixed).
// Roles of the 12 warps:
//   warps 0-3, 4-7  softmax of tile 0 and 1: a thread owns a row.  It takes the row's 128
//                   scores from TMEM, writes p in 16 bits over them, and at the end scales
//                   and stores the row's output.  m stays up to kSlack behind the maximum,
//                   so that most steps leave the accumulated output alone.
//   warps 8, 11     issue the MMAs of tile 0 and 1: S = Q K^T (both operands in shared memory)
//                   and O += P V (P in TMEM, V's tile read with its keys along K), PV(j - 1)
//                   then S(j).  A warp for each tile: the waits of one warp for both were
//                   the longest chain of the kernel.
//   warp 9          finds the items and loads Q and the ring of K and V tiles by TMA.
//   warp 10         checks the V tiles that hold keys some row must not see.  A product with
//                   p = 0 would turn an infinity or NaN there into NaN, so they are set to
//                   zero in shared memory; values that other rows do see are added to those
//                   rows at the end.
// Every wait is bounded; on expiry the block unwinds as the GEMMs do.
//
// Measured on one B200, launches of a captured graph over changing inputs (and calls among
// others): 16384 tokens, 32 over 8 heads of 128, 2.04 ms (2.10 ms; both at the power cap, 1.08
// PFLOP/s of causal work; a single launch 1.8 to 1.9 ms); 64 x 760 frames, 8 heads of 64, every key,
// 139 us (156 us); 64 x 256 tokens, 20 heads of 64, 56.2 us (57.1 us).  Bound by the chain S ->
// maximum -> exponentials -> PV -> next S of a tile (P lies over S): a step of both tiles of the
// long case takes about 3800 cycles, of them 2048 in the special function unit and as many in the
// tensor pipe, each busy for 0.6 of the time; over the frames they are for 0.52 and 0.32.  Finding
// an item scans the sequences' bounds a few times, which shows from about a thousand short
// sequences on (8192 sequences of 1 to 64 tokens, 8 heads: 11 ms, 512 of them 137 us).
// Tried and slower: half of the exponentials or fewer by polynomial (5 to 25%, the warps are
// bound by their own instruction chains), a second read of S in a rolled loop (15%; for masked
// tiles alone 3 to 7%), two threads a row (5 to 20% on long items), half of S(j + 1) before PV(j),
// P over S all the same (4%), no turns (10 to 18%).  The roles' code has to stay small, they share
// the instruction cache: rolling the output and the repair of non-finite values alone took 3 to
// 8% off, two scores to an instruction (f32x2) in the products and sums of the exponentials
// another 3 to 9%.
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
constexpr int kTmemColumns = 512;
constexpr float kSlack = 8.f;
constexpr int kTurnSteps = 4;               // key tiles from which on the two query tiles take turns
// Registers of a softmax thread and of the other warps' threads.  They draw on the launch's
// 384 x 168; a larger sum would wait for ever, so the host checks the build's count.
constexpr int kSoftmaxRegs = 208, kOtherRegs = 80;
static_assert(2 * 128 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168, "");

template <int kD>
struct Layout {
  static constexpr int kTileBytes = kTile * kD * 2;            // a tile of Q, K or V: kD / 64 boxes of 128 rows x 128 bytes
  static constexpr int kStages = kD == 64 ? 8 : 5;             // K and V tiles in flight
  static constexpr int kQBuffers = kD == 64 ? 2 : 1;           // blocks of Q: the next item's is loaded early where it fits
  static constexpr int kQ = 0;
  static constexpr int kRing = kQBuffers * 2 * kTileBytes;
  static constexpr int kBars = kRing + kStages * kTileBytes;
  static constexpr int kBytes = kBars + 1024;
  // TMEM columns of tile t: S, with P over its first half; O
  static constexpr int s(int t) { return t * kTile; }
  static constexpr int o(int t) { return 2 * kTile + t * kD; }
};

struct Item {
  int stop;              // no more items
  int head;
  int q0, rows;          // first query row, queries of the block
  int k0, keys;          // first key row, keys of the sequence
  int off;               // row r of the block sees the first min(keys, r + off + 1) keys
  int swap;              // query tile t has the block's half t ^ swap
  int steps[2];          // key tiles of each query tile
  int edge;              // first key tile that some row does not see whole
  int flagged;           // the V check found non-finite values in view
  int pad[4];
};

struct Bars {
  uint64_t full[8], empty[8];                        // K and V ring
  uint64_t q_full[2], q_free[2];
  uint64_t s_full[2], p_full[2][2], o_full[2], o_free[2];   // p: keys 0-63, then 64-127
  // V tiles through the check, in order: their loads complete on v_in instead of the ring's
  // barrier (which the producer completes by hand), the check answers on v_ok.  The ring
  // holds at most four V tiles, so neither side is more than these ahead.
  uint64_t v_in[4], v_ok[4];
  uint64_t item_full[kItemSlots], item_free[kItemSlots];
  uint64_t drained;
  Item items[kItemSlots];
  uint32_t turn[2];      // steps whose exponentials a tile has taken, times its four warps
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

// Bounded wait of a converged warp.  It lies on the chain between the softmax and the MMAs,
// so the clock is read only after a while (reading it takes longer than most waits).
ISP_D bool wait_all(uint64_t* bar, uint32_t parity, volatile int* abort) {
#pragma unroll 1
  for (int i = 0; i < 256; ++i)
    if (__all_sync(0xffffffffu, gemm::mbar_try_wait(bar, parity))) return true;
  return gemm::wait_warp(bar, parity, abort);
}

// Wait until a count is reached, or for some time: nothing depends on it but the schedule.
ISP_D void hint_wait(volatile uint32_t* count, uint32_t target) {
#pragma unroll 1
  for (int i = 0; i < 128; ++i)
    if (static_cast<int32_t>(*count - target) >= 0) return;
}

template <bool kBf16>
ISP_D uint32_t pack(float a, float b) {
  return kBf16 ? gemm::pack_bf16(a, b) : gemm::pack_f16(a, b);
}

// ---- 32 of a thread's row of scores ----
ISP_D void hide(uint32_t (&s)[32], int left) {
  const uint32_t seen = left >= 32 ? 0xFFFFFFFFu : (1u << max(left, 0)) - 1u;   // bits turn into predicates in groups
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = (seen >> i) & 1u ? s[i] : 0xFF800000u;
}
ISP_D void take_from(uint32_t (&s)[32], float shift) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float2 d = __fadd2_rn(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), make_float2(-shift, -shift));
    s[i] = __float_as_uint(d.x);
    s[i + 1] = __float_as_uint(d.y);
  }
}
ISP_D void chunk_max(const uint32_t (&s)[32], float (&top)[4]) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
#pragma unroll
    for (int e = 0; e < 4; ++e) top[e] = max3_nan(top[e], __uint_as_float(s[i + 2 * e]), __uint_as_float(s[i + 2 * e + 1]));
}
// 2^(s * scale - base) in 16 bits to TMEM, their sum to l.
template <bool kBf16>
ISP_D void chunk_weights(const uint32_t (&s)[32], float scale, float base, float2 (&l)[2], uint32_t taddr) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])),
                                make_float2(scale, scale), make_float2(-base, -base));
    const float a = ex2(x.x), b = ex2(x.y);
    l[i & 1] = __fadd2_rn(l[i & 1], make_float2(a, b));
    w[i] = pack<kBf16>(a, b);
  }
  tmem_st16(taddr, w);
}

template <bool kBf16>
ISP_D float to_float(uint16_t bits) {
  return kBf16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16) : __half2float(__ushort_as_half(bits));
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
ISP_D void find_item(const Params& p, int64_t x, int top, int swap, int lane, Item& it) {
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
    const int half = t ^ swap;
    const int last = min(it.rows, (half + 1) * kTile) - 1;
    const int seen = it.rows > half * kTile ? min(static_cast<int64_t>(it.keys), static_cast<int64_t>(last) + it.off + 1) : 0;
    it.steps[t] = max(0, (seen + kTile - 1) / kTile);
  }
  it.edge = max(0, min(it.keys, it.off < it.keys ? it.off + 1 : it.keys)) / kTile;
  it.flagged = 0;
  it.swap = swap;
}

// 0 x + z of two 16-bit values each (one instruction for four of a test of the bits: 2.5% of 64 x 256 tokens).
template <bool kBf16>
ISP_D uint32_t times_zero(uint32_t x, uint32_t z) {
  uint32_t r;
  if constexpr (kBf16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(z));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(z));
  return r;
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
      gemm::mbar_init(&bars.empty[i], 2);
    }
    for (int t = 0; t < 2; ++t) {
      gemm::mbar_init(&bars.q_full[t], 1);
      gemm::mbar_init(&bars.q_free[t], 2);
      gemm::mbar_init(&bars.s_full[t], 1);
      gemm::mbar_init(&bars.p_full[t][0], 4);
      gemm::mbar_init(&bars.p_full[t][1], 4);
      gemm::mbar_init(&bars.o_full[t], 1);
      gemm::mbar_init(&bars.o_free[t], 4);
      bars.turn[t] = 0;
    }
    for (int i = 0; i < 4; ++i) {
      gemm::mbar_init(&bars.v_in[i], 1);
      gemm::mbar_init(&bars.v_ok[i], 1);
    }
    for (int i = 0; i < kItemSlots; ++i) {
      gemm::mbar_init(&bars.item_full[i], 1);
      gemm::mbar_init(&bars.item_free[i], 11);
    }
    gemm::mbar_init(&bars.drained, 2);
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
        // The tiles take the halves of a block in alternation: in a causal block the second half
        // has more keys, and in a short one the first is alone (64 x 256 tokens 57 us, with
        // fixed halves 60 us; long items alike).
        if (x < total) find_item(p, x, top, static_cast<int>(n & 1), lane, it);
        if (n >= kItemSlots && !gemm::wait_warp(&bars.item_free[slot], static_cast<uint32_t>((n / kItemSlots - 1) & 1), abort)) break;
        if (lane == 0) {
          bars.items[slot] = it;
          gemm::mbar_arrive(&bars.item_full[slot]);
        }
        __syncwarp();
        if (it.stop) break;
        const int steps = max(it.steps[0], it.steps[1]);
        if (steps == 0) continue;
        const auto load_q = [&]() {
          const int buf = loaded % L::kQBuffers;
          if (loaded >= L::kQBuffers && !gemm::wait_warp(&bars.q_free[buf], (loaded / L::kQBuffers - 1) & 1, abort)) return false;
          ++loaded;
          if (lane == 0) {
            const int tiles = (it.steps[0] > 0) + (it.steps[1] > 0);
            gemm::mbar_expect_tx(&bars.q_full[buf], tiles * L::kTileBytes);
            for (int t = 0; t < 2; ++t) {
              if (it.steps[t] == 0) continue;
              for (int c = 0; c < kD / 64; ++c)
                gemm::tma_load_3d(smem + L::kQ + (buf * 2 + t) * L::kTileBytes + c * kTile * 128, &q_map, &bars.q_full[buf], c * 64,
                                  it.head, it.q0 + (t ^ it.swap) * kTile);
            }
          }
          __syncwarp();
          return true;
        };
        // where Q has one buffer, the first K and V go ahead of it: it is free last
        if (L::kQBuffers == 2 && !(ok = load_q())) break;
        for (int j = 0; j < 2 * steps; ++j, ++kv) {      // K0, V0, K1, V1, ...
          if (L::kQBuffers == 1 && j == 2 && !(ok = load_q())) break;
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
        if (L::kQBuffers == 1 && ok && steps == 1) ok = load_q();
      }
      // loads in flight land before the block ends
      if (*abort) {
        for (int i = 0; i < L::kQBuffers; ++i)
          if (loaded > i) gemm::wait_warp_drain(&bars.q_full[i], ((loaded - 1 - i) / L::kQBuffers) & 1);
        for (int i = 0; i < L::kStages; ++i)
          if (kv > static_cast<uint32_t>(i))               // (kv - 1 - i) / kStages: fills of stage i so far, minus one
            gemm::wait_warp_drain(&bars.full[i], ((kv - 1 - i) / L::kStages) & 1);
        for (int i = 0; i < 4; ++i)
          if (edges > static_cast<uint32_t>(i)) gemm::wait_warp_drain(&bars.v_in[i], ((edges - 1 - i) / 4) & 1);
      }
    } else if (warp != 10) {
      // ---- MMAs of tile t ----
      const int t = warp == 8 ? 0 : 1;
      const uint32_t s_desc = idesc(kBf16, kTile, false), o_desc = idesc(kBf16, kD, true);
      const uint32_t ring = gemm::smem_u32(smem + L::kRing);
      const uint32_t s_tmem = tmem + L::s(t), o_tmem = tmem + L::o(t);
      uint64_t q = 0;
      uint32_t stage = 0, phase = 0;                     // of the ring's next tile
      uint32_t loaded = 0, edges = 0, count = 0, o_count = 0;
      bool ok = true;
      const auto next = [&]() {
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1;
        }
      };
      const auto scores = [&](uint32_t k_stage) {
        gemm::tc_fence_after();
        const uint64_t k = gemm::smem_desc_sw128(ring + k_stage * L::kTileBytes);
#pragma unroll
        for (int i = 0; i < kD / 16; ++i) {              // 16 head dimensions: 32 bytes of a row
          const int o = ((i / 4) * kTile * 128 + (i % 4) * 32) >> 4;
          mma_ss(s_tmem, q + o, k + o, s_desc, i > 0);
        }
        gemm::mma_commit_elect<false>(&bars.s_full[t]);
      };
      // Give a tile or Q back after the MMAs issued, or at once (the fill was waited for, so the
      // two warps' arrivals belong to one fill).
      const auto release = [&](uint64_t* bar, bool used) {
        if (used) gemm::mma_commit_elect<false>(bar);
        else if (lane == 0) gemm::mbar_arrive(bar);
        __syncwarp();
      };
      for (uint32_t n = 0; ok; ++n) {
        const uint32_t slot = n % kItemSlots;
        if (!wait_all(&bars.item_full[slot], (n / kItemSlots) & 1, abort)) break;
        const int stop = bars.items[slot].stop, edge = bars.items[slot].edge, mine = bars.items[slot].steps[t];
        const int steps = max(mine, bars.items[slot].steps[t ^ 1]);
        __syncwarp();
        if (lane == 0) gemm::mbar_arrive(&bars.item_free[slot]);
        if (stop) break;
        if (steps == 0) continue;
        const uint32_t q_buf = loaded % L::kQBuffers;
        if (!(ok = wait_all(&bars.q_full[q_buf], (loaded / L::kQBuffers) & 1, abort))) break;
        ++loaded;
        q = gemm::smem_desc_sw128(gemm::smem_u32(smem + L::kQ) + (q_buf * 2 + t) * L::kTileBytes);
        if (!(ok = wait_all(&bars.full[stage], phase, abort))) break;
        if (mine > 0) scores(stage);                     // S(0)
        release(&bars.empty[stage], mine > 0);
        if (mine <= 1) release(&bars.q_free[q_buf], mine == 1);
        next();
        for (int j = 0; j < steps; ++j) {
          const uint32_t v_stage = stage, v_phase = phase;             // V_j, then K_(j + 1)
          next();
          const uint32_t k_stage = stage;
          if (j + 1 < steps) {
            if (!(ok = wait_all(&bars.full[stage], phase, abort))) break;
            next();
          }
          if (j >= edge) {
            if (!(ok = wait_all(&bars.v_ok[edges & 3], (edges >> 2) & 1, abort))) break;
            ++edges;
          } else if (!(ok = wait_all(&bars.full[v_stage], v_phase, abort))) {
            break;
          }
          if (j < mine) {
            if (j == 0 && o_count++ > 0 && !(ok = wait_all(&bars.o_free[t], o_count & 1, abort))) break;
            const uint64_t v = v_desc(ring + v_stage * L::kTileBytes);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (!(ok = wait_all(&bars.p_full[t][half], count & 1, abort))) break;
              gemm::tc_fence_after();
#pragma unroll
              for (int i = 0; i < kTile / 32; ++i) {     // 16 keys: 8 columns of P, 2048 bytes of V
                const int k = half * (kTile / 32) + i;
                mma_ts(o_tmem, s_tmem + k * 8, v + ((k * 2048) >> 4), o_desc, j > 0 || k > 0);
              }
            }
            if (!ok) break;
            ++count;
            if (j + 1 == mine) gemm::mma_commit_elect<false>(&bars.o_full[t]);
            else scores(k_stage);                        // over P, in order behind the products that read it
          }
          release(&bars.empty[v_stage], j < mine);
          if (j + 1 < steps) {
            release(&bars.empty[k_stage], j + 1 < mine);
            if (j + 2 == mine) release(&bars.q_free[q_buf], true);
          }
        }
      }
      // the MMAs issued end before TMEM is freed
      gemm::mma_commit_elect<false>(&bars.drained);
      gemm::wait_warp_drain(&bars.drained, 0);
    } else {
      // ---- V check ----
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
          uint32_t zero[4] = {0u, 0u, 0u, 0u};           // sums of 0 x: 0, or NaN for an infinity or NaN
#pragma unroll 8
          for (int c = 0; c < L::kTileBytes / 512; ++c) {                // 4 rows of 128 bytes a step
            const uint4 w = *reinterpret_cast<const uint4*>(tile + c * 512 + lane * 16);
            zero[0] = times_zero<kBf16>(w.x, zero[0]);
            zero[1] = times_zero<kBf16>(w.y, zero[1]);
            zero[2] = times_zero<kBf16>(w.z, zero[2]);
            zero[3] = times_zero<kBf16>(w.w, zero[3]);
          }
          const bool bad = not_finite<kBf16>(zero[0]) || not_finite<kBf16>(zero[1]) || not_finite<kBf16>(zero[2]) ||
                           not_finite<kBf16>(zero[3]);
          if (__any_sync(0xffffffffu, bad)) {
            for (int c = 0; c < L::kTileBytes / 512; ++c) {
              const int row = (c % 32) * 4 + lane / 8;
              uint32_t* w = reinterpret_cast<uint32_t*>(tile + c * 512 + lane * 16);
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
    const uint32_t s_tmem = tmem + L::s(t) + lanes, o_tmem = tmem + L::o(t) + lanes;
    const float slack = kSlack / p.scale;
    constexpr float kPlace = kBf16 ? 0.f : 15.f - kSlack;                // FP16 weights as high as FP16 allows
    uint32_t s_count = 0, o_count = 0, turns = 0;                        // turns: of the other tile, in the items before
    bool ok = true;
    for (uint32_t n = 0; ok; ++n) {
      const uint32_t slot = n % kItemSlots;
      if (!wait_all(&bars.item_full[slot], (n / kItemSlots) & 1, abort)) break;
      const Item& it = bars.items[slot];
      if (it.stop) break;
      const int steps = it.steps[t], steps_other = it.steps[t ^ 1];
      const int first = (t ^ it.swap) * kTile, row = first + (warp & 3) * 32 + lane;   // rows of the block
      // keys that this row, and the tile's first row, see (<= 0: none)
      const int sees = static_cast<int>(min(static_cast<int64_t>(it.keys), static_cast<int64_t>(it.off) + row + 1));
      const int whole = min(it.keys, it.off + first + 1);
      const bool take_turns = min(steps, steps_other) >= kTurnSteps;
      float m = -INFINITY, shift = 0.f, base = -kPlace;                      // m in units of q.k
      bool far = false;
      float2 l[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      for (int j = 0; j < steps; ++j) {
        if (!(ok = wait_all(&bars.s_full[t], s_count & 1, abort))) break;
        ++s_count;
        gemm::tc_fence_after();
        const bool masked = (j + 1) * kTile > whole;
        const int left = sees - j * kTile;                               // keys of this tile that the row sees
        uint32_t x[4][32];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        gemm::tmem_ld32(s_tmem, x[0]);
        gemm::tmem_ld32(s_tmem + 32, x[1]);
        gemm::tmem_ld_wait(x[0], x[1]);
        gemm::tmem_ld32(s_tmem + 64, x[2]);
        gemm::tmem_ld32(s_tmem + 96, x[3]);
        if (masked) hide(x[0], left), hide(x[1], left - 32);
        chunk_max(x[0], tops);
        chunk_max(x[1], tops);
        gemm::tmem_ld_wait(x[2], x[3]);
        if (masked) hide(x[2], left - 64), hide(x[3], left - 96);
        chunk_max(x[2], tops);
        chunk_max(x[3], tops);
        const float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
        if (__any_sync(0xffffffffu, top > m + slack)) {
          const float now = top > m + slack ? top : m;
          const float keep = m == -INFINITY ? 0.f : ex2((m - now) * p.scale);
          m = now;
          l[0] = __fmul2_rn(l[0], make_float2(keep, keep));
          l[1] = __fmul2_rn(l[1], make_float2(keep, keep));
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < kD / 32; ++c) {
              uint32_t o[32];
              gemm::tmem_ld32(o_tmem + c * 32, o);
              gemm::tmem_ld_wait(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st32(o_tmem + c * 32, o);
            }
          }
          // s * scale - m * scale in one rounding; where the second product's own rounding would
          // count (scores beyond 2^16), the difference is taken first
          shift = m == -INFINITY ? 0.f : m;
          far = __any_sync(0xffffffffu, fabsf(shift * p.scale) > 65536.f);
          base = (far ? 0.f : shift * p.scale) - kPlace;
        }
        if (far) {
#pragma unroll
          for (int c = 0; c < 4; ++c) take_from(x[c], shift);
        }
        // In long items the tiles take their exponentials in turn, tile 0 of step j, tile 1, tile
        // 0 of step j + 1: side by side they would share the special function unit and then both
        // wait for the MMAs.  Only a hint: whoever has waited long goes on.
        if (take_turns && j > 0)
          hint_wait(&bars.turn[t ^ 1], 4 * (turns + min(t == 0 ? j : j + 1, steps_other)));
#pragma unroll
        for (int c = 0; c < 4; ++c) {                                    // p replaces the scores
          chunk_weights<kBf16>(x[c], p.scale, base, l, s_tmem + c * 16);
          if (c == 2 && lane == 0) atomicAdd(&bars.turn[t], 1u);     // the last quarter may overlap
          __syncwarp();
          if (c >= 2) {                                                  // half a tile, a chunk later
            tmem_st_wait();
            gemm::tc_fence_before();
            __syncwarp();
            if (lane == 0) gemm::mbar_arrive(&bars.p_full[t][c - 2]);
            __syncwarp();
          }
        }
        if (!(top < INFINITY)) l[0].x = __int_as_float(0x7fc00000);      // a NaN or an infinite score: the row is NaN
      }
      if (!ok) break;
      turns += steps_other;
      // ---- the row's output ----
      const bool mine = row < it.rows;
      uint8_t* dst = p.out + ((static_cast<int64_t>(it.q0) + row) * p.o_token + it.head * p.o_head) * 2;
      const float sum = (l[0].x + l[0].y) + (l[1].x + l[1].y);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (steps > 0) {
        if (!(ok = wait_all(&bars.o_full[t], o_count & 1, abort))) break;
        ++o_count;
        gemm::tc_fence_after();
      }
#pragma unroll 1
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t o[32];
        if (steps > 0) {
          gemm::tmem_ld32(o_tmem + c * 32, o);
          gemm::tmem_ld_wait(o);
          if (c == kD / 32 - 1) {
            gemm::tc_fence_before();
            __syncwarp();
            if (lane == 0) gemm::mbar_arrive(&bars.o_free[t]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (mine) {
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack<kBf16>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
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
        __syncwarp();                                                    // the next read of TMEM is the whole warp's
      }
      if (steps > 0 && mine && *reinterpret_cast<const volatile int*>(&it.flagged) != 0) {
        // what the V check set to zero and this row sees: infinities and NaN, which take the element over
        const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v) + (it.head / p.group) * p.v_head;
        uint16_t* out = reinterpret_cast<uint16_t*>(dst);
#pragma unroll 1
        for (int k = it.edge * kTile; k < sees; ++k)
#pragma unroll 1
          for (int i = 0; i < kD; ++i) {
            const uint16_t bits = v[(static_cast<int64_t>(it.k0) + k) * p.v_token + i];
            if (!not_finite<kBf16>(bits)) continue;
            const uint32_t sum = pack<kBf16>(to_float<kBf16>(out[i]) + to_float<kBf16>(bits), 0.f);
            out[i] = static_cast<uint16_t>(sum);
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
