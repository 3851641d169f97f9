// Attention's backward pass on the tensor cores, recomputing the probabilities from the row
// statistics that the forward kept (attention.cu, the lse output):
//   P_ij = exp(c q_i . k_j - lse_i)      delta_i = dO_i . O_i       dP_ij = dO_i . v_j
//   dS_ij = P_ij (dP_ij - delta_i)
//   dV_j = sum_i P_ij dO_i     dK_j = c sum_i dS_ij q_i     dQ_i = c sum_j dS_ij k_j
// over the visible pairs (key_lo[b] <= j < key_hi[b] and, when causal, j <= i + Sk - Sq), dK and dV
// summed over the query heads of a key head.
//
// One launch of two kinds of CTA (twelve warps), neither of which adds to memory atomically, so that
// equal calls give equal bits:
//   key CTAs    own 128 keys of one key head and walk the query tiles of its heads:
//               S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q;
//   query CTAs  own 128 queries of one head and walk the key tiles:
//               S = Q K^T, dP = dO V^T, dQ += dS K.
// Forming S and dP twice costs 7 products instead of 5, and saves the fp32 dQ that would have to be
// added up in memory in a fixed order. P and dS are the first operands of their products straight from
// TMEM (over the columns of the S and dP they came from, where there is no room beside them), so shared memory
// holds operand tiles only (three Q and two dO stages, or three K and two V stages, beside the resident pair).
// Columns that a product reads are taken by the next S or dP once a commit has told that it has run: only MMAs
// of the same accumulator and shape are promised to run in the order they are issued.
//
// What bounds it, at head dimension 128: a key CTA's pair of tiles is a chain, S -> P (1100 cycles, of
// which the special-function unit's 1024) -> dV -> next S (1024 of tensor work), about 2700 cycles with
// the hand-overs for 2048 of tensor work, and the commits that tell of dV and dK on top (3 to 11 % of this kernel's
// time); dS, dK and the next dP run beside it. A query CTA's pair takes about 2500 for 1536: P and dS in turn in
// the same warps. TMEM (512 columns: S, dP, dV, dK, or two S, dP, dQ) leaves no second buffer to break the chains.
// A Llama-3-70B-shaped layer (4096 tokens, 64 and 8 heads, causal): 0.87 ms, 790 TFLOP/s of the five products, 1110
// of the seven; one of 2048 tokens with 32 and 8 heads: 0.132 ms. Over seconds the GPU's 1000 W set the pace.
#include <atomic>
#include <cfloat>

#include "attention_common.cuh"

namespace muzo {
namespace {

using namespace tc;
using namespace attn;

constexpr int B_THREADS = 384;   // warp 0 TMA, warp 1 MMA, warp 2 waits for a key CTA's loads, warps 4..11
                                 // probabilities: two groups of four, one warp of each per TMEM lane quarter
constexpr uint32_t B_TMEM_COLS = 512;
constexpr float kLog2e = 1.4426950408889634f;

template <int D>
struct BwdLayout {
  static constexpr int NKB = D / ABK;
  static constexpr int TILE_BYTES = NKB * SUB_BYTES;   // 128 rows of one operand
  static constexpr int TILES = 7;                      // key CTA: K, V, 3 Q, 2 dO; query CTA: Q, dO, 3 K, 2 V
  static constexpr int STAT_BYTES = 5 * 512;           // key CTA: -delta with each Q stage, -lse with each dO stage
  static constexpr int BAR_BYTES = 256;
  static constexpr int NEED = TILES * TILE_BYTES + STAT_BYTES + BAR_BYTES;
  static constexpr int SMEM_BYTES = NEED > 116 * 1024 ? NEED : 116 * 1024;   // one CTA per SM: it takes all of TMEM
};

struct BwdArgs {
  int64_t sq, sk, shift;
  int batch, hq, hkv, group, nqt, nkt, causal, hd, parts;
  int64_t key_items, query_items;
  float scale, scale_log2;
  const int32_t* key_lo;
  const int32_t* key_hi;
  const float* stats;    // [B * Hq][nqt][2][128]: -lse in log2 units (fp16: plus 10; -inf: no key seen, or no such
                         // row), -delta
  const uint32_t* largest;  // fp16: the bits of the largest |dO_i|^2 of rows that see a key and, of visible keys, |v_j|^2
  float* partial;        // [parts][B * Hkv][nkt * 128][2][D] sums of dV and c dK, or null when parts == 1
  uint16_t *dq, *dk, *dv;   // any may be null
  int64_t dq_sb, dq_sh, dq_ss, dk_sb, dk_sh, dk_ss, dv_sb, dv_sh, dv_ss;
  int32_t* status;
};

// D = A B with A from TMEM (128 lanes, 8 columns of packed 16-bit pairs per K = 16) and B from shared memory.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// `bytes` (a multiple of 16) of contiguous global memory into shared memory, counted on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int FMT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  return FMT == 1 ? pack_bf16(lo, hi) : pack_half(lo, hi);
}

// Bounded waits of one thread and of a warp (one lane polls, all get its answer). A phase that is
// complete costs one poll; the abort flag and the clock are read between polls only. The waits on the
// path between the tensor cores and the probabilities poll with test_wait: a thread that try_wait
// has suspended wakes 250 to 650 cycles after the phase, in one of eight warps or the other.
__device__ __forceinline__ bool poll(uint32_t addr, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(addr), "r"(parity)
      : "memory");
  return done != 0;
}
template <bool SPIN = true>
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, const int* abort_flag) {
  const uint32_t addr = smem_u32(bar);
  if (SPIN ? poll(addr, parity) : mbar_try_wait(addr, parity)) return true;
  const long long start = clock64();
  while (!(SPIN ? poll(addr, parity) : mbar_try_wait(addr, parity))) {
    if (*reinterpret_cast<const volatile int*>(abort_flag)) return false;
    if (static_cast<unsigned long long>(clock64() - start) > kWaitLimitCycles) return false;
  }
  return true;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const int* abort_flag) {
  bool ready = true;
  if ((threadIdx.x & 31) == 0) ready = wait_one(bar, parity, abort_flag);
  __syncwarp();
  return __shfl_sync(0xffffffffu, ready ? 1 : 0, 0) != 0;
}

// Query tiles [first, first + count) that see a key of key tile kt in batch row b.
__device__ __forceinline__ void key_tile_queries(const BwdArgs& g, int b, int kt, int64_t& lo, int64_t& hi, int& first,
                                                 int& count) {
  key_range(g.key_lo, g.key_hi, g.sk, b, lo, hi);
  first = 0;
  count = 0;
  const int64_t key0 = static_cast<int64_t>(kt) * AN;
  const int64_t a = key0 > lo ? key0 : lo;                        // first and last visible key of the tile
  const int64_t z = key0 + AN < hi ? key0 + AN : hi;
  if (a >= z) return;
  if (g.causal) {
    const int64_t q = a - g.shift;                                // the first query that sees key a
    if (q >= g.sq) return;
    first = q > 0 ? static_cast<int>(q / AM) : 0;
  }
  count = g.nqt - first;
}

// Key tiles [first, first + count) that query tile qt of batch row b sees.
__device__ __forceinline__ void query_tile_keys(const BwdArgs& g, int b, int qt, int64_t& lo, int64_t& hi, int& first,
                                                int& count) {
  key_range(g.key_lo, g.key_hi, g.sk, b, lo, hi);
  int64_t end = hi;
  if (g.causal) {
    const int64_t q = static_cast<int64_t>(qt) * AM + AM - 1;
    const int64_t last = (q < g.sq - 1 ? q : g.sq - 1) + g.shift + 1;
    if (last < end) end = last;
  }
  first = static_cast<int>(lo / AN);
  count = end > lo ? static_cast<int>((end + AN - 1) / AN) - first : 0;
}

// Rows of an accumulator to global memory, one warp: this thread's row of 128 bytes (`w`, 8 pieces of 16)
// goes through 4 KB of shared memory, so that 8 lanes write one row's 128 bytes (a thread that wrote its
// own row touched 32 rows with every instruction: 8000 cycles for a key CTA's 64 KB). `dst` is the
// warp's first row at the first of these columns, `pitch` the bytes between rows; `rows` rows and
// `pieces` pieces of each exist.
__device__ __forceinline__ void store_rows(uint8_t* stage, const uint4 (&w)[8], uint8_t* dst, int64_t pitch, int64_t rows,
                                           int pieces) {
  const int lane = threadIdx.x & 31;
  __syncwarp();   // the last call's reads are done
#pragma unroll
  for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = w[c];
  __syncwarp();
  const int c = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = 4 * i + (lane >> 3);
    const uint4 x = *reinterpret_cast<const uint4*>(stage + row * 128 + ((c ^ (row & 7)) << 4));
    if (row < rows && c < pieces) *reinterpret_cast<uint4*>(dst + row * pitch + 16 * c) = x;
  }
}

// 64 accumulator columns times f as 16-bit values, 32 as fp32.
template <int FMT>
__device__ __forceinline__ void pack_row(const uint32_t (&v)[64], float f, uint4 (&w)[8]) {
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    uint32_t x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = pack16<FMT>(__uint_as_float(v[8 * c + 2 * e]) * f, __uint_as_float(v[8 * c + 2 * e + 1]) * f);
    w[c] = make_uint4(x[0], x[1], x[2], x[3]);
  }
}
__device__ __forceinline__ void scale_row(const uint32_t (&v)[32], float f, uint4 (&w)[8]) {
#pragma unroll
  for (int c = 0; c < 8; ++c)
    w[c] = make_uint4(__float_as_uint(__uint_as_float(v[4 * c]) * f), __float_as_uint(__uint_as_float(v[4 * c + 1]) * f),
                      __float_as_uint(__uint_as_float(v[4 * c + 2]) * f), __float_as_uint(__uint_as_float(v[4 * c + 3]) * f));
}

// Barriers of both kinds of CTA. Every arrival that an issuer commits to is waited for before the CTA ends (a
// stage that no later tile takes is not released): two commits behind the same product have no stated order,
// and one that came after the other's waiters had left would write to shared memory that is another's.
enum : int {
  kFull = 0,        // key CTA: K, V, Q[3], dO[2]; query CTA: Q, dO, K[3], V[2]
  kEmpty = 7,       // key CTA: Q[3], dO[2] (at 2 and 5); query CTA: K[3], V[2] (at 2 and 5)
  kS = 14,          // S computed (query CTA: two, by buffer)
  kDp = 16,         // dP computed
  kP = 17,          // key CTA: P written, S read, by halves of each warp's columns; with the second half, the
                    // next tile's loads are here. Query CTA, the first: dP read
  kDs = 19,         // dS written, and in a key CTA dP read (query CTA: two, by buffer: its readers run apart)
  kDone = 21,
  kDrain = 22,
  kStall = 23,
  kOrder = 24,      // two: a product has read its A operand from TMEM, and the next S or dP may take the columns
  kBars = 26
};

// Loads issued by the producer thread: which full barriers are armed, and with which parity.
struct Armed {
  uint32_t mask = 0, parity = 0;
  __device__ __forceinline__ void arm(uint64_t* bars, int i, uint32_t phase, uint32_t bytes) {
    mbar_arrive_expect_tx(bars + kFull + i, bytes);
    mask |= 1u << i;
    parity = (parity & ~(1u << i)) | (phase << i);
  }
  __device__ __forceinline__ void wait_all(uint64_t* bars) const {
    for (int i = 0; i < 7; ++i)
      if (mask & (1u << i)) mbar_wait(bars + kFull + i, (parity >> i) & 1u);
  }
};

template <int NKB>
__device__ __forceinline__ void load_tile(const CUtensorMap* map, uint64_t* bar, uint8_t* dst, int row, int h, int b) {
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb) tma_load_4d(map, bar, dst + kb * SUB_BYTES, kb * ABK, row, h, b);
}

// D (128 x 128) = A B^T, both operands K-major tiles of D columns in shared memory.
template <int NKB>
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, const uint8_t* a, const uint8_t* b, uint32_t idesc) {
  const uint32_t sa = smem_u32(a), sb = smem_u32(b);
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
    for (int k = 0; k < ABK / 16; ++k)
      umma_f16(tmem_d, make_sdesc(sa + kb * SUB_BYTES + k * 32, 16, 1024), make_sdesc(sb + kb * SUB_BYTES + k * 32, 16, 1024),
               idesc, (kb > 0 || k > 0) ? 1u : 0u);
}

// D (128 x NKB*64) (+)= A B: A packed in TMEM (K rows 0..63 in columns 0..31, K rows 64..127 from column
// `second` on), B a tile of 128 rows in shared memory read MN-major. `part` 0 takes the K rows 0..31
// and 64..95, 1 the others, 2 all.
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, const uint8_t* b, uint32_t idesc, bool accumulate,
                                       int second, int part = 2) {
  const uint32_t sb = smem_u32(b);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if (part == 1 - ((k >> 1) & 1)) continue;
    umma_f16_ts(tmem_d, tmem_a + (k < 4 ? 8 * k : second + 8 * (k - 4)), make_sdesc(sb + k * (16 * 128), SUB_BYTES, 1024), idesc,
                (accumulate || k > (part == 1 ? 2 : 0) || part == 1) ? 1u : 0u);
  }
}

// The kernel may start while the one that writes the statistics still runs (programmatic launch): who
// reads them waits for its end first.
__device__ __forceinline__ void wait_for_statistics() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// TMEM loads and stores are instructions of a whole converged warp: each stands behind a __syncwarp, since a
// lane may have polled or arrived alone before it.

// What a role that gave up does: the first code stays in the status word.
__device__ __forceinline__ void give_up(const BwdArgs& g, int* abort_flag, int code) {
  atomicCAS(g.status, kErrNone, code);
  atomicExch(abort_flag, 1);
}

// What a CTA that gave up leaves, so that nobody takes old memory or half a sum for gradients: NaN in all of its
// rows, or in its part of the sums, which the join passes on.
template <int D>
__device__ __forceinline__ void lose_rows(const BwdArgs& g, bool key_cta, int kt, int bh, int b, int qt) {
  if (!key_cta) {
    lose_tile(g.dq + b * g.dq_sb + (bh % g.hq) * g.dq_sh, g.dq_ss, static_cast<int64_t>(qt) * AM, AM, g.sq, g.hd);
  } else if (g.parts > 1) {
    const int64_t part = blockIdx.x % static_cast<unsigned>(g.parts);
    float* sums = g.partial + ((part * g.batch * g.hkv + bh) * g.nkt + kt) * AN * 2 * D;
    for (int i = threadIdx.x; i < AN * 2 * D; i += B_THREADS) sums[i] = __int_as_float(0x7fffffff);
  } else {
    const int64_t key0 = static_cast<int64_t>(kt) * AN;
    if (g.dk != nullptr) lose_tile(g.dk + b * g.dk_sb + (bh % g.hkv) * g.dk_sh, g.dk_ss, key0, AN, g.sk, g.hd);
    if (g.dv != nullptr) lose_tile(g.dv + b * g.dv_sb + (bh % g.hkv) * g.dv_sh, g.dv_ss, key0, AN, g.sk, g.hd);
  }
}

// Powers of two that P and dS carry on their way through 16 bits. bf16 has fp32's range and needs none.
// In fp16 a probability below 2^-14 would lose bits, and dS, a probability times a gradient, most of them
// (or overflow): P is taken 2^10-fold, and dS times the largest 2^k that keeps |dS| <= 2 max|dO_i| max|v_j|
// (|delta| <= |dO_i| max|v_j|: O is a mean of the v_j) at or below 2^15. The products' results are divided
// again in fp32.
struct Powers {
  float ds = 1.0f;          // factor of dP and delta: 2^(k - 10)
  float dv = 1.0f, dqk = 1.0f;   // 2^-10 and 2^-k
};
template <int FMT>
__device__ __forceinline__ Powers powers_of(const BwdArgs& g) {
  Powers p;
  if (FMT == 0) {
    wait_for_statistics();
    const float a = __uint_as_float(g.largest[0]), b = __uint_as_float(g.largest[1]);
    const float bound = 2.0f * sqrtf(a) * sqrtf(b);
    int k = 0;
    if (bound > 0.0f && bound < INFINITY) {
      int e;
      frexpf(bound, &e);      // bound < 2^e
      k = 15 - e;
      k = k < -24 ? -24 : (k > 40 ? 40 : k);
    }
    p.ds = ldexpf(1.0f, k - 10);
    p.dv = 1.0f / 1024.0f;
    p.dqk = ldexpf(1.0f, -k);
  }
  return p;
}

template <int FMT, int D>
__global__ void __launch_bounds__(B_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, BwdArgs g) {
  using L = BwdLayout<D>;
  constexpr int NKB = L::NKB;
  constexpr int TILE = L::TILE_BYTES;
  extern __shared__ __align__(1024) uint8_t smem[];   // 1024: the swizzled tiles' alignment
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::TILES * TILE + L::STAT_BYTES);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(bars + kBars);
  int* abort_flag = reinterpret_cast<int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stall = *reinterpret_cast<volatile int*>(g.status + 1);
  const bool key_cta = static_cast<int64_t>(blockIdx.x) < g.key_items;

  if (threadIdx.x == 0) {
    // One thread initialises every barrier, and no load is issued before the CTA's barrier below. (Loads issued 2 to 4
    // us earlier, behind barriers that a lane each had initialised, were part of a form whose launches faulted now and
    // then; what made them fault was not shown.)
    // arrivals: the eight probability warps on kP and kDs, the warp that waits for a key CTA's loads on its second
    // kP
    for (int i = 0; i < kBars; ++i) mbar_init(bars + i, i == kP + 1 ? 9 : (i >= kP && i < kDone ? 8 : 1));
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(B_TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // The CTA's work
  Armed armed;
  int kt = 0, qt_own = 0, b, bh_own, first, count, begin = 0, n;
  int64_t lo, hi;
  if (key_cta) {
    const unsigned per_tile = static_cast<unsigned>(g.batch * g.hkv * g.parts);
    kt = static_cast<int>(blockIdx.x / per_tile);   // causal: the first key tiles see the most queries
    const unsigned rest = blockIdx.x % per_tile;
    const int part = static_cast<int>(rest % g.parts);
    bh_own = static_cast<int>(rest / g.parts);
    b = bh_own / g.hkv;
    key_tile_queries(g, b, kt, lo, hi, first, count);
    // this CTA's share of the (head, query tile) pairs
    const int total = g.group * count;
    const int chunk = (total + g.parts - 1) / g.parts;
    begin = part * chunk < total ? part * chunk : total;
    n = (begin + chunk < total ? begin + chunk : total) - begin;
  } else {
    const unsigned item = blockIdx.x - static_cast<unsigned>(g.key_items);
    const unsigned bh_count = static_cast<unsigned>(g.batch * g.hq);
    qt_own = g.nqt - 1 - static_cast<int>(item / bh_count);   // causal: the last query tiles see the most keys
    bh_own = static_cast<int>(item % bh_count);
    b = bh_own / g.hq;
    query_tile_keys(g, b, qt_own, lo, hi, first, n);
    count = n;
  }
  // A key CTA's tile t: one Q stage with -delta, one dO stage with -lse, as the buffers below are laid out.
  auto load_query_tile = [&](int t, bool q_part, uint32_t phase) {
    const int pair = begin + t, head = (bh_own % g.hkv) * g.group + pair / count, qt = first + pair % count;
    const float* st = g.stats + ((static_cast<int64_t>(b) * g.hq + head) * g.nqt + qt) * 256;
    float* stat_base = reinterpret_cast<float*>(smem + L::TILES * TILE);   // -delta [3][128], -lse [2][128]
    const int s = q_part ? t % 3 : t & 1, bar = (q_part ? 2 : 5) + s;
    armed.arm(bars, bar, phase, TILE + 512);
    load_tile<NKB>(q_part ? &map_q : &map_do, bars + kFull + bar, smem + bar * TILE, qt * AM, head, b);
    if (t == 0) wait_for_statistics();
    bulk_load(stat_base + (q_part ? s : 3 + s) * 128, q_part ? st + 128 : st, 512, bars + kFull + bar);
  };
  // A query CTA's key tile t: a K or a V stage.
  auto load_key_tile = [&](int t, bool k_part, uint32_t phase) {
    const int bar = k_part ? 2 + t % 3 : 5 + (t & 1);
    armed.arm(bars, bar, phase, TILE);
    load_tile<NKB>(k_part ? &map_k : &map_v, bars + kFull + bar, smem + bar * TILE, (first + t) * AN,
                   (bh_own % g.hq) / g.group, b);
  };
  auto load_own = [&](const CUtensorMap* map, int bar, int row, int head) {
    armed.arm(bars, bar, 0, TILE);
    load_tile<NKB>(map, bars + kFull + bar, smem + bar * TILE, row, head, b);
  };
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns: they begin at 0. (An address that says otherwise is reported, and the CTA does nothing.)
  constexpr uint32_t tmem = 0;
  const bool tmem_ok = *reinterpret_cast<volatile uint32_t*>(tmem_holder) == tmem;
  if (!tmem_ok) {
    give_up(g, abort_flag, kErrTimeoutMma);
    n = 0;
  }
  if (threadIdx.x == 0 && n > 0) {
    if (key_cta) {
      load_own(&map_k, 0, kt * AN, bh_own % g.hkv);
      load_query_tile(0, true, 0);
      load_own(&map_v, 1, kt * AN, bh_own % g.hkv);
      load_query_tile(0, false, 0);
    } else {
      load_own(&map_q, 0, qt_own * AM, bh_own % g.hq);
      load_key_tile(0, true, 0);
      load_own(&map_do, 1, qt_own * AM, bh_own % g.hq);
      load_key_tile(0, false, 0);
    }
  }
  if (warp == 3) wait_for_statistics();   // in CTAs that read none too: this launch ends after the one it may overlap
  constexpr uint32_t idesc_s = make_idesc_fmt(128, 128, false, false, FMT);   // S, dP: both operands K-major
  constexpr uint32_t idesc_g = make_idesc_fmt(128, D, false, true, FMT);      // gradients: B MN-major
  const int quarter = warp & 3, half = (warp - 4) >> 2;
  const int r = 32 * quarter + lane;                                          // row of the tile == TMEM lane
  const uint32_t lane_addr = static_cast<uint32_t>(32 * quarter) << 16;

  if (key_cta) {
    // ================================================================ 128 keys: dK, dV
    const int bh = bh_own, kvh = bh % g.hkv;
    const int part = static_cast<int>(blockIdx.x % static_cast<unsigned>(g.parts));
    uint8_t* sK = smem;
    uint8_t* sV = smem + TILE;
    uint8_t* sQ = smem + 2 * TILE;        // 3 stages
    uint8_t* sO = smem + 5 * TILE;        // 2 stages
    float* neg_delta = reinterpret_cast<float*>(smem + L::TILES * TILE);   // [3][128], with Q
    float* neg_lse = neg_delta + 3 * 128;                                  // [2][128], with dO
    // Tiles of 64 columns leave room for P and dS beside S and dP. Those of 128 do not: P and dS lie over the first
    // halves of the columns that their warps read, and the next S and dP, which overwrite them, have to wait until
    // dV and dK have read them: MMAs of different accumulators or shapes have no promised order.
    constexpr bool kOwn = D == 64;
    constexpr int kSecond = kOwn ? 32 : 64;   // columns from the first 64 K rows to the others
    const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = t_dv + D;
    const uint32_t t_p = kOwn ? tmem + 384 : t_s, t_ds = kOwn ? tmem + 448 : t_dp;
    // The first rows of a head's first tile may see no key (left padding under causality, more queries than keys).
    // Their P and dS are 0, but 0 times a non-finite dO or Q would still reach dV and dK: warp 2 clears those rows
    // before the products.
    const int64_t blind = g.causal ? lo - g.shift - static_cast<int64_t>(first) * AM : 0;
    const int blind_rows = n > 0 && blind > 0 ? static_cast<int>(blind) : 0;   // fewer than a tile's: `first` sees a key

    if (warp == 0) {
      if (lane == 0 && n > 0) {
        bool ok = stall != kErrTimeoutProducer || mbar_wait(bars + kStall, 0, kStallLimitCycles);
        for (int t = 1; t < n && ok; ++t) {   // a Q stage is free after its dK, a dO stage after its dV (issued behind dP)
          const int sq = t % 3, so = t & 1;
          const uint32_t pq = (t / 3) & 1, po = (t >> 1) & 1;
          ok = wait_one<false>(bars + kEmpty + 2 + sq, pq ^ 1, abort_flag);
          if (ok) load_query_tile(t, true, pq);
          ok = ok && wait_one<false>(bars + kEmpty + 5 + so, po ^ 1, abort_flag);
          if (ok) load_query_tile(t, false, po);
        }
        if (!ok) give_up(g, abort_flag, kErrTimeoutProducer);
        armed.wait_all(bars);   // every load of this CTA has landed before it may exit (bounded)
      }
      __syncwarp();
    } else if (warp == 1) {
      if (n > 0 && elect_one()) {
        auto ready = [&](int bar, uint32_t parity) -> bool {
          if (!wait_one(bars + bar, parity, abort_flag)) return false;
          tc_fence_after();
          return true;
        };
        auto read_by_now = [&](int which, int t) -> bool {   // what has been issued has run
          umma_commit(bars + kOrder + which);
          return ready(kOrder + which, t & 1);
        };
        bool ok = stall != kErrTimeoutMma || mbar_wait(bars + kStall, 0, kStallLimitCycles);
        ok = ok && ready(kFull, 0) && ready(kFull + 2, 0);
        if (ok) {
          mma_ss<NKB>(t_s, sK, sQ, idesc_s);
          umma_commit(bars + kS);
          ok = ready(kFull + 1, 0) && ready(kFull + 5, 0);
        }
        if (ok) {
          mma_ss<NKB>(t_dp, sV, sO, idesc_s);
          umma_commit(bars + kDp);
        }
        for (int t = 0, pos = begin % count; t < n && ok; ++t, pos = pos + 1 < count ? pos + 1 : 0) {
          const int so = t & 1;
          // P(t) written, S(t) read, the next Q and dO loaded and rows cleared (warp 2 arrives for them): dV, then
          // the next S
          if (blind_rows > 0 && pos == 0 && !ready(kP + 1, t & 1)) { ok = false; break; }
          if (!ready(kP, t & 1)) { ok = false; break; }
          mma_ts(t_dv, t_p, sO + so * TILE, idesc_g, t > 0, kSecond, 0);
          if (!ready(kP + 1, t & 1)) { ok = false; break; }
          mma_ts(t_dv, t_p, sO + so * TILE, idesc_g, true, kSecond, 1);
          if (t + 2 < n) umma_commit(bars + kEmpty + 5 + so);
          if (t + 1 < n) {
            if (!kOwn && !read_by_now(0, t)) { ok = false; break; }
            mma_ss<NKB>(t_s, sK, sQ + ((t + 1) % 3) * TILE, idesc_s);
            umma_commit(bars + kS);
          }
          if (!ready(kDs, t & 1)) { ok = false; break; }
          mma_ts(t_dk, t_ds, sQ + (t % 3) * TILE, idesc_g, t > 0, kSecond);
          if (t + 3 < n) umma_commit(bars + kEmpty + 2 + t % 3);
          if (t + 1 < n) {
            if (!kOwn && !read_by_now(1, t)) { ok = false; break; }
            mma_ss<NKB>(t_dp, sV, sO + (so ^ 1) * TILE, idesc_s);
            umma_commit(bars + kDp);
          }
        }
        if (ok) umma_commit(bars + kDone);
        else give_up(g, abort_flag, kErrTimeoutMma);
      }
      __syncwarp();
    } else if (warp == 2) {
      // Waits for the loads in the issuer's place: its polls queue behind the MMAs it has issued (150 to
      // 270 cycles each, with the tensor cores idle), so it is left with two per tile. And clears the rows of Q and dO
      // that see no key.
      bool ok = true;
      for (int t = 0, pos = n > 0 ? begin % count : 0; t < n && ok; ++t, pos = pos + 1 < count ? pos + 1 : 0) {
        if (lane == 0 && t > 0) ok = wait_one<false>(bars + kP + 1, (t - 1) & 1, abort_flag);
        if (blind_rows > 0 && pos == 0) {
          if (lane == 0) ok = ok && wait_one<false>(bars + kDp, t & 1, abort_flag);   // S(t) and dP(t) have read them
          if (__shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0) {
            uint8_t *q_rows = sQ + (t % 3) * TILE, *o_rows = sO + (t & 1) * TILE;   // contiguous in each block of 64 columns
            for (int i = lane; i < 8 * blind_rows; i += 32)
#pragma unroll
              for (int kb = 0; kb < NKB; ++kb) {
                *reinterpret_cast<uint4*>(q_rows + kb * SUB_BYTES + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
                *reinterpret_cast<uint4*>(o_rows + kb * SUB_BYTES + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
              }
            fence_proxy_async_smem();
          }
          __syncwarp();
        }
        if (lane == 0) {
          if (ok && t + 1 < n)
            ok = wait_one<false>(bars + kFull + 2 + (t + 1) % 3, ((t + 1) / 3) & 1, abort_flag) &&
                 wait_one<false>(bars + kFull + 5 + ((t + 1) & 1), ((t + 1) >> 1) & 1, abort_flag);
          if (ok) mbar_arrive(bars + kP + 1);
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      }
      if (!ok && lane == 0) give_up(g, abort_flag, kErrTimeoutMma);
      __syncwarp();
    } else if (warp >= 4) {
      const Powers two = n > 0 ? powers_of<FMT>(g) : Powers();
      const int64_t key = static_cast<int64_t>(kt) * AN + r;
      const bool key_seen = key >= lo && key < hi;
      bool ok = true;
      if (stall == kErrTimeoutEpilogue) {
        bool waited = true;
        if (lane == 0) waited = mbar_wait(bars + kStall, 0, kStallLimitCycles);
        ok = __shfl_sync(0xffffffffu, waited ? 1 : 0, 0) != 0;
      }
      for (int t = 0; t < n && ok; ++t) {
        const int sq = t % 3, so = t & 1;
        const int qt = first + (begin + t) % count;
        // first of this warp's 64 columns whose query sees the key
        int c_lo = 64;
        if (key_seen) {
          const int64_t c = g.causal ? key - g.shift - static_cast<int64_t>(qt) * AM - 64 * half : 0;
          c_lo = c < 0 ? 0 : (c > 64 ? 64 : static_cast<int>(c));
        }
        const bool all_seen = __all_sync(0xffffffffu, c_lo == 0);
        // the statistics came with Q and dO: their readers wait for those barriers too
        if (!warp_wait(bars + kFull + 5 + so, (t >> 1) & 1, abort_flag) ||
            !warp_wait(bars + kFull + 2 + sq, (t / 3) & 1, abort_flag) || !warp_wait(bars + kS, t & 1, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const float4* nl = reinterpret_cast<const float4*>(neg_lse + so * 128 + half * 64);
        const float4* dl = reinterpret_cast<const float4*>(neg_delta + sq * 128 + half * 64);
        float p[64];
        {
          uint32_t v[64];
          __syncwarp();
          tmem_ld64(t_s + lane_addr + half * 64, v);
          // P by halves, so that dV begins while the second half's exponentials run
#pragma unroll
          for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int c = 32 * part; c < 32 * part + 32; c += 4) {
              const float4 m = nl[c >> 2];
#pragma unroll
              for (int e = 0; e < 4; ++e) p[c + e] = __uint_as_float(v[c + e]);
              fma_pair(p[c], p[c + 1], g.scale_log2, m.x, m.y);
              fma_pair(p[c + 2], p[c + 3], g.scale_log2, m.z, m.w);
#pragma unroll
              for (int e = 0; e < 4; ++e) p[c + e] = fast_exp2(p[c + e]);
            }
            if (!all_seen) {
#pragma unroll
              for (int c = 32 * part; c < 32 * part + 32; ++c) p[c] = c >= c_lo ? p[c] : 0.0f;
            }
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 16; ++c) w[c] = pack16<FMT>(p[32 * part + 2 * c], p[32 * part + 2 * c + 1]);
            __syncwarp();
            tmem_st16(t_p + lane_addr + half * kSecond + 16 * part, w);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kP + part);
          }
        }
        if (!warp_wait(bars + kDp, t & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        uint32_t w[32];
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          uint32_t v[32];
          __syncwarp();
          tmem_ld32(t_dp + lane_addr + half * 64 + ch * 32, v);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 m = dl[(ch * 32 + c) >> 2];
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[c + e]);
            add_pair(x[0], x[1], m.x, m.y);
            add_pair(x[2], x[3], m.z, m.w);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              if (FMT == 0) mul_pair(x[e], x[e + 1], two.ds, two.ds);
              mul_pair(p[ch * 32 + c + e], p[ch * 32 + c + e + 1], x[e], x[e + 1]);
            }
          }
        }
        if (!all_seen) {   // a masked pair's dP may be anything (a key's V outside its range)
#pragma unroll
          for (int c = 0; c < 64; ++c) p[c] = c >= c_lo ? p[c] : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) w[c] = pack16<FMT>(p[2 * c], p[2 * c + 1]);
        __syncwarp();
        tmem_st32(t_ds + lane_addr + half * kSecond, w);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kDs);
      }
      if (ok && n > 0) {
        ok = warp_wait(bars + kDone, 0, abort_flag);
        tc_fence_after();
      }
      if (!ok) {
        if (lane == 0) give_up(g, abort_flag, kErrTimeoutEpilogue);
      } else if (g.parts == 1 || n > 0) {
        // the first four warps write dV, the others c dK, 32 keys each; the operand stages are free now
        const uint32_t acc = (half == 0 ? t_dv : t_dk) + lane_addr;
        const float f = half == 0 ? two.dv : g.scale * two.dqk;
        uint8_t* stage = smem + 2 * TILE + (warp - 4) * 4096;
        const int64_t key0 = static_cast<int64_t>(kt) * AN + 32 * quarter;
        if (g.parts > 1) {
          uint8_t* sum = reinterpret_cast<uint8_t*>(
              g.partial + (((static_cast<int64_t>(part) * g.batch * g.hkv + bh) * g.nkt * AN + key0) * 2 + half) * D);
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[32];
            uint4 w[8];
            __syncwarp();
            tmem_ld32(acc + c * 32, v);
            scale_row(v, f, w);
            store_rows(stage, w, sum + c * 128, 2 * D * 4, 32, 8);
          }
        } else {
          uint16_t* out = half == 0 ? g.dv : g.dk;
          if (out != nullptr) {
            const int64_t ss = half == 0 ? g.dv_ss : g.dk_ss;
            out += half == 0 ? b * g.dv_sb + kvh * g.dv_sh + key0 * ss : b * g.dk_sb + kvh * g.dk_sh + key0 * ss;
#pragma unroll 1
            for (int c = 0; c < D / 64; ++c) {
              uint4 w[8];
              if (n > 0) {
                uint32_t v[64];
                __syncwarp();
                tmem_ld64(acc + c * 64, v);
                pack_row<FMT>(v, f, w);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = make_uint4(0u, 0u, 0u, 0u);
              }
              store_rows(stage, w, reinterpret_cast<uint8_t*>(out + c * 64), ss * 2, g.sk - key0, (g.hd - c * 64) / 8);
            }
          }
        }
      }
    }
  } else {
    // ================================================================ 128 queries: dQ
    const int qt = qt_own, h = bh_own % g.hq, kvh = h / g.group;
    const int64_t bh = bh_own;
    uint8_t* sQ = smem;
    uint8_t* sO = smem + TILE;
    uint8_t* sK = smem + 2 * TILE;    // 3 stages
    uint8_t* sV = smem + 5 * TILE;    // 2 stages
    const uint32_t t_s = tmem, t_dp = tmem + 256, t_dq = tmem + 384;   // two S buffers

    if (warp == 0) {
      if (lane == 0 && n > 0) {
        bool ok = stall != kErrTimeoutProducer || mbar_wait(bars + kStall, 0, kStallLimitCycles);
        for (int t = 1; t < n && ok; ++t) {
          const uint32_t pk = (t / 3) & 1, pv = (t >> 1) & 1;
          ok = wait_one<false>(bars + kEmpty + 2 + t % 3, pk ^ 1, abort_flag);
          if (ok) load_key_tile(t, true, pk);
          ok = ok && wait_one<false>(bars + kEmpty + 5 + (t & 1), pv ^ 1, abort_flag);
          if (ok) load_key_tile(t, false, pv);
        }
        if (!ok) give_up(g, abort_flag, kErrTimeoutProducer);
        armed.wait_all(bars);
      }
      __syncwarp();
    } else if (warp == 1) {
      // One issuer, as in a key CTA. (A second warp for the dP products and polls ahead of time in the probability
      // warps made a long backward pass 4 % faster. Only grids with query CTAs are known to have faulted, rarely and
      // from a cause that was not shown, and these were what query CTAs had beside a key CTA's parts.)
      if (n > 0 && elect_one()) {
        auto ready = [&](int bar, uint32_t parity) -> bool {
          if (!wait_one(bars + bar, parity, abort_flag)) return false;
          tc_fence_after();
          return true;
        };
        auto issue_s = [&](int t) {
          mma_ss<NKB>(t_s + 128 * (t & 1), sQ, sK + (t % 3) * TILE, idesc_s);
          umma_commit(bars + kS + (t & 1));
        };
        auto issue_dp = [&](int t) {
          mma_ss<NKB>(t_dp, sO, sV + (t & 1) * TILE, idesc_s);
          umma_commit(bars + kDp);
          if (t + 2 < n) umma_commit(bars + kEmpty + 5 + (t & 1));
        };
        bool ok = stall != kErrTimeoutMma || mbar_wait(bars + kStall, 0, kStallLimitCycles);
        ok = ok && ready(kFull, 0) && ready(kFull + 2, 0);
        if (ok) issue_s(0);
        ok = ok && ready(kFull + 1, 0) && ready(kFull + 5, 0);
        if (ok) issue_dp(0);
        if (ok && n > 1) {
          ok = ready(kFull + 3, 0);
          if (ok) issue_s(1);
        }
        for (int t = 0; t < n && ok; ++t) {
          if (t + 1 < n) {   // dP(t) read: the next one
            if (!ready(kFull + 5 + ((t + 1) & 1), ((t + 1) >> 1) & 1) || !ready(kP, t & 1)) { ok = false; break; }
            issue_dp(t + 1);
          }
          if (!ready(kDs + (t & 1), (t >> 1) & 1)) { ok = false; break; }
          mma_ts(t_dq, t_s + 128 * (t & 1), sK + (t % 3) * TILE, idesc_g, t > 0, 64);
          if (t + 3 < n) umma_commit(bars + kEmpty + 2 + t % 3);
          if (t + 2 < n) {   // S(t+2) over dS(t), once dQ has read it: no order of MMAs is promised
            umma_commit(bars + kOrder);
            if (!ready(kOrder, t & 1) || !ready(kFull + 2 + (t + 2) % 3, ((t + 2) / 3) & 1)) { ok = false; break; }
            issue_s(t + 2);
          }
        }
        if (ok) umma_commit(bars + kDone);
        else give_up(g, abort_flag, kErrTimeoutMma);
      }
      __syncwarp();
    } else if (warp >= 4) {
      const int64_t row = static_cast<int64_t>(qt) * AM + r;
      const bool row_in = row < g.sq;
      const float* st = g.stats + (bh * g.nqt + qt) * 256;
      wait_for_statistics();
      const Powers two = n > 0 ? powers_of<FMT>(g) : Powers();
      const float nl = n > 0 ? st[r] : 0.0f, nd = n > 0 ? st[128 + r] * two.ds : 0.0f;
      int64_t end = hi;                                      // visible keys of this row: [lo, end)
      if (g.causal && row + g.shift + 1 < end) end = row + g.shift + 1;
      if (!row_in) end = lo;
      bool ok = true;
      if (stall == kErrTimeoutEpilogue) {
        bool waited = true;
        if (lane == 0) waited = mbar_wait(bars + kStall, 0, kStallLimitCycles);
        ok = __shfl_sync(0xffffffffu, waited ? 1 : 0, 0) != 0;
      }
      for (int t = 0; t < n && ok; ++t) {
        const int64_t key0 = static_cast<int64_t>(first + t) * AN;
        const int64_t a0 = lo - key0 - 64 * half, a1 = end - key0 - 64 * half;
        const int c_lo = a0 < 0 ? 0 : (a0 > 64 ? 64 : static_cast<int>(a0));
        const int c_hi = a1 < 0 ? 0 : (a1 > 64 ? 64 : static_cast<int>(a1));
        const bool all_seen = __all_sync(0xffffffffu, c_lo == 0 && c_hi == 64);
        const uint32_t my_s = t_s + 128 * (t & 1) + lane_addr + half * 64;
        if (!warp_wait(bars + kS + (t & 1), (t >> 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        float p[64];
        {
          uint32_t v[64];
          __syncwarp();
          tmem_ld64(my_s, v);
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            p[c] = __uint_as_float(v[c]);
            p[c + 1] = __uint_as_float(v[c + 1]);
            fma_pair(p[c], p[c + 1], g.scale_log2, nl, nl);
            p[c] = fast_exp2(p[c]);
            p[c + 1] = fast_exp2(p[c + 1]);
          }
        }
        if (!warp_wait(bars + kDp, t & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        {
          uint32_t v[64];
          __syncwarp();
          tmem_ld64(t_dp + lane_addr + half * 64, v);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + kP);   // dP(t) read: the next one may be formed
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            float x0 = __uint_as_float(v[c]), x1 = __uint_as_float(v[c + 1]);
            if (FMT == 1) add_pair(x0, x1, nd, nd);
            else fma_pair(x0, x1, two.ds, nd, nd);
            mul_pair(p[c], p[c + 1], x0, x1);
          }
        }
        if (!all_seen) {   // a masked pair's dP may be anything (V of a key outside the range)
#pragma unroll
          for (int c = 0; c < 64; ++c) p[c] = c >= c_lo && c < c_hi ? p[c] : 0.0f;
        }
        uint32_t w[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) w[c] = pack16<FMT>(p[2 * c], p[2 * c + 1]);
        __syncwarp();
        tmem_st32(my_s, w);
        // keys outside [lo, hi) beside visible ones: their dS is 0, but 0 times a non-finite key would
        // still reach dQ, so their K rows (S(t) has read them) are cleared
        if (half == 0 && (lo > key0 || hi < (g.sk < key0 + AN ? g.sk : key0 + AN)) && (key0 + r < lo || key0 + r >= hi)) {
          uint8_t* krow = sK + (t % 3) * TILE + r * 128;
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int e = 0; e < 8; ++e) *reinterpret_cast<uint4*>(krow + kb * SUB_BYTES + 16 * e) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + kDs + (t & 1));
      }
      if (ok && n > 0) {
        ok = warp_wait(bars + kDone, 0, abort_flag);
        tc_fence_after();
      }
      if (!ok) {
        if (lane == 0) give_up(g, abort_flag, kErrTimeoutEpilogue);
      } else {
        // 32 rows and, of 128 columns, one half per warp; of 64, the first four warps' all
        if (D == 128 || half == 0) {
          const int col0 = D == 128 ? 64 * half : 0;
          const int64_t row0 = static_cast<int64_t>(qt) * AM + 32 * quarter;
          uint4 w[8];
          if (n > 0) {
            uint32_t v[64];
            __syncwarp();
            tmem_ld64(t_dq + lane_addr + col0, v);
            pack_row<FMT>(v, g.scale * two.dqk, w);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = make_uint4(0u, 0u, 0u, 0u);
          }
          store_rows(smem + 2 * TILE + (warp - 4) * 4096, w,
                     reinterpret_cast<uint8_t*>(g.dq + b * g.dq_sb + h * g.dq_sh + row0 * g.dq_ss + col0), g.dq_ss * 2,
                     g.sq - row0, (g.hd - col0) / 8);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*reinterpret_cast<volatile int*>(abort_flag)) {   // every role has ended: the same answer in all threads
    // the MMAs that an aborted CTA issued end before its TMEM is released (bounded), and the arrivals of commits that
    // nobody waits for any more, which have no stated order, get 50 us
    if (warp == 1 && elect_one()) {
      umma_commit(bars + kDrain);
      mbar_wait(bars + kDrain, 0);
      mbar_wait(bars + kStall, 0, kSettleCycles);
    }
    __syncthreads();
    lose_rows<D>(g, key_cta, kt, bh_own, b, qt_own);
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*reinterpret_cast<volatile uint32_t*>(tmem_holder)), "r"(B_TMEM_COLS) : "memory");
  }
}

// The largest of the block's values (not negative, or NaN) into *word, as its bits.
__device__ __forceinline__ void block_largest(float v, uint32_t* word) {
  __shared__ uint32_t most;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
  if ((threadIdx.x & 31) == 0) atomicMax(&most, w);
  __syncthreads();
  if (threadIdx.x == 0) atomicMax(word, most);   // the largest is the same in whatever order
}

// The larger of two values, NaN if either is.
__device__ __forceinline__ float larger(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int s = 8; s > 0; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s, 16);
  return v;
}

constexpr int kStatThreads = 512, kStatGroups = kStatThreads / 16;

struct Rows16 {   // a [B][H][S][D] operand of 16-bit elements
  const uint16_t* p;
  int64_t sb, sh, ss;
};

// Per query row: -lse in log2 units (with the power of two that P carries; -inf for a row that sees no
// key, so that its probabilities are 0) and -delta = -dO . O, in tiles of 128 rows padded with such rows: one
// block per tile, 16 lanes per row (8 elements each), four rows per lane with their loads in flight
// together. O is what the caller has, 16 bits: its rounding leaves an error of dO . (half a step of O) in delta, which
// dP - delta does not outgrow where P is close to one-hot. For fp16 also the largest |dO_i|^2 of the rows that see a key and, in the blocks behind the query
// tiles', the largest |v_j|^2 of the keys inside their range.
template <int FMT>
__global__ void __launch_bounds__(kStatThreads, 2)
attn_bwd_stats_kernel(Rows16 o, Rows16 d, Rows16 v, const float* lse, float* stats, uint32_t* largest, int hq, int64_t sq,
                      int nqt, int hd, unsigned query_tiles, int hkv, int64_t sk, int nkt, const int32_t* key_lo,
                      const int32_t* key_hi) {
  constexpr int type = FMT == 1 ? MUZO_BF16 : MUZO_F16;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int l = threadIdx.x & 15, group = threadIdx.x >> 4;
  const bool here = 8 * l < hd;
  float square = 0.0f;
  if (FMT == 0 && blockIdx.x >= query_tiles) {
    const unsigned t = blockIdx.x - query_tiles;
    const int bh = static_cast<int>(t / nkt), kt = static_cast<int>(t % nkt), b = bh / hkv;
    int64_t lo, hi;
    key_range(key_lo, key_hi, sk, b, lo, hi);
    const uint16_t* base = v.p + b * v.sb + (bh % hkv) * v.sh + (here ? 8 * l : 0);
    float x[AM / kStatGroups][8];
#pragma unroll
    for (int r = 0; r < AM / kStatGroups; ++r) {
      const int64_t j = static_cast<int64_t>(kt) * AN + kStatGroups * r + group;
      load8(base, (j < sk ? j : sk - 1) * v.ss, type, x[r]);
    }
#pragma unroll
    for (int r = 0; r < AM / kStatGroups; ++r) {
      const int64_t j = static_cast<int64_t>(kt) * AN + kStatGroups * r + group;
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x[r][e], x[r][e], s);
      square = larger(square, sum16(here && j >= lo && j < hi ? s : 0.0f));
    }
    block_largest(square, largest + 1);
    return;
  }
  const int bh = static_cast<int>(blockIdx.x / nqt), qt = static_cast<int>(blockIdx.x % nqt), b = bh / hq, h = bh % hq;
  const int64_t col = here ? 8 * l : 0;
  const uint16_t* ob = o.p + b * o.sb + h * o.sh + col;
  const uint16_t* db = d.p + b * d.sb + h * d.sh + col;
  float* tile = stats + static_cast<int64_t>(blockIdx.x) * 256;
  constexpr int R = AM / kStatGroups;
  // every load is issued before the first is used (lanes and rows that do not exist read one that does)
  float x[R][8], y[R][8], w[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = static_cast<int64_t>(qt) * AM + kStatGroups * r + group;
    const int64_t at = i < sq ? i : sq - 1;
    load8(ob, at * o.ss, type, x[r]);
    load8(db, at * d.ss, type, y[r]);
    w[r] = l == 0 && i < sq ? lse[static_cast<int64_t>(bh) * sq + i] : -INFINITY;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = kStatGroups * r + group;
    const bool in = static_cast<int64_t>(qt) * AM + row < sq;
    float sum = 0.0f, s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum = fmaf(x[r][e], y[r][e], sum);
      if (FMT == 0) s = fmaf(y[r][e], y[r][e], s);
    }
    sum = sum16(here && in ? sum : 0.0f);
    if (FMT == 0) {   // a row that sees no key may hold anything
      const bool seen = __shfl_sync(0xffffffffu, w[r], 0, 16) != -INFINITY;
      square = larger(square, sum16(here && in && seen ? s : 0.0f));
    }
    if (l == 0) {
      tile[row] = w[r] == -INFINITY ? -INFINITY : fmaf(-w[r], kLog2e, FMT == 0 ? 10.0f : 0.0f);   // fp16: 2^10 P
      tile[128 + row] = -sum;
    }
  }
  if (FMT == 0) block_largest(square, largest);
}

// dK, dV of every key: the sums of its tile's parts, in order.
template <int FMT>
__global__ void __launch_bounds__(256) attn_bwd_join_kernel(BwdArgs g, int dpad) {
  const int per_row = 2 * dpad / 8;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t keys = static_cast<int64_t>(g.batch) * g.hkv * g.sk;
  if (idx >= keys * per_row) return;
  const int64_t row = idx / per_row;
  const int e = static_cast<int>(idx % per_row);
  const int which = e >= per_row / 2, c = (e % (per_row / 2)) * 8;
  const int bh = static_cast<int>(row / g.sk);
  const int64_t key = row % g.sk;
  const int b = bh / g.hkv, kvh = bh % g.hkv;
  uint16_t* out = which ? g.dk : g.dv;
  if (out == nullptr || c >= g.hd) return;
  int64_t lo, hi;
  int first, count;
  key_tile_queries(g, b, static_cast<int>(key / AN), lo, hi, first, count);
  const int total = g.group * count;
  const int chunk = (total + g.parts - 1) / g.parts;
  const int used = chunk > 0 ? (total + chunk - 1) / chunk : 0;
  float v[8] = {};
  for (int p = 0; p < used; ++p) {
    const float4* src = reinterpret_cast<const float4*>(
        g.partial + (((static_cast<int64_t>(p) * g.batch * g.hkv + bh) * g.nkt * AN + key) * 2 + which) * dpad + c);
    const float4 x = src[0], y = src[1];
    v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
    v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
  }
  const int64_t at = which ? b * g.dk_sb + kvh * g.dk_sh + key * g.dk_ss : b * g.dv_sb + kvh * g.dv_sh + key * g.dv_ss;
  *reinterpret_cast<uint4*>(out + at + c) = make_uint4(pack16<FMT>(v[0], v[1]), pack16<FMT>(v[2], v[3]),
                                                       pack16<FMT>(v[4], v[5]), pack16<FMT>(v[6], v[7]));
}

template <int FMT, int D>
int launch_bwd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& md,
               const BwdArgs& g, cudaStream_t s) {
  auto kern = attn_bwd_kernel<FMT, D>;
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  MUZO_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return MUZO_ERR_UNSUPPORTED;
  if (!configured[dev].load(std::memory_order_acquire)) {
    MUZO_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, BwdLayout<D>::SMEM_BYTES));
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(g.key_items + g.query_items));
  cfg.blockDim = dim3(B_THREADS);
  cfg.dynamicSmemBytes = BwdLayout<D>::SMEM_BYTES;
  cfg.stream = s;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  // Early only where all CTAs fit at once: 15.5 -> 11.9 us for 27 of them when it came. With 640, launched early, the
  // short query CTAs ran before the long key CTAs instead of beside them: 152 against 124 us (32 and 8 heads,
  // 2048 tokens). Without a pair no statistics kernel precedes this one.
  cfg.numAttrs = g.nqt > 0 && g.nkt > 0 && g.key_items + g.query_items <= 148 ? 1 : 0;
  MUZO_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, mq, mk, mv, md, g));
  count_launches(1);
  int st = launch_status();
  if (st != MUZO_OK || g.parts == 1 || g.key_items == 0) return st;
  const int64_t threads = static_cast<int64_t>(g.batch) * g.hkv * g.sk * (2 * D / 8);   // key_items <= 2^31: fewer than 2^40
  attn_bwd_join_kernel<FMT><<<static_cast<unsigned>((threads + 255) / 256), 256, 0, s>>>(g, D);
  count_launches(1);
  return launch_status();
}

// Parts that the (head, query tile) pairs of a key tile are divided into, of four pairs at least: the
// fewest with which the longest key CTA does not outlast the average SM by more than 15 % (a division
// costs the sums' way through memory and a launch). In units of one pair of a key CTA, a pair of a query
// CTA takes 0.85 and a CTA's start and end 2.5 (2800, 2400 and 7000 cycles); causal CTAs start longest
// first, and the short query CTAs fill what is left. Measured (before the commits of kOrder), us for 1 / 2 / 3 / 4 / 8 parts: 32 query
// and 8 key heads, 2048 tokens 125 / 146 / 157 / 167 / 198; 8 and 1 heads, 2048 tokens 226 / 122 / 88 /
// 71 / 45; 8 and 1 heads, 16384 tokens 1783 / 1476 / 1583 / 1569 / 1491.
int64_t key_parts(int64_t batch, int64_t hkv, int64_t group, int64_t nqt, int64_t nkt, bool causal, bool queries) {
  const double sms = 148.0, query_step = 0.85, cta = 2.5;
  const int64_t pairs = group * nqt;
  if (batch <= 0 || nkt <= 0 || pairs <= 1) return 1;
  double tiles = static_cast<double>(nqt) * static_cast<double>(nkt);   // visible tile pairs of a head
  if (causal) {
    const double m = static_cast<double>(nqt < nkt ? nqt : nkt);
    tiles = nqt <= nkt ? tiles - m * (m - 1) / 2 : m * (m + 1) / 2;
  }
  const double heads = static_cast<double>(batch) * static_cast<double>(hkv * group);
  const double items = static_cast<double>(batch) * static_cast<double>(hkv) * static_cast<double>(nkt);
  const double steps = heads * tiles * (queries ? 1.0 + query_step : 1.0) + (queries ? heads * nqt * cta : 0.0);
  const int64_t most = pairs / 4 < 32 ? pairs / 4 : 32;
  for (int64_t parts = 1; parts < most; ++parts)
    if (static_cast<double>((pairs + parts - 1) / parts) + cta <= 1.15 * (steps + items * parts * cta) / sms) return parts;
  return most > 1 ? most : 1;
}

int64_t stats_bytes(int64_t batch, int64_t hq, int64_t nqt) { return batch * hq * nqt * 1024; }

int bwd_shape(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t sq, int64_t sk, int64_t hd) {
  if (batch < 0 || hq <= 0 || hkv <= 0 || hq % hkv != 0 || sq < 0 || sk < 0) return MUZO_ERR_ARG;
  if (dtype != MUZO_BF16 && dtype != MUZO_F16) return MUZO_ERR_DTYPE;
  if (hd < 8 || hd % 8 != 0 || hd > 128) return MUZO_ERR_UNSUPPORTED;
  if (batch > 0x7fffffffLL || hq > 0x7fffffffLL || sq > 0x7fffff00LL || sk > 0x7fffff00LL) return MUZO_ERR_UNSUPPORTED;
  return MUZO_OK;
}

}  // namespace
}  // namespace muzo

using namespace muzo;

extern "C" {

int64_t muzo_attention_backward_workspace(int dtype, int64_t batch, int64_t hq, int64_t hkv, int64_t seq_q, int64_t seq_k,
                                          int64_t head_dim, int causal) {
  if (bwd_shape(dtype, batch, hq, hkv, seq_q, seq_k, head_dim) != MUZO_OK) return -1;
  const int64_t nqt = (seq_q + AM - 1) / AM, nkt = (seq_k + AN - 1) / AN;
  // without dQ the key tiles are divided into at least as many parts as with it
  const int64_t parts = key_parts(batch, hkv, hq / hkv, nqt, nkt, causal != 0, false);
  const int64_t sums = parts > 1 ? parts * batch * hkv * nkt * AN * 2 * (head_dim <= 64 ? 64 : 128) * 4 : 0;
  return stats_bytes(batch, hq, nqt) + sums + 16;
}

int muzo_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* dout,
                            const float* lse, void* dq, void* dk, void* dv, int dtype, int64_t batch, int64_t hq,
                            int64_t hkv, int64_t seq_q, int64_t seq_k, int64_t head_dim, const int64_t* strides,
                            int causal, float scale, const int32_t* d_key_lo, const int32_t* d_key_hi,
                            void* d_workspace, int64_t workspace_bytes, int32_t* d_status, void* stream) {
  int st = bwd_shape(dtype, batch, hq, hkv, seq_q, seq_k, head_dim);
  if (st != MUZO_OK) return st;
  if (strides == nullptr || d_status == nullptr || !(scale > 0.0f && scale <= FLT_MAX)) return MUZO_ERR_ARG;
  if (batch == 0 || (seq_q == 0 && seq_k == 0)) return MUZO_OK;
  const bool none = seq_q == 0 || seq_k == 0;   // no pair: the gradients that exist are zero
  if (!none && (q == nullptr || k == nullptr || v == nullptr || out == nullptr || dout == nullptr || lse == nullptr ||
                d_workspace == nullptr))
    return MUZO_ERR_ARG;
  for (int i = 0; i < 24; ++i)
    if (strides[i] % 8 != 0) return MUZO_ERR_ALIGN;
  const void* bases[8] = {q, k, v, out, dout, dq, dk, dv};
  for (const void* p : bases)
    if (!aligned16p(p)) return MUZO_ERR_ALIGN;
  if (!none && !aligned16p(d_workspace)) return MUZO_ERR_ALIGN;
  if (!none && workspace_bytes < muzo_attention_backward_workspace(dtype, batch, hq, hkv, seq_q, seq_k, head_dim, causal))
    return MUZO_ERR_CAPACITY;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  BwdArgs g = {};
  g.sq = seq_q; g.sk = seq_k; g.shift = seq_k - seq_q;
  g.batch = static_cast<int>(batch); g.hq = static_cast<int>(hq); g.hkv = static_cast<int>(hkv);
  g.group = static_cast<int>(hq / hkv); g.hd = static_cast<int>(head_dim); g.causal = causal ? 1 : 0;
  g.nqt = static_cast<int>((seq_q + AM - 1) / AM);
  g.nkt = static_cast<int>((seq_k + AN - 1) / AN);
  g.parts = static_cast<int>(key_parts(batch, hkv, g.group, g.nqt, g.nkt, causal != 0, dq != nullptr));
  g.scale = scale; g.scale_log2 = scale * kLog2e;
  g.key_lo = d_key_lo; g.key_hi = d_key_hi;
  g.dq = static_cast<uint16_t*>(dq); g.dk = static_cast<uint16_t*>(dk); g.dv = static_cast<uint16_t*>(dv);
  const int64_t* t = strides + 15;
  g.dq_sb = t[0]; g.dq_sh = t[1]; g.dq_ss = t[2];
  g.dk_sb = t[3]; g.dk_sh = t[4]; g.dk_ss = t[5];
  g.dv_sb = t[6]; g.dv_sh = t[7]; g.dv_ss = t[8];
  g.status = d_status;
  if (none) g.parts = 1;
  g.key_items = (dk != nullptr || dv != nullptr) ? batch * hkv * g.nkt * g.parts : 0;
  g.query_items = dq != nullptr ? batch * hq * g.nqt : 0;
  if (g.key_items + g.query_items == 0) return MUZO_OK;
  if (g.key_items + g.query_items > 0x7fffffffLL) return MUZO_ERR_UNSUPPORTED;
  float* stats = static_cast<float*>(d_workspace);
  g.stats = stats;
  CUtensorMap mq = {}, mk = {}, mv = {}, md = {};
  if (!none) {
    g.partial = g.parts > 1 ? stats + stats_bytes(batch, hq, g.nqt) / 4 + 4 : nullptr;
    st = encode_attn_map(&mq, q, dtype, head_dim, seq_q, hq, batch, strides[2], strides[1], strides[0], AM);
    if (st != MUZO_OK) return st;
    st = encode_attn_map(&mk, k, dtype, head_dim, seq_k, hkv, batch, strides[5], strides[4], strides[3], AN);
    if (st != MUZO_OK) return st;
    st = encode_attn_map(&mv, v, dtype, head_dim, seq_k, hkv, batch, strides[8], strides[7], strides[6], AN);
    if (st != MUZO_OK) return st;
    st = encode_attn_map(&md, dout, dtype, head_dim, seq_q, hq, batch, strides[14], strides[13], strides[12], AM);
    if (st != MUZO_OK) return st;
    uint32_t* largest = reinterpret_cast<uint32_t*>(stats + stats_bytes(batch, hq, g.nqt) / 4);
    g.largest = largest;
    const int64_t query_tiles = batch * hq * g.nqt, value_tiles = dtype == MUZO_F16 ? batch * hkv * g.nkt : 0;
    if (query_tiles + value_tiles > 0x7fffffffLL) return MUZO_ERR_UNSUPPORTED;
    if (dtype == MUZO_F16) MUZO_CUDA_CHECK(cudaMemsetAsync(largest, 0, 8, s));
    auto pre = dtype == MUZO_BF16 ? attn_bwd_stats_kernel<1> : attn_bwd_stats_kernel<0>;
    pre<<<static_cast<unsigned>(query_tiles + value_tiles), kStatThreads, 0, s>>>(
        Rows16{static_cast<const uint16_t*>(out), strides[9], strides[10], strides[11]},
        Rows16{static_cast<const uint16_t*>(dout), strides[12], strides[13], strides[14]},
        Rows16{static_cast<const uint16_t*>(v), strides[6], strides[7], strides[8]}, lse, stats, largest, g.hq, seq_q, g.nqt,
        g.hd, static_cast<unsigned>(query_tiles), g.hkv, seq_k, g.nkt, d_key_lo, d_key_hi);
    count_launches(1);
    st = launch_status();
    if (st != MUZO_OK) return st;
  }
  if (dtype == MUZO_BF16)
    return head_dim <= 64 ? launch_bwd<1, 64>(mq, mk, mv, md, g, s) : launch_bwd<1, 128>(mq, mk, mv, md, g, s);
  return head_dim <= 64 ? launch_bwd<0, 64>(mq, mk, mv, md, g, s) : launch_bwd<0, 128>(mq, mk, mv, md, g, s);
}

}  // extern "C"
