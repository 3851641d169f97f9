// Attention forward on the tensor cores with the per-head maximum of the pre-softmax logits as a
// side output: QK-Clip's capture (qk_clip.py:173-196) computed by the attention that the forward
// runs anyway, so Q K^T is formed once. For training it also keeps each row's log-sum-exp, from which
// the backward pass (attention_bwd.cu) recomputes the probabilities.
//
// One CTA per (batch, query head, block of 256 queries), 12 warps. The block is two query tiles
// of 128 rows that share every K / V tile of 128 keys, so each K / V byte loaded serves 256 rows:
//   warp 0      TMA producer (one thread): both query tiles once, then K tiles (K-major) into a
//               1-stage ring, refilled once both tiles' S = Q K^T has read it;
//   warp 10     TMA producer (one thread): V tiles (MN-major, the second operand of P V) into a
//               2-stage ring, refilled once both tiles' P V has read it;
//   warps 1, 11 MMA issuers of query tiles 0 and 1 (one thread each; warp 1 owns TMEM): S_s = Q_s
//               K_j^T into its S buffer (fp32 in TMEM) as soon as the softmax holds the last S in
//               registers, so that it is formed while that tile's exponentials run, then
//               O_s += P_s V_j into its fp32 accumulator, which stays in TMEM;
//   warps 2..9  two softmax streams of four warps, stream s for query tile s, one warp per TMEM
//               lane quarter, one query row per thread, all 128 keys of each tile: the raw
//               logits' maximum (the side output, over visible logits only), the online softmax
//               in base 2 with a lazy rescale (O and the row sum are rescaled only when the row
//               maximum grows by more than 2^8), P in bf16/fp16 written to shared memory in the
//               128-byte swizzled K-major layout the MMA reads, and at the end O / l stored to
//               [B, Sq, Hq, D]. The streams take turns at their exponentials: one has the
//               special-function unit to itself while the other waits for its S, finds its maxima
//               and hands its P over.
// A Llama-3-70B-shaped layer (4096 tokens, 64 and 8 heads of 128, causal) takes 0.269 ms, 1020 TFLOP/s:
// about 3400 cycles per K / V tile for both streams, of which 2048 are the special-function unit's and
// 2048 the tensor cores'. A turn takes 1500 cycles, not 1024, one warp per scheduler being all that
// issues in it, and its hand-over 150.
// Visibility: key j of batch b is visible to query i when key_lo[b] <= j < key_hi[b] (padding)
// and, when causal, j <= i + Sk - Sq. Rows without a visible key are written as zeros.
// Every wait is bounded; on timeout the kernel records a code in the status word, raises its
// abort flag, drains its loads and MMAs, writes NaN to its rows, frees TMEM and returns.
#include <atomic>
#include <cfloat>
#include <cstdlib>

#include "attention_common.cuh"

namespace muzo {
namespace {

using namespace tc;
using namespace attn;

constexpr int AMB = 2 * AM;      // query rows per CTA: two query tiles share each K / V tile
constexpr int A_THREADS = 384;   // warp 0 TMA of Q and K, warps 1 and 11 MMA of streams 0 and 1, warps 2..9
                                 // softmax (two streams of four warps, one warp per TMEM lane quarter),
                                 // warp 10 TMA of V
constexpr int K_STAGES = 1;      // K ring depth (tile j uses K stage j % K_STAGES)
constexpr int BOX_BYTES = 64 * ABK * 2;      // one 64 x 64 box of the MN-major V operand (8 KB)
constexpr uint32_t TMEM_COLS = 512;          // S of each stream at 0 and 128, O of each stream from 256
constexpr float kRescaleLog2 = 8.0f;          // lazy rescale threshold: P stays below 2^8

template <int D>
struct AttnLayout {
  static constexpr int Q_BYTES = (D / ABK) * SUB_BYTES;
  static constexpr int K_BYTES = (D / ABK) * SUB_BYTES;
  static constexpr int V_BYTES = 2 * (D / ABK) * BOX_BYTES;
  static constexpr int P_BYTES = 2 * SUB_BYTES;   // one 128 x 128 P tile per stream
  // V ring depth: two stages next to two Q tiles, one K stage and two P tiles (224 KB for D = 128)
  static constexpr int V_STAGES = 2;
  static constexpr int TILES_BYTES = 2 * Q_BYTES + K_STAGES * K_BYTES + V_STAGES * V_BYTES + 2 * P_BYTES;
  static constexpr int BAR_BYTES = 256;           // barriers, TMEM address, flags
  // tiles, barriers and 1 KB of alignment (225.25 KB for D = 128, within the 227 KB a CTA may
  // use); at least 116 KB so that one CTA holds an SM (every CTA allocates all 512 TMEM columns)
  static constexpr int NEED = TILES_BYTES + BAR_BYTES + 1024;
  static constexpr int SMEM_BYTES = NEED > 116 * 1024 ? NEED : 116 * 1024;
};

struct AttnArgs {
  int64_t sq, sk, shift;       // shift = Sk - Sq: causal key j is visible to query i when j <= i + shift
  int hq, group, nqb, causal, batch;
  int64_t num_items;           // batch * hq * nqb
  float scale_log2;            // softmax scale * log2(e)
  const int32_t* key_lo;       // per batch, or null (0)
  const int32_t* key_hi;       // per batch, or null (Sk)
  void* out;
  int64_t o_sb, o_sh, o_ss;    // output strides in elements; D contiguous
  int hd;                      // head dimension (at most D: the tiles' further columns hold zeros)
  float* lse;                  // log of each row's sum of exp(scaled logit), [B][Hq][Sq], or null
  int* enc;                    // per-head running maximum of the raw logits (order-preserving ints), or null
  int32_t* valid;
  int32_t* status;
};

__device__ __forceinline__ int encode_max(float f) {
  const int b = __float_as_int(f);
  return b >= 0 ? b : b ^ 0x7fffffff;
}

// Work item -> (batch, head, block of 256 queries); the longest query blocks (last, when causal) first.
__device__ __forceinline__ void attn_item(const AttnArgs& g, int64_t t, int& b, int& h, int& qb) {
  const int64_t bh_count = static_cast<int64_t>(g.batch) * g.hq;
  qb = g.nqb - 1 - static_cast<int>(t / bh_count);
  const int64_t bh = t % bh_count;
  b = static_cast<int>(bh / g.hq);
  h = static_cast<int>(bh % g.hq);
}

// First key tile of a work item and the tile counts of its two query tiles (zero for a tile with
// no row inside the sequence or no visible key).
__device__ __forceinline__ void attn_tiles(const AttnArgs& g, int b, int qb, int64_t& lo, int64_t& hi, int& t0,
                                           int& n0, int& n1) {
  key_range(g.key_lo, g.key_hi, g.sk, b, lo, hi);
  t0 = static_cast<int>(lo / AN);
  int n[2];
  for (int t = 0; t < 2; ++t) {
    const int64_t first = static_cast<int64_t>(qb) * AMB + t * AM;   // first row of query tile t
    n[t] = 0;
    if (first >= g.sq) continue;
    const int64_t last_row = first + AM - 1 < g.sq - 1 ? first + AM - 1 : g.sq - 1;
    int64_t end = hi;
    if (g.causal && last_row + g.shift + 1 < end) end = last_row + g.shift + 1;  // keys the tile's last row sees
    if (end > lo) n[t] = static_cast<int>((end + AN - 1) / AN) - t0;
  }
  n0 = n[0];
  n1 = n[1];
}

// The two softmax streams take turns at their exponentials: one fills the special-function unit while
// the other takes its tile's maximum and waits for its products. Without turns both did the same at
// the same time (4300 cycles a tile for both, 2050 of them the unit's). Stream 0 waits from its second
// tile on for stream 1's last tile, stream 1 for stream 0's same tile; where the other stream has no
// such tile there is nothing to wait for. Both streams execute every turn, after a timeout too, so the
// hardware barriers (which have no time limit) always complete.
constexpr int kTurnBarrier = 1;   // named barriers 1 (stream 0's turn) and 2
__device__ __forceinline__ void turn_wait(int stream, int u, int n0, int n1) {
  __syncwarp();   // the barrier instructions want their warp converged
  if (stream == 0 ? (u >= 1 && u - 1 < n1) : u < n0)
    asm volatile("bar.sync %0, 256;" ::"r"(kTurnBarrier + stream) : "memory");
}
__device__ __forceinline__ void turn_pass(int stream, int u, int n0, int n1) {
  __syncwarp();
  if (stream == 0 ? u < n1 : u + 1 < n0) asm volatile("bar.arrive %0, 256;" ::"r"(kTurnBarrier + 1 - stream) : "memory");
}

// Three-input maximum (NaN-propagating) and minimum (sm_100).
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int FMT, int D, bool REC>
__global__ void __launch_bounds__(A_THREADS, 1)
attn_fwd_max_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, AttnArgs g) {
  using L = AttnLayout<D>;
  constexpr int NKB = D / ABK;   // 64-wide slices of the head dimension
  constexpr int VS = L::V_STAGES;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw_addr & 1023u)) & 1023u);
  // Two query tiles of 128 rows (streams 0 and 1) share every K / V tile of 128 keys: K through a
  // K_STAGES ring (a stage is free once both tiles' S has read it), V through a VS-stage ring (free
  // once both tiles' P V has read it). Each stream owns an S buffer and an O accumulator in TMEM
  // and a P tile in shared memory.
  uint8_t* sQ = smem;                                   // [2][NKB][128 x 64]
  uint8_t* sK = sQ + 2 * L::Q_BYTES;
  uint8_t* sV = sK + K_STAGES * L::K_BYTES;
  uint8_t* sP = sV + VS * L::V_BYTES;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::TILES_BYTES);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + K_STAGES;
  uint64_t* v_full = k_empty + K_STAGES;
  uint64_t* v_empty = v_full + VS;
  uint64_t* s_full = v_empty + VS;          // [stream]: S of the stream's next tile computed
  uint64_t* p_full = s_full + 2;            // [stream]: P written (and S read) by the stream's 4 warps
  uint64_t* o_done = p_full + 2;            // [stream]: P V of the stream's last tile done
  uint64_t* s_free = o_done + 2;            // [stream]: S in registers, its buffer may take the next S
  uint64_t* drain = s_free + 2;             // [stream]
  uint64_t* stall_bar = drain + 2;          // nothing arrives here: a stall request waits on it
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(stall_bar + 1);
  int* abort_flag = reinterpret_cast<int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int b, h, qb;
  attn_item(g, blockIdx.x, b, h, qb);
  int64_t lo, hi;
  int t0, n0, n1;
  attn_tiles(g, b, qb, lo, hi, t0, n0, n1);
  const int ntiles = n0 > n1 ? n0 : n1;   // K / V tiles loaded (stream 1's rows come later: n1 >= n0)
  const int kvh = h / g.group;
  // status word 1: a role (1 producer, 2 MMA, 3 softmax) whose first wait is made to expire
  const int stall = *reinterpret_cast<volatile int*>(g.status + 1);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < K_STAGES; ++s) { mbar_init(k_full + s, 1); mbar_init(k_empty + s, 2); }
    for (int s = 0; s < VS; ++s) { mbar_init(v_full + s, 1); mbar_init(v_empty + s, 2); }
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full + s, 1); mbar_init(p_full + s, 4); mbar_init(o_done + s, 1); mbar_init(s_free + s, 4);
      mbar_init(drain + s, 1);
    }
    mbar_init(stall_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  const uint32_t tmem_o = tmem_base + 2 * AN;   // O of stream s at tmem_o + s * D

  if (warp == 0 || warp == 10) {
    // ------------------------------------------------------------------ TMA producers
    // warp 0: both query tiles once, then K_j into its stage once S_{j - K_STAGES} of both streams has
    // read it; warp 10: V_j into V stage j % VS once P_{j-VS} V_{j-VS} of both streams has read it
    if (lane == 0 && ntiles > 0) {
      const bool keys = warp == 0;
      const int stages = keys ? K_STAGES : VS;
      uint64_t* full = keys ? k_full : v_full;
      uint64_t* empty = keys ? k_empty : v_empty;
      const uint32_t stage_bytes = keys ? L::K_BYTES : L::V_BYTES;
      bool ok = !(keys && stall == kErrTimeoutProducer && !mbar_wait(stall_bar, 0, kStallLimitCycles));
      if (keys && ok) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_q)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
        mbar_arrive_expect_tx(q_full, 2 * L::Q_BYTES);
        for (int t = 0; t < 2; ++t)
          for (int kb = 0; kb < NKB; ++kb)
            tma_load_4d(&map_q, q_full, sQ + t * L::Q_BYTES + kb * SUB_BYTES, kb * ABK, qb * AMB + t * AM, h, b);
      } else if (!keys) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
      }
      const bool q_armed = keys && ok;
      uint32_t armed = 0, armed_parity = 0;
      for (int j = 0; j < ntiles && ok; ++j) {
        const int stage = j % stages;
        const uint32_t phase = static_cast<uint32_t>((j / stages) & 1);
        if (!mbar_wait(empty + stage, phase ^ 1)) { ok = false; break; }
        if (*reinterpret_cast<volatile int*>(abort_flag)) { ok = false; break; }
        mbar_arrive_expect_tx(full + stage, stage_bytes);
        armed |= 1u << stage;
        armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
        const int key0 = (t0 + j) * AN;
        if (keys) {
          uint8_t* dst = sK + stage * L::K_BYTES;
          for (int kb = 0; kb < NKB; ++kb) tma_load_4d(&map_k, full + stage, dst + kb * SUB_BYTES, kb * ABK, key0, kvh, b);
        } else {
          uint8_t* dst = sV + stage * L::V_BYTES;
          for (int kc = 0; kc < 2; ++kc)
            for (int dc = 0; dc < NKB; ++dc)
              tma_load_4d(&map_v, full + stage, dst + (kc * NKB + dc) * BOX_BYTES, dc * ABK, key0 + kc * 64, kvh, b);
        }
      }
      if (!ok) {
        atomicCAS(g.status, kErrNone, kErrTimeoutProducer);
        atomicExch(abort_flag, 1);
        if (g.valid) atomicExch(g.valid, 0);
      }
      // every load of this CTA must have landed before it may exit (bounded)
      if (q_armed) mbar_wait(q_full, 0);
      for (int s2 = 0; s2 < stages; ++s2)
        if (armed & (1u << s2)) mbar_wait(full + s2, (armed_parity >> s2) & 1u);
    }
    __syncwarp();
  } else if (warp == 1 || warp == 11) {
    // ------------------------------------------------------------------ MMA issuers, one per stream
    // Stream s: S_s(0); then per tile j S_s(j + 1) as soon as the softmax holds S_s(j) in registers, and
    // O_s += P_s(j) V_j once P_s(j) is written. A K or V stage is released by both issuers: by a commit
    // behind the product that read it, or by an arrival where the stream has no such tile.
    if (ntiles > 0 && elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_fmt(AM, AN, false, false, FMT);
      constexpr uint32_t idesc_pv = make_idesc_fmt(AM, D, false, true, FMT);
      const int s = warp == 1 ? 0 : 1;
      const int mine = s == 0 ? n0 : n1;
      const uint32_t sq_ = smem_u32(sQ + s * L::Q_BYTES), sp = smem_u32(sP + s * L::P_BYTES);
      auto ready = [&](uint64_t* bar, int phase) -> bool {
        if (!mbar_wait(bar, static_cast<uint32_t>(phase & 1))) return false;
        if (*reinterpret_cast<volatile int*>(abort_flag)) return false;
        tc_fence_after();
        return true;
      };
      auto issue_s = [&](int j) -> bool {
        const int stage = j % K_STAGES;
        if (!ready(k_full + stage, j / K_STAGES)) return false;
        if (j >= mine) {
          mbar_arrive(k_empty + stage);
          return true;
        }
        if (j > 0 && !ready(s_free + s, j - 1)) return false;
        const uint32_t sk_ = smem_u32(sK + stage * L::K_BYTES);
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int k = 0; k < ABK / 16; ++k)
            umma_f16(tmem_base + s * AN, make_sdesc(sq_ + kb * SUB_BYTES + k * 32, 16, 1024),
                     make_sdesc(sk_ + kb * SUB_BYTES + k * 32, 16, 1024), idesc_s, (kb > 0 || k > 0) ? 1u : 0u);
        umma_commit(s_full + s);
        if (j + K_STAGES < ntiles) umma_commit(k_empty + stage);   // nothing is committed that nobody waits for:
        return true;                                               // it might arrive after the CTA's end
      };
      auto issue_pv = [&](int j) -> bool {
        const int stage = j % VS;
        if (!ready(v_full + stage, j / VS)) return false;
        if (j >= mine) {
          mbar_arrive(v_empty + stage);
          return true;
        }
        if (!ready(p_full + s, j)) return false;
        const uint32_t sv = smem_u32(sV + stage * L::V_BYTES);
#pragma unroll
        for (int kc = 0; kc < 2; ++kc)
#pragma unroll
          for (int k = 0; k < ABK / 16; ++k)
            umma_f16(tmem_o + s * D, make_sdesc(sp + kc * SUB_BYTES + k * 32, 16, 1024),
                     make_sdesc(sv + kc * NKB * BOX_BYTES + k * (16 * 128), BOX_BYTES, 1024), idesc_pv,
                     (j > 0 || kc > 0 || k > 0) ? 1u : 0u);
        if (j + VS < ntiles) umma_commit(v_empty + stage);
        umma_commit(o_done + s);        // P buffer of the stream free, O_s holds its tiles up to j
        return true;
      };
      bool ok = stall != kErrTimeoutMma || mbar_wait(stall_bar, 0, kStallLimitCycles);
      ok = ok && ready(q_full, 0) && issue_s(0);
      for (int j = 0; j < ntiles && ok; ++j) {
        if (j + 1 < ntiles) ok = issue_s(j + 1);
        ok = ok && issue_pv(j);
      }
      if (!ok) {
        atomicCAS(g.status, kErrNone, kErrTimeoutMma);
        atomicExch(abort_flag, 1);
        if (g.valid) atomicExch(g.valid, 0);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax streams and epilogue
    // Stream s (warps 2..5: s = 0, warps 6..9: s = 1) owns query tile s of the block: one warp per
    // TMEM lane quarter, one query row per thread, all 128 keys of each tile. The two streams work on
    // the same K / V tiles and take turns at their exponentials. (Eight warps per stream, 64 keys each,
    // fill a turn better but have to exchange their rows' maxima: 283 us against 269 for a
    // Llama-3-70B-shaped layer.)
    const int quarter = warp & 3;
    const int stream = (warp - 2) >> 2;
    const int r = 32 * quarter + lane;                 // row of the tile == TMEM lane
    const int64_t row = static_cast<int64_t>(qb) * AMB + stream * AM + r;
    const bool row_in = row < g.sq;
    const int64_t jmax = g.causal ? row + g.shift : g.sk - 1;  // last key visible by causality
    const uint32_t lane_addr = static_cast<uint32_t>(32 * quarter) << 16;
    const uint32_t s_cols = tmem_base + lane_addr + stream * AN;
    const uint32_t o_cols = tmem_o + lane_addr + stream * D;
    uint8_t* my_p = sP + stream * L::P_BYTES;
    const int n_mine = stream == 0 ? n0 : n1;
    float m_run = -INFINITY;    // running maximum of the scaled logits (log2 units) used by P
    float l_run = 0.0f;         // running sum of P
    float raw_max = -INFINITY;  // side output: maximum of the visible raw logits q . k (NaN-propagating)
    float raw_min = INFINITY;   // a visible -inf logit shows here
    bool ok = true;
    if (stall == kErrTimeoutEpilogue) {
      bool waited = true;
      if (lane == 0) waited = mbar_wait(stall_bar, 0, kStallLimitCycles);
      ok = __shfl_sync(0xffffffffu, waited ? 1 : 0, 0) != 0;
    }
    int turns = 0;   // turns taken and passed on
    for (int u = 0; u < n_mine && ok; ++u) {
      bool ready = true;
      if (lane == 0) ready = mbar_wait(s_full + stream, static_cast<uint32_t>(u & 1));
      ready = __shfl_sync(0xffffffffu, ready ? 1 : 0, 0) != 0;
      if (!ready || *reinterpret_cast<volatile int*>(abort_flag)) { ok = false; break; }
      tc_fence_after();
      // visible key columns [c_lo, c_hi) of this tile for this row
      const int64_t key0 = static_cast<int64_t>(t0 + u) * AN;
      const int64_t end = hi < jmax + 1 ? hi : jmax + 1;
      int c_lo = 0, c_hi = 0;
      if (row_in) {
        const int64_t a0 = lo - key0, a1 = end - key0;
        c_lo = a0 < 0 ? 0 : (a0 > AN ? AN : static_cast<int>(a0));
        c_hi = a1 < 0 ? 0 : (a1 > AN ? AN : static_cast<int>(a1));
        if (c_hi < c_lo) c_hi = c_lo;
      }
      const bool all_visible = c_lo == 0 && c_hi == AN;
      // S into registers, once: the columns are free for the next S while this tile's exponentials
      // run. 128 of the thread's 168 registers hold the row (both passes reading TMEM instead:
      // 314 us against 286 for a Llama-3-70B-shaped layer).
      uint32_t v[AN];
      __syncwarp();
      tmem_ld128(s_cols, v);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free + stream);
      // the tile's maximum (and, to record, minimum) over the visible logits; the others become -inf
      float mx[4], mn[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) { mx[q] = -INFINITY; mn[q] = INFINITY; }
      if (!all_visible) {
#pragma unroll
        for (int c = 0; c < AN; ++c) {
          const bool visible = c >= c_lo && c < c_hi;
          if (REC) mn[c & 3] = fminf(mn[c & 3], visible ? __uint_as_float(v[c]) : INFINITY);
          if (!visible) v[c] = 0xff800000u;
        }
      }
#pragma unroll
      for (int c = 0; c < AN; c += 2) {
        const float x0 = __uint_as_float(v[c]), x1 = __uint_as_float(v[c + 1]);
        mx[(c >> 1) & 3] = max3_nan(mx[(c >> 1) & 3], x0, x1);
        if (REC && all_visible) mn[(c >> 1) & 3] = min3(mn[(c >> 1) & 3], x0, x1);
      }
      const float mt = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], -INFINITY);
      if (REC) {
        raw_max = max3_nan(raw_max, mt, -INFINITY);
        raw_min = min3(min3(raw_min, mn[0], mn[1]), mn[2], mn[3]);
      }
      // lazy online softmax in base 2
      const float mt2 = mt * g.scale_log2;
      float alpha = 1.0f;
      bool rescale = false;
      if (mt2 > m_run + kRescaleLog2 || mt != mt) {   // a NaN logit makes its row NaN
        alpha = m_run == -INFINITY ? 0.0f : fast_exp2(m_run - mt2);
        rescale = u > 0;
        m_run = mt2;
      }
      // P V of this stream's previous tile must be done: its P buffer is reused and O may be rescaled
      if (u > 0) {
        bool done = true;
        if (lane == 0) done = mbar_wait(o_done + stream, static_cast<uint32_t>((u - 1) & 1));
        done = __shfl_sync(0xffffffffu, done ? 1 : 0, 0) != 0;
        if (!done) { ok = false; break; }
        tc_fence_after();
      }
      if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {   // 16 at a time: S holds most of the registers
          uint32_t o[16];
          __syncwarp();
          tmem_ld16(o_cols + c * 16, o);
          if (rescale) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          }
          __syncwarp();
          tmem_st16(o_cols + c * 16, o);
        }
      }
      // P = 2^(s * scale_log2 - m_run), its row sum, and P in the 128-byte swizzled K-major layout
      // (chunk c16 of 8 keys of K block c16 / 8 sits at row * 128 + ((c16 ^ (row & 7)) * 16, modulo 8).
      // A row that has seen no logit above -inf has all of this tile's there: 1 * -inf + 0 gives P = 0.
      const float nm = m_run == -INFINITY ? 0.0f : -m_run, mul = m_run == -INFINITY ? 1.0f : g.scale_log2;
      turn_wait(stream, u, n0, n1);
      float lsum[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) lsum[q] = 0.0f;
#pragma unroll
      for (int c16 = 0; c16 < AN / 8; ++c16) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = 8 * c16 + 2 * e;
          float x0 = __uint_as_float(v[c]), x1 = __uint_as_float(v[c + 1]);
          fma_pair(x0, x1, mul, nm, nm);
          const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
          add_pair(lsum[2 * e], lsum[2 * e + 1], p0, p1);
          w[e] = FMT == 1 ? pack_bf16(p0, p1) : pack_half(p0, p1);
        }
        *reinterpret_cast<uint4*>(my_p + (c16 >> 3) * SUB_BYTES + r * 128 + (((c16 ^ r) & 7) << 4)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
      turn_pass(stream, u, n0, n1);
      turns = u + 1;
      l_run = l_run * alpha + (((lsum[0] + lsum[1]) + (lsum[2] + lsum[3])) + ((lsum[4] + lsum[5]) + (lsum[6] + lsum[7])));
      // keys outside [lo, hi) that share a tile with visible ones: their P is 0, but 0 times a
      // non-finite V would still reach O, so their V rows are cleared before P V reads them
      if (lo > key0 || hi < (g.sk < key0 + AN ? g.sk : key0 + AN)) {
        const int stage = u % VS;
        if (!mbar_wait(v_full + stage, static_cast<uint32_t>((u / VS) & 1))) ok = false;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (key0 + r < lo || key0 + r >= hi) {
          uint8_t* vrow = sV + stage * L::V_BYTES + (r >> 6) * (NKB * BOX_BYTES) + (r & 63) * 128;
#pragma unroll
          for (int dc = 0; dc < NKB; ++dc)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(vrow + dc * BOX_BYTES + 16 * e) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full + stream);
    }
    for (; turns < n_mine; ++turns) {   // this warp gave up: its turns pass all the same
      turn_wait(stream, turns, n0, n1);
      turn_pass(stream, turns, n0, n1);
    }
    // this stream's last P V must be done before O_s is read
    if (ok && n_mine > 0) {
      bool done = true;
      if (lane == 0) done = mbar_wait(o_done + stream, static_cast<uint32_t>((n_mine - 1) & 1));
      done = __shfl_sync(0xffffffffu, done ? 1 : 0, 0) != 0;
      if (!done) ok = false;
      tc_fence_after();
    }
    if (ok) {
      // O / l of this row (zeros for a row without a visible key or a tile without one)
      const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
      if (g.lse != nullptr && row_in)
        g.lse[(static_cast<int64_t>(b) * g.hq + h) * g.sq + row] =
            l_run == 0.0f ? -INFINITY : (m_run + log2f(l_run)) * 0.6931471805599453f;
      uint16_t* orow = reinterpret_cast<uint16_t*>(g.out) + static_cast<int64_t>(b) * g.o_sb +
                       static_cast<int64_t>(h) * g.o_sh + row * g.o_ss;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (n_mine > 0) {
          __syncwarp();
          tmem_ld32(o_cols + c * 32, v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        if (row_in) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (c * 32 + 8 * q >= g.hd) break;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float o0 = __uint_as_float(v[8 * q + 2 * e]) * inv;
              const float o1 = __uint_as_float(v[8 * q + 2 * e + 1]) * inv;
              w[e] = FMT == 1 ? pack_bf16(o0, o1) : pack_half(o0, o1);
            }
            *reinterpret_cast<uint4*>(orow + c * 32 + 8 * q) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (REC) {
        float m = raw_max;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max3_nan(m, __shfl_xor_sync(0xffffffffu, m, o), -INFINITY);
        float mnv = raw_min;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mnv = fminf(mnv, __shfl_xor_sync(0xffffffffu, mnv, o));
        if (lane == 0) {
          if (m != m || m == INFINITY || mnv == -INFINITY) atomicExch(g.valid, 0);
          else if (m > -INFINITY) atomicMax(g.enc + h, encode_max(m));
        }
      }
    } else if (lane == 0) {
      atomicCAS(g.status, kErrNone, kErrTimeoutEpilogue);
      atomicExch(abort_flag, 1);
      if (g.valid) atomicExch(g.valid, 0);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (*reinterpret_cast<volatile int*>(abort_flag)) {   // every role has ended: the same answer in all threads
    // the MMAs that an aborted CTA issued end before its TMEM is released (bounded), and the arrivals of commits that
    // nobody waits for any more, which have no stated order, get 50 us
    if ((warp == 1 || warp == 11) && elect_one()) {
      uint64_t* drained = drain + (warp == 1 ? 0 : 1);
      umma_commit(drained);
      mbar_wait(drained, 0);
      mbar_wait(stall_bar, 0, kSettleCycles);
    }
    __syncthreads();
    // a CTA that gave up leaves NaN in all of its rows, so that nobody takes old memory for its output
    const int64_t row0 = static_cast<int64_t>(qb) * AMB;
    lose_tile(static_cast<uint16_t*>(g.out) + b * g.o_sb + h * g.o_sh, g.o_ss, row0, AMB, g.sq, g.hd);
    if (g.lse != nullptr && threadIdx.x < AMB && row0 + threadIdx.x < g.sq)
      g.lse[(static_cast<int64_t>(b) * g.hq + h) * g.sq + row0 + threadIdx.x] = __int_as_float(0x7fffffff);
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS)
                 : "memory");
  }
}

template <int FMT, int D, bool REC>
int launch_attn(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AttnArgs& g,
                cudaStream_t s) {
  auto kern = attn_fwd_max_kernel<FMT, D, REC>;
  static std::atomic<bool> configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return MUZO_ERR_UNSUPPORTED;
  if (!configured[dev].load(std::memory_order_acquire)) {
    MUZO_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, AttnLayout<D>::SMEM_BYTES));
    configured[dev].store(true, std::memory_order_release);
  }
  kern<<<static_cast<unsigned>(g.num_items), A_THREADS, AttnLayout<D>::SMEM_BYTES, s>>>(mq, mk, mv, g);
  count_launches(1);
  return launch_status();
}

// With or without the maxima (whose minima, for a visible -inf, cost a third of the first pass).
template <int FMT, int D>
int launch_head(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const AttnArgs& g, cudaStream_t s) {
  return g.enc != nullptr ? launch_attn<FMT, D, true>(mq, mk, mv, g, s) : launch_attn<FMT, D, false>(mq, mk, mv, g, s);
}

__global__ void init_attn_max_kernel(int* enc, int n, int32_t* valid) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i < n) enc[i] = encode_max(-INFINITY);
  if (i == 0) *valid = 1;
}

// smax[h] = dtype(dtype(max raw logit) * scale), the eager logit's rounding (monotonic, so the
// rounded maximum is the maximum of the rounded logits); heads without a visible logit stay -inf.
__global__ void finalize_attn_max_kernel(int* enc, int n, int dtype, float scale) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int e = enc[i];
  float v = __int_as_float(e >= 0 ? e : e ^ 0x7fffffff);
  if (v > -INFINITY) v = round_to(round_to(v, dtype) * scale, dtype);
  reinterpret_cast<float*>(enc)[i] = v;
}

}  // namespace
}  // namespace muzo

using namespace muzo;

extern "C" {

int muzo_attention_max_lse(const void* q, const void* k, const void* v, void* out, float* lse, int dtype, int64_t batch,
                           int64_t hq, int64_t hkv, int64_t seq_q, int64_t seq_k, int64_t head_dim,
                       int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
                       int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
                       int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
                       int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s, int causal, float scale,
                       const int32_t* d_key_lo, const int32_t* d_key_hi, float* smax, int32_t* d_valid,
                       int32_t* d_status, void* stream) {
  if (q == nullptr || ((k == nullptr || v == nullptr) && seq_k != 0) || out == nullptr || d_status == nullptr || batch < 0 ||
      hq <= 0 || hkv <= 0 || hq % hkv != 0 || seq_q < 0 || seq_k < 0 ||
      (smax != nullptr && d_valid == nullptr) || (lse != nullptr && !(scale > 0.0f && scale <= FLT_MAX)))
    return MUZO_ERR_ARG;
  if (dtype != MUZO_BF16 && dtype != MUZO_F16) return MUZO_ERR_DTYPE;
  if (head_dim < 8 || head_dim % 8 != 0 || head_dim > 128) return MUZO_ERR_UNSUPPORTED;
  const int64_t strides[12] = {q_stride_b, q_stride_h, q_stride_s, k_stride_b, k_stride_h, k_stride_s,
                               v_stride_b, v_stride_h, v_stride_s, o_stride_b, o_stride_h, o_stride_s};
  for (int64_t st : strides)
    if (st % 8 != 0) return MUZO_ERR_ALIGN;
  if (!aligned16p(q) || !aligned16p(k) || !aligned16p(v) || !aligned16p(out)) return MUZO_ERR_ALIGN;
  if (batch > 0x7fffffffLL || hq > 0x7fffffffLL || seq_q > 0x7fffffffLL || seq_k > 0x7fffffffLL)
    return MUZO_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int* enc = reinterpret_cast<int*>(smax);
  if (enc != nullptr) {
    init_attn_max_kernel<<<static_cast<unsigned>((hq + 255) / 256), 256, 0, s>>>(enc, static_cast<int>(hq), d_valid);
    count_launches(1);
  }
  const int64_t nqb = (seq_q + AMB - 1) / AMB;
  const int64_t items = batch * hq * nqb;
  if (items > 0) {
    if (items > 0x7fffffffLL) return MUZO_ERR_UNSUPPORTED;
    CUtensorMap mq, mk, mv;
    if (seq_k == 0) {   // no key tile is loaded: any valid map will do
      k = v = q;
      k_stride_b = v_stride_b = k_stride_h = v_stride_h = k_stride_s = v_stride_s = 8;
    }
    const int64_t map_keys = seq_k > 0 ? seq_k : 1;
    int st = encode_attn_map(&mq, q, dtype, head_dim, seq_q, hq, batch, q_stride_s, q_stride_h, q_stride_b, AM);
    if (st != MUZO_OK) return st;
    st = encode_attn_map(&mk, k, dtype, head_dim, map_keys, hkv, batch, k_stride_s, k_stride_h, k_stride_b, AN);
    if (st != MUZO_OK) return st;
    st = encode_attn_map(&mv, v, dtype, head_dim, map_keys, hkv, batch, v_stride_s, v_stride_h, v_stride_b, 64);
    if (st != MUZO_OK) return st;
    AttnArgs g;
    g.sq = seq_q; g.sk = seq_k; g.shift = seq_k - seq_q;
    g.hq = static_cast<int>(hq); g.group = static_cast<int>(hq / hkv); g.nqb = static_cast<int>(nqb);
    g.causal = causal ? 1 : 0; g.batch = static_cast<int>(batch);
    g.num_items = items;
    g.scale_log2 = scale * 1.4426950408889634f;
    g.key_lo = d_key_lo; g.key_hi = d_key_hi;
    g.out = out; g.o_sb = o_stride_b; g.o_sh = o_stride_h; g.o_ss = o_stride_s;
    g.hd = static_cast<int>(head_dim); g.lse = lse;
    g.enc = enc; g.valid = d_valid; g.status = d_status;
    if (dtype == MUZO_BF16)
      st = head_dim <= 64 ? launch_head<1, 64>(mq, mk, mv, g, s) : launch_head<1, 128>(mq, mk, mv, g, s);
    else
      st = head_dim <= 64 ? launch_head<0, 64>(mq, mk, mv, g, s) : launch_head<0, 128>(mq, mk, mv, g, s);
    if (st != MUZO_OK) return st;
  }
  if (enc != nullptr) {
    finalize_attn_max_kernel<<<static_cast<unsigned>((hq + 255) / 256), 256, 0, s>>>(enc, static_cast<int>(hq), dtype,
                                                                                     scale);
    count_launches(1);
  }
  return launch_status();
}

int muzo_attention_max(const void* q, const void* k, const void* v, void* out, int dtype, int64_t batch,
                       int64_t hq, int64_t hkv, int64_t seq_q, int64_t seq_k, int64_t head_dim,
                       int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_s,
                       int64_t k_stride_b, int64_t k_stride_h, int64_t k_stride_s,
                       int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_s,
                       int64_t o_stride_b, int64_t o_stride_h, int64_t o_stride_s, int causal, float scale,
                       const int32_t* d_key_lo, const int32_t* d_key_hi, float* smax, int32_t* d_valid,
                       int32_t* d_status, void* stream) {
  return muzo_attention_max_lse(q, k, v, out, nullptr, dtype, batch, hq, hkv, seq_q, seq_k, head_dim, q_stride_b,
                                q_stride_h, q_stride_s, k_stride_b, k_stride_h, k_stride_s, v_stride_b, v_stride_h,
                                v_stride_s, o_stride_b, o_stride_h, o_stride_s, causal, scale, d_key_lo, d_key_hi, smax,
                                d_valid, d_status, stream);
}

}  // extern "C"
