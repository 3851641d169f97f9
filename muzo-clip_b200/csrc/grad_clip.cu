// The norm over all gradients of a model, and the gradients scaled by it:
//   norm = sqrt(sum over tensors and elements of g^2), or max |g|
//   factor = min(1, max_norm / (norm + 1e-6)),  out = dtype(factor * g)
// Both passes are bound by memory: the norm reads every gradient once, the scaling reads it again
// (from L2 where it still is there: the second pass walks the chunks backwards) and writes it.
//
// The tensors' addresses and sizes travel as kernel parameters, so that a call needs no table in
// device memory, no copy and no allocation beyond its partial sums, and can be captured into a
// graph. Tensors are cut into chunks of a power of two of elements; a fixed set of CTAs walks them.
// Each CTA leaves one partial sum and every reader adds the partial sums in the same order: equal
// calls give equal bits.
#include <algorithm>
#include <new>
#include <vector>

#include "muzo_common.cuh"

namespace muzo {
namespace {

constexpr int kThreads = 256;
// CTAs of a launch: what is resident at once (at most 42 and 51 registers a thread)
constexpr int kNormPerSm = 6, kScalePerSm = 5;
constexpr int kMaxCtas = 148 * kNormPerSm;  // and partial sums of a launch
constexpr int kSmallTable = 140;            // tensors in a launch whose parameters fit 4 KB
constexpr int kLargeTable = 1150;           // ... 32 KB

template <int N>
struct Table {
  uint64_t src[N];
  uint64_t dst[N];
  uint64_t numel[N];          // elements | source dtype << 56 | destination dtype << 60
  uint32_t first[N + 1];      // first chunk of each tensor, and the number of chunks
  int count;
  int chunk_shift;            // log2 of the elements per chunk
};
static_assert(sizeof(Table<kSmallTable>) <= 4096 - 64, "parameters of the small launch");
static_assert(sizeof(Table<kLargeTable>) <= 32764 - 64, "parameters of the large launch");

template <int N>
__device__ __forceinline__ int find_tensor(const Table<N>& t, uint32_t chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Elements of a chunk: [begin, end) of the tensor.
template <int N>
__device__ __forceinline__ void chunk_range(const Table<N>& t, int i, uint32_t chunk, int64_t& begin, int64_t& end) {
  const int64_t n = static_cast<int64_t>(t.numel[i] & ((1ull << 56) - 1));
  begin = static_cast<int64_t>(chunk - t.first[i]) << t.chunk_shift;
  end = begin + (1ll << t.chunk_shift);
  if (end > n) end = n;
}

__device__ __forceinline__ float max_abs_nan(float m, float x) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(m), "f"(fabsf(x)));
  return d;
}

// V consecutive elements, loaded and stored as one access of 8 or 16 bytes each; LAST: nothing reads
// them again (the norm's reads stay in L2 for the scaling).
template <int DTYPE, bool LAST = true, int V>
__device__ __forceinline__ void load_vec(const char* p, float (&v)[V]) {
  if constexpr (DTYPE == MUZO_F32) {
    static_assert(V == 4, "16 bytes of fp32");
    const float4 a = LAST ? __ldcs(reinterpret_cast<const float4*>(p)) : *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    uint32_t w[V / 2];
    if constexpr (V == 8) {
      const uint4 u = LAST ? __ldcs(reinterpret_cast<const uint4*>(p)) : *reinterpret_cast<const uint4*>(p);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const uint2 u = LAST ? __ldcs(reinterpret_cast<const uint2*>(p)) : *reinterpret_cast<const uint2*>(p);
      w[0] = u.x; w[1] = u.y;
    }
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
      v[2 * q] = DTYPE == MUZO_BF16 ? bf16_lo(w[q]) : half_lo(w[q]);
      v[2 * q + 1] = DTYPE == MUZO_BF16 ? bf16_hi(w[q]) : half_hi(w[q]);
    }
  }
}
template <int DTYPE, int V>
__device__ __forceinline__ void store_vec(char* p, const float (&v)[V]) {
  if constexpr (DTYPE == MUZO_F32) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  } else {
    uint32_t w[V / 2];
#pragma unroll
    for (int q = 0; q < V / 2; ++q)
      w[q] = DTYPE == MUZO_BF16 ? pack_bf16(v[2 * q], v[2 * q + 1]) : pack_half(v[2 * q], v[2 * q + 1]);
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
}

// Sum of squares of a few values. The squares are added in fp32 where that is safe; a sum outside
// [1e-30, 1e37], or not finite, is formed again in fp64 (squares of fp32 values reach 1e77, and
// those of small ones vanish).
template <int V>
__device__ __forceinline__ double sum_squares(const float (&v)[V]) {
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < V; ++k) s = fmaf(v[k], v[k], s);
  if (s >= 1e-30f && s <= 1e37f) return s;
  uint32_t any = 0;
#pragma unroll
  for (int k = 0; k < V; ++k) any |= __float_as_uint(v[k]);
  if ((any & 0x7fffffffu) == 0) return 0.0;
  double d = 0.0;
#pragma unroll
  for (int k = 0; k < V; ++k) d = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), d);
  return d;
}

// Running result of one thread: the sum of squares, or the largest magnitude.
template <bool INF>
struct Total {
  double sum = 0.0;
  float top = 0.0f;
  template <int V>
  __device__ __forceinline__ void add_vec(const float (&v)[V]) {
    if (INF) {
#pragma unroll
      for (int k = 0; k < V; ++k) top = max_abs_nan(top, v[k]);
    } else {
      sum += sum_squares(v);
    }
  }
  __device__ __forceinline__ void add(float v) {
    if (INF) top = max_abs_nan(top, v);
    else sum += static_cast<double>(v) * v;
  }
};

// The CTA's total in thread 0, in a fixed order.
template <bool INF>
__device__ __forceinline__ double cta_total(double sum, float top) {
  __shared__ double red[kThreads / 32];
  double v = INF ? static_cast<double>(top) : sum;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double w = __shfl_xor_sync(0xffffffffu, v, o);
    v = INF ? ((v != v || w != w) ? v + w : (v > w ? v : w)) : v + w;
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) {
    const double w = red[i];
    v = INF ? ((v != v || w != w) ? v + w : (v > w ? v : w)) : v + w;
  }
  return v;
}

// Elements before the first 16-byte boundary of an array of `size`-byte elements, at most n.
__device__ __forceinline__ int64_t head_elements(uint64_t address, int size, int64_t n) {
  const int64_t h = static_cast<int64_t>((16u - (address & 15u)) & 15u) / size;
  return h < n ? h : n;
}

__device__ __forceinline__ int elem_size(int dtype) { return dtype == MUZO_F32 ? 4 : 2; }

template <bool INF, int DTYPE>
__device__ __forceinline__ void norm_chunk(const char* base, int64_t n, Total<INF>& total) {
  constexpr int size = DTYPE == MUZO_F32 ? 4 : 2, V = 16 / size, sweep = kThreads * V;
  const int64_t head = head_elements(reinterpret_cast<uint64_t>(base), size, n);
  if (threadIdx.x < head) total.add(load_elem(base, threadIdx.x, DTYPE));
  const char* body = base + head * size;
  const int64_t m = n - head;
  int64_t i = threadIdx.x * V;
  for (; i + 3 * sweep + V <= m; i += 4 * sweep) {   // four loads in flight per thread
    float v[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) load_vec<DTYPE, false>(body + (i + u * sweep) * size, v[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) total.add_vec(v[u]);
  }
  for (; i + V <= m; i += sweep) {
    float v[V];
    load_vec<DTYPE, false>(body + i * size, v);
    total.add_vec(v);
  }
  for (; i < m; ++i) total.add(load_elem(body, i, DTYPE));   // the one thread whose V straddle the end
}

template <int N, bool INF>
__global__ void __launch_bounds__(kThreads, kNormPerSm) grad_norm_kernel(const __grid_constant__ Table<N> t, double* partial) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Total<INF> total;
  const uint32_t chunks = t.first[t.count];
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find_tensor(t, c);
    int64_t begin, end;
    chunk_range(t, i, c, begin, end);
    const int dtype = static_cast<int>((t.numel[i] >> 56) & 15);
    const char* base = reinterpret_cast<const char*>(t.src[i]) + begin * elem_size(dtype);
    if (dtype == MUZO_BF16) norm_chunk<INF, MUZO_BF16>(base, end - begin, total);
    else if (dtype == MUZO_F16) norm_chunk<INF, MUZO_F16>(base, end - begin, total);
    else norm_chunk<INF, MUZO_F32>(base, end - begin, total);
  }
  const double v = cta_total<INF>(total.sum, total.top);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

// The norm from the partial sums, the same value in every thread of every CTA.
template <bool INF>
__device__ __forceinline__ float total_norm(const double* partial, int count) {
  double sum = 0.0;
  float top = 0.0f;
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const double v = partial[i];
    if (INF) top = max_abs_nan(top, static_cast<float>(v));
    else sum += v;
  }
  const double v = cta_total<INF>(sum, top);
  return static_cast<float>(INF ? v : sqrt(v));
}

template <bool INF>
__global__ void __launch_bounds__(kThreads) grad_norm_finish_kernel(const double* partial, int count, float* norm) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float v = total_norm<INF>(partial, count);
  if (threadIdx.x == 0) *norm = v;
}

// out = dst dtype(factor * g) of one chunk; vector path where source and destination can both be
// accessed in whole vectors from the same element on. A vector has 16 bytes of the wider type, so that
// a warp's stores are contiguous (with 8 elements to fp32, each store instruction wrote half of every
// 32-byte sector it touched: 4.8 TB/s over six Llama-3-8B-shaped layers).
template <int SRC, int DST>
__device__ __forceinline__ void scale_chunk(const char* src, char* dst, int64_t n, float f) {
  constexpr int ss = SRC == MUZO_F32 ? 4 : 2, ds = DST == MUZO_F32 ? 4 : 2;
  constexpr int V = DST == MUZO_F32 ? 4 : 8, U = 16 / ss * 4 / V, sweep = kThreads * V;   // U loads: 64 bytes
  int64_t head = head_elements(reinterpret_cast<uint64_t>(dst), ds, n);
  if (((reinterpret_cast<uint64_t>(src) + head * ss) & (V * ss - 1)) != 0) {
    for (int64_t i = threadIdx.x; i < n; i += kThreads) store_elem(dst, i, DST, load_elem(src, i, SRC) * f);
    return;
  }
  if (threadIdx.x < head) store_elem(dst, threadIdx.x, DST, load_elem(src, threadIdx.x, SRC) * f);
  src += head * ss;
  dst += head * ds;
  const int64_t m = n - head;
  int64_t i = threadIdx.x * V;
  for (; i + (U - 1) * sweep + V <= m; i += U * sweep) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<SRC>(src + (i + u * sweep) * ss, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[u][k] *= f;
      store_vec<DST>(dst + (i + u * sweep) * ds, v[u]);
    }
  }
  for (; i + V <= m; i += sweep) {
    float v[V];
    load_vec<SRC>(src + i * ss, v);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] *= f;
    store_vec<DST>(dst + i * ds, v);
  }
  for (; i < m; ++i) store_elem(dst, i, DST, load_elem(src, i, SRC) * f);
}

template <int N, bool INF>
__global__ void __launch_bounds__(kThreads, kScalePerSm)
grad_scale_kernel(const __grid_constant__ Table<N> t, const double* partial, int count, float max_norm, float* norm) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float total = total_norm<INF>(partial, count);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm != nullptr) *norm = total;
  float f = __fdiv_rn(max_norm, __fadd_rn(total, 1e-6f));
  if (f > 1.0f) f = 1.0f;   // a NaN norm stays NaN and reaches every gradient
  const uint32_t chunks = t.first[t.count];
  for (uint32_t at = blockIdx.x; at < chunks; at += gridDim.x) {
    const uint32_t c = chunks - 1 - at;   // backwards: the norm's last reads may still be in L2
    const int i = find_tensor(t, c);
    const int kinds = static_cast<int>(t.numel[i] >> 56);
    const int s = kinds & 15, d = kinds >> 4;
    if (f == 1.0f && t.src[i] == t.dst[i]) continue;   // in place and nothing to scale
    int64_t begin, end;
    chunk_range(t, i, c, begin, end);
    const char* src = reinterpret_cast<const char*>(t.src[i]) + begin * elem_size(s);
    char* dst = reinterpret_cast<char*>(t.dst[i]) + begin * elem_size(d);
    const int64_t n = end - begin;
    if (s == MUZO_BF16) {
      if (d == MUZO_BF16) scale_chunk<MUZO_BF16, MUZO_BF16>(src, dst, n, f);
      else scale_chunk<MUZO_BF16, MUZO_F32>(src, dst, n, f);
    } else if (s == MUZO_F16) {
      if (d == MUZO_F16) scale_chunk<MUZO_F16, MUZO_F16>(src, dst, n, f);
      else scale_chunk<MUZO_F16, MUZO_F32>(src, dst, n, f);
    } else {
      scale_chunk<MUZO_F32, MUZO_F32>(src, dst, n, f);
    }
  }
}

// ---------------------------------------------------------------- host

struct Call {
  const uint64_t* src;
  const uint64_t* dst;      // null: the norm alone
  const int64_t* numel;
  const int32_t* src_dtype;
  const int32_t* dst_dtype;
  int64_t count;
};

// Sweeps per chunk: as many as keep every CTA of a launch busy, at most 8 (16 K elements).
int chunk_shift(int64_t elements) {
  int shift = 11;   // one sweep
  while (shift < 14 && (elements >> (shift + 1)) >= 4 * kMaxCtas) ++shift;
  return shift;
}

// Launch that may begin before its predecessor on the stream has ended: the kernel waits for it
// (griddepcontrol.wait) before it reads what that one wrote.
int launch_dependent(const void* kernel, unsigned grid, cudaStream_t s, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  MUZO_CUDA_CHECK(cudaLaunchKernelExC(&cfg, kernel, args));
  count_launches(1);
  return MUZO_OK;
}

// Fills the table with non-empty tensors from `at` on; returns the index behind the last one.
template <int N>
int64_t fill(Table<N>& t, const Call& c, int64_t at, int shift, uint32_t& chunks) {
  t.count = 0;
  t.chunk_shift = shift;
  uint64_t n = 0;
  for (; at < c.count && t.count < N; ++at) {
    if (c.numel[at] == 0) continue;
    const uint64_t more = (static_cast<uint64_t>(c.numel[at]) + (1ull << shift) - 1) >> shift;
    if (n + more > 0x7fffffffull) break;   // refused for a single tensor by the caller's check
    t.src[t.count] = c.src[at];
    t.dst[t.count] = c.dst ? c.dst[at] : 0;
    t.numel[t.count] = static_cast<uint64_t>(c.numel[at]) | static_cast<uint64_t>(c.src_dtype[at]) << 56 |
                       static_cast<uint64_t>(c.dst ? c.dst_dtype[at] : 0) << 60;
    t.first[t.count] = static_cast<uint32_t>(n);
    n += more;
    ++t.count;
  }
  t.first[t.count] = static_cast<uint32_t>(n);
  chunks = static_cast<uint32_t>(n);
  return at;
}

template <int N, bool INF>
int run(const Call& c, int shift, float max_norm, double* partial, float* norm, cudaStream_t s) {
  Table<N> t;
  int64_t at = 0;
  int sums = 0;
  while (at < c.count) {
    uint32_t chunks = 0;
    at = fill(t, c, at, shift, chunks);
    if (chunks == 0) continue;
    const unsigned grid = chunks < kMaxCtas ? chunks : kMaxCtas;
    double* mine = partial + sums;
    void* args[] = {&t, &mine};
    MUZO_CUDA_CHECK(cudaLaunchKernel(reinterpret_cast<const void*>(grad_norm_kernel<N, INF>), dim3(grid), dim3(kThreads),
                                     args, 0, s));
    count_launches(1);
    sums += static_cast<int>(grid);
  }
  if (c.dst == nullptr || sums == 0) {
    void* args[] = {&partial, &sums, &norm};
    return launch_dependent(reinterpret_cast<const void*>(grad_norm_finish_kernel<INF>), 1, s, args);
  }
  for (at = 0; at < c.count;) {
    uint32_t chunks = 0;
    at = fill(t, c, at, shift, chunks);
    if (chunks == 0) continue;
    const unsigned grid = chunks < 148 * kScalePerSm ? chunks : 148 * kScalePerSm;
    void* args[] = {&t, &partial, &sums, &max_norm, &norm};
    const int st = launch_dependent(reinterpret_cast<const void*>(grad_scale_kernel<N, INF>), grid, s, args);
    if (st != MUZO_OK) return st;
    norm = nullptr;   // written by the first launch
  }
  return MUZO_OK;
}

int check_call(const Call& c, bool clip) {
  if (c.count < 0 || (c.count > 0 && (c.src == nullptr || c.numel == nullptr || c.src_dtype == nullptr))) return MUZO_ERR_ARG;
  if (clip && c.count > 0 && (c.dst == nullptr || c.dst_dtype == nullptr)) return MUZO_ERR_ARG;
  for (int64_t i = 0; i < c.count; ++i) {
    if (c.numel[i] < 0) return MUZO_ERR_ARG;
    const int s = c.src_dtype[i];
    if (s != MUZO_F32 && s != MUZO_BF16 && s != MUZO_F16) return MUZO_ERR_DTYPE;
    if (clip && c.dst_dtype[i] != s && c.dst_dtype[i] != MUZO_F32) return MUZO_ERR_DTYPE;
    if (c.numel[i] == 0) continue;
    if (c.numel[i] > (1ll << 40)) return MUZO_ERR_UNSUPPORTED;
    if (c.src[i] == 0 || (clip && c.dst[i] == 0)) return MUZO_ERR_ARG;
    if (c.src[i] % (s == MUZO_F32 ? 4 : 2) != 0 || (clip && c.dst[i] % (c.dst_dtype[i] == MUZO_F32 ? 4 : 2) != 0))
      return MUZO_ERR_ALIGN;
  }
  return MUZO_OK;
}

// Whether anything that is written overlaps anything else that is written or read (a tensor scaled
// in place overlaps only itself).
int check_overlap(const Call& c) {
  struct Span { uint64_t a, z; int64_t tensor; bool written; };
  std::vector<Span> spans;
  spans.reserve(2 * c.count);
  for (int64_t i = 0; i < c.count; ++i) {
    const uint64_t n = static_cast<uint64_t>(c.numel[i]);
    if (n == 0) continue;
    const uint64_t dz = c.dst[i] + n * (c.dst_dtype[i] == MUZO_F32 ? 4 : 2);
    spans.push_back({c.dst[i], dz, i, true});
    if (c.src[i] != c.dst[i] || c.src_dtype[i] != c.dst_dtype[i])
      spans.push_back({c.src[i], c.src[i] + n * (c.src_dtype[i] == MUZO_F32 ? 4 : 2), i, false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
  uint64_t any = 0, written = 0;   // furthest end so far, of all spans and of the written ones
  for (const Span& s : spans) {
    if (s.a < written || (s.written && s.a < any)) return MUZO_ERR_ARG;
    any = std::max(any, s.z);
    if (s.written) written = std::max(written, s.z);
  }
  return MUZO_OK;
}

int64_t launches_needed(int64_t count, int64_t elements) {
  // every launch but the last is full: kLargeTable tensors, or 2^31 chunks less one tensor's
  return count / kLargeTable + 2 + (elements >> 40);
}

int dispatch(const Call& c, bool inf, float max_norm, float* d_norm, void* ws, int64_t ws_bytes, cudaStream_t s) {
  int64_t elements = 0, used = 0;
  for (int64_t i = 0; i < c.count; ++i) {
    elements += c.numel[i];
    used += c.numel[i] > 0;
  }
  if (ws_bytes < launches_needed(c.count, elements) * kMaxCtas * 8) return MUZO_ERR_CAPACITY;
  double* partial = static_cast<double*>(ws);
  const int shift = chunk_shift(elements);
  if (used <= kSmallTable)
    return inf ? run<kSmallTable, true>(c, shift, max_norm, partial, d_norm, s)
               : run<kSmallTable, false>(c, shift, max_norm, partial, d_norm, s);
  return inf ? run<kLargeTable, true>(c, shift, max_norm, partial, d_norm, s)
             : run<kLargeTable, false>(c, shift, max_norm, partial, d_norm, s);
}

}  // namespace
}  // namespace muzo

using namespace muzo;

extern "C" {

int64_t muzo_grad_workspace(int64_t count, int64_t elements) {
  if (count < 0 || elements < 0) return -1;
  return launches_needed(count, elements) * kMaxCtas * 8;
}

int muzo_grad_norm(const uint64_t* src, const int64_t* numel, const int32_t* dtype, int64_t count, int inf_norm,
                   float* d_norm, void* d_workspace, int64_t workspace_bytes, void* stream) {
  const Call c = {src, nullptr, numel, dtype, nullptr, count};
  const int st = check_call(c, false);
  if (st != MUZO_OK) return st;
  if (d_norm == nullptr || d_workspace == nullptr) return MUZO_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(d_workspace) & 7u) != 0) return MUZO_ERR_ALIGN;
  return dispatch(c, inf_norm != 0, 0.0f, d_norm, d_workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int muzo_grad_clip(const uint64_t* src, const uint64_t* dst, const int64_t* numel, const int32_t* src_dtype,
                   const int32_t* dst_dtype, int64_t count, int inf_norm, float max_norm, float* d_norm,
                   void* d_workspace, int64_t workspace_bytes, void* stream) {
  const Call c = {src, dst, numel, src_dtype, dst_dtype, count};
  int st = check_call(c, true);
  if (st != MUZO_OK) return st;
  if (d_norm == nullptr || d_workspace == nullptr || !(max_norm >= 0.0f)) return MUZO_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(d_workspace) & 7u) != 0) return MUZO_ERR_ALIGN;
  try {
    st = check_overlap(c);
  } catch (const std::bad_alloc&) {
    return MUZO_ERR_CAPACITY;
  }
  if (st != MUZO_OK) return st;
  return dispatch(c, inf_norm != 0, max_norm, d_norm, d_workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
