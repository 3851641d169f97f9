// What the attention forward and backward kernels share: tile sizes, the exponential, the range of
// keys a batch row attends to, and the tensor map of a [B][H][S][D] operand.
#pragma once

#include "tcgen05_common.cuh"

namespace muzo {
namespace attn {

constexpr int AM = 128;          // rows of a query tile (UMMA M)
constexpr int AN = 128;          // keys of a key tile
constexpr int ABK = 64;          // 128-byte swizzle row of 16-bit elements
constexpr int SUB_BYTES = 128 * ABK * 2;     // one swizzled block of 128 rows x 64 elements (16 KB)

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in one instruction of the FMA pipe, each rounded once as its scalar form is:
// x = x * a + (b0, b1), x += y, x *= y.
__device__ __forceinline__ void fma_pair(float& x0, float& x1, float a, float b0, float b1) {
  asm("{\n\t.reg .b64 x, a, b;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 a, {%2, %2};\n\t"
      "mov.b64 b, {%3, %4};\n\t"
      "fma.rn.f32x2 x, x, a, b;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(a), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add_pair(float& x0, float& x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(y0), "f"(y1));
}
__device__ __forceinline__ void mul_pair(float& x0, float& x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\t"
      "mov.b64 y, {%2, %3};\n\t"
      "mul.rn.f32x2 x, x, y;\n\t"
      "mov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1)
      : "f"(y0), "f"(y1));
}

// Visible keys [lo, hi) of batch row b, clamped to the sequence.
__device__ __forceinline__ void key_range(const int32_t* key_lo, const int32_t* key_hi, int64_t sk, int b, int64_t& lo,
                                          int64_t& hi) {
  lo = key_lo ? key_lo[b] : 0;
  hi = key_hi ? key_hi[b] : sk;
  if (lo < 0) lo = 0;
  if (hi > sk) hi = sk;
}

// Rows [row0, row0 + rows) of a head's [S][hd] 16-bit result, as far as they exist, become NaN (0x7fff is one in
// bf16 and in fp16). Called by all threads of a CTA.
__device__ __forceinline__ void lose_tile(uint16_t* head, int64_t stride, int64_t row0, int rows, int64_t s, int hd) {
  const int pieces = hd / 8;   // of 16 bytes
  for (int i = threadIdx.x; i < rows * pieces; i += blockDim.x) {
    const int64_t row = row0 + i / pieces;
    if (row < s)
      *reinterpret_cast<uint4*>(head + row * stride + 8 * (i % pieces)) =
          make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  }
}

// 4-D tensor map over [B][H][S][D] (element strides ss, sh, sb; D contiguous), box 64 x rows. A
// head dimension below the box's 64 or 128 columns reads zeros behind its end.
inline int encode_attn_map(CUtensorMap* map, const void* base, int dtype, int64_t d, int64_t s, int64_t h, int64_t b,
                           int64_t ss, int64_t sh, int64_t sb, int rows) {
  auto fn = tc::encode_fn();
  if (fn == nullptr) return MUZO_ERR_UNSUPPORTED;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(s), static_cast<cuuint64_t>(h),
                        static_cast<cuuint64_t>(b)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(ss * 2), static_cast<cuuint64_t>(sh * 2),
                           static_cast<cuuint64_t>(sb * 2)};
  cuuint32_t box[4] = {ABK, static_cast<cuuint32_t>(rows), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType dt = dtype == MUZO_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUresult res = fn(map, dt, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return res == CUDA_SUCCESS ? MUZO_OK : MUZO_ERR_ARG;
}

inline bool aligned16p(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace attn
}  // namespace muzo
