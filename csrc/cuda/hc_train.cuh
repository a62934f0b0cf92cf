// What the kernels of the training step's operators share: element types, aligned pieces of rows, sums over a warp
// and a block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace hc {

enum ElementType : int { kF32 = 0, kBf16 = 1, kF16 = 2 };
inline size_t element_bytes(int type) { return type == kF32 ? 4 : 2; }
// nothing, or something that begins where elements of so many bytes may
inline bool lies_at(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// The status of the kernels of a source: 0, or 3 after a wait that ran out, kept until it is cleared.
int norm_status(int clear);
int logprob_status(int clear);
int attention_status(int clear);
template <typename S>
int take_status(S& symbol, int clear) {
  unsigned int status = 0;
  if (cudaMemcpyFromSymbol(&status, symbol, sizeof(status)) != cudaSuccess) return 5;  // kErrCuda
  const unsigned int zero = 0;
  if (clear && status && cudaMemcpyToSymbol(symbol, &zero, sizeof(zero)) != cudaSuccess) return 5;
  return (int)status;
}
inline bool element_type_ok(int type) { return type >= kF32 && type <= kF16; }

namespace dev {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

// two values of a 16-bit type in one word, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t w, float& a, float& b) {
  float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
  a = f.x;
  b = f.y;
}

// Eight neighbouring values as floats.  `p` is aligned to eight values.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  unpack2<T>(w.x, v[0], v[1]);
  unpack2<T>(w.y, v[2], v[3]);
  unpack2<T>(w.z, v[4], v[5]);
  unpack2<T>(w.w, v[6], v[7]);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  uint4 w;
  w.x = pack2<T>(v[0], v[1]);
  w.y = pack2<T>(v[2], v[3]);
  w.z = pack2<T>(v[4], v[5]);
  w.w = pack2<T>(v[6], v[7]);
  *reinterpret_cast<uint4*>(p) = w;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// Rows whose length eight does not divide start anywhere within an aligned group of eight.  A row is then worked on in
// the aligned groups that it touches: value j of group g is column 8 g + j - shift, and only the first and last group
// are taken element by element.  `row`: the row's first value; columns outside [0, width) read as 0.
template <typename T>
__device__ __forceinline__ void load_group(const T* row, int64_t first, int64_t width, float (&v)[8]) {
  if (first >= 0 && first + 8 <= width) {
    load8(row + first, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = first + j >= 0 && first + j < width ? to_float(row[first + j]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_group(T* row, int64_t first, int64_t width, const float (&v)[8]) {
  if (first >= 0 && first + 8 <= width) {
    store8(row + first, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (first + j >= 0 && first + j < width) row[first + j] = from_float<T>(v[j]);
  }
}

__device__ __forceinline__ float param_at(const void* p, int type, int64_t i) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  if (type == kBf16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void param_put(void* p, int type, int64_t i, float v) {
  if (type == kF32) static_cast<float*>(p)[i] = v;
  else if (type == kBf16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// sums of two values over T threads (a warp, or a block of T); every thread gets them
template <int T>
__device__ __forceinline__ void group_sum2(float& a, float& b, float2* shared) {
  a = warp_sum(a);
  b = warp_sum(b);
  if (T > 32) {
    __syncthreads();  // the sums of the round before have been read
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 32; ++w) {
      const float2 s = shared[w];
      a += s.x;
      b += s.y;
    }
  }
}

// Two values at a time: one instruction for both
struct Pair {
  uint64_t w;
};
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.w) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void parts(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.w)); }
__device__ __forceinline__ float both(Pair p) {
  float a, b;
  parts(p, a, b);
  return a + b;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.w) : "l"(a.w), "l"(b.w), "l"(c.w));
  return r;
}
// mma.sync: d (16 x 8) += a (16 x 16) b (16 x 8).  Lane 4g + t has of a row g, columns 2t and 2t + 1 (a0), row g + 8 (a1), columns 2t + 8 and on (a2, a3); of b column g, rows 2t (b0) and 2t + 8 (b1) and
// the next ones; of d rows g and g + 8, columns 2t and 2t + 1.
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace dev
}  // namespace hc
