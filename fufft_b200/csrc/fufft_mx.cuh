// fufft_mx.cuh -- microscaled (block floating point) element formats shared by
// the 4-bit matrix and the sequence-cache kernels.
//
// A block is 32 consecutive values with one power-of-two scale 2^(s - 127)
// held as the byte s (E8M0; 255 = NaN).  For elements whose largest binade is
// emax, s - 127 = floor(log2 max|x|) - emax, not below -127, and an element is
// x / 2^(s - 127) rounded to nearest even, saturating at the format's largest
// value:
//   E2M1 (4 bits):  0 .5 1 1.5 2 3 4 6, sign in bit 3, emax 2
//   E4M3 (8 bits):  up to 448, sign in bit 7, emax 8
// A block that holds an infinity or a NaN gets s = 255: all of it reads as NaN
// (E2M1 has neither, and a saturated infinity would pass for a value).
// The division by the scale is an exact multiplication by 2^(127 - s) unless
// the quotient is subnormal, which rounds to a zero code either way, so the
// codes do not depend on the order of anything: the same input gives the same
// bits everywhere.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fufft_internal.cuh"

namespace fufft {
namespace host {
// lets `kern` use `bytes` of dynamic shared memory on the current device, once per device (a bit of `done` each)
template<class K> fufft_status allow_smem(K kern, int bytes, std::atomic<uint64_t>& done)
{
   int dev = 0;
   fufft_status s = check(cudaGetDevice(&dev));
   if(s != FUFFT_OK) return s;
   const uint64_t bit = 1ull << (dev & 63);
   if(done.load(std::memory_order_acquire) & bit) return FUFFT_OK;
   s = check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
   if(s == FUFFT_OK) done.fetch_or(bit, std::memory_order_acq_rel);
   return s;
}
}  // namespace host
namespace mx {

constexpr int BLOCK = 32;         // values per scale
constexpr int K_PAD = 256;        // columns of a 4-bit matrix are padded to this
constexpr int TILE_ROWS = 128;    // a scale tile: 128 rows x 4 blocks, 512 bytes
constexpr int TILE_BYTES = 512;

__host__ __device__ inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
__host__ __device__ inline long long mx4_pitch(long long cols) { return ceil_div(cols, K_PAD) * (K_PAD / 2); }
__host__ __device__ inline long long mx4_scale_tiles(long long cols) { return ceil_div(cols, K_PAD) * 2; }
// byte of the scale word (4 blocks = 128 columns) of `row` inside its tile
__host__ __device__ inline int tile_word(int row) { return (row & 31) * 16 + ((row >> 5) & 3) * 4; }

template<class T> __device__ __forceinline__ float to_f(T v);
template<> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template<> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template<> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template<class T> __device__ __forceinline__ T from_f(float v);
template<> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template<> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template<> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two values rounded to T in one register
template<class T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template<> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b)
{
   const __half2 h = __floats2half2_rn(a, b);
   return *reinterpret_cast<const uint32_t*>(&h);
}
template<> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b)
{
   const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
   return *reinterpret_cast<const uint32_t*>(&h);
}
template<class T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template<> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w)
{
   return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template<> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w)
{
   return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// eight consecutive values; vec: p is 16-byte aligned and all eight exist
template<class T> __device__ __forceinline__ void load8(const T* p, bool vec, int count, float* v)
{
   if(vec) {
      if constexpr(sizeof(T) == 4) {
         const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
         v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
         v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
         const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
         const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
         for(int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
         }
      }
      return;
   }
#pragma unroll
   for(int i = 0; i < 8; ++i) v[i] = i < count ? to_f(p[i]) : 0.0f;
}
template<class T> __device__ __forceinline__ void store8(T* p, bool vec, int count, const float* v)
{
   if(vec) {
      if constexpr(sizeof(T) == 4) {
         reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
         reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
         *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                   pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
      }
      return;
   }
#pragma unroll
   for(int i = 0; i < 8; ++i)
      if(i < count) p[i] = from_f<T>(v[i]);
}

// |x| as bits: they order like the values, an infinity above every number and
// a NaN above an infinity, so an integer maximum keeps both
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// scale byte of a block from the maximum of abs_bits
template<int EMAX> __device__ __forceinline__ uint32_t scale_byte(uint32_t max_bits)
{
   const int e = (int)(max_bits >> 23);
   return e == 255 ? 255u : (uint32_t)max(e - EMAX, 0);
}
// 2^(127 - s); 0 for a NaN block, so that its codes are zero
__device__ __forceinline__ float scale_inverse(uint32_t s) { return s == 255u ? 0.0f : __uint_as_float((254u - s) << 23); }
// 2^(s - 127); NaN for s = 255
__device__ __forceinline__ float scale_value(uint32_t s)
{
   return __uint_as_float(s == 0u ? 0x00400000u : s == 255u ? 0x7fffffffu : s << 23);
}

// eight values already divided by the scale -> eight E2M1 codes, first in the low bits
__device__ __forceinline__ uint32_t e2m1_encode8(const float* v)
{
   uint32_t r;
   asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
       "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
       "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
       "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
       : "=r"(r)
       : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
   return r;
}
// eight codes -> four half2 (exact)
__device__ __forceinline__ void e2m1_decode8(uint32_t c, uint32_t* h)
{
   asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
       "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
       "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
       : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(c));
}
__device__ __forceinline__ uint32_t e4m3_encode4(const float* v)
{
   uint16_t lo, hi;
   asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(v[0]), "f"(v[1]));
   asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(v[2]), "f"(v[3]));
   return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ void e4m3_decode4(uint32_t c, uint32_t* h)
{
   asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[0]) : "h"((uint16_t)(c & 0xffffu)));
   asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[1]) : "h"((uint16_t)(c >> 16)));
}
__device__ __forceinline__ float2 half2_f(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// the two formats a cache stores; eight codes are CODE_BYTES bytes in CODE_WORDS words
template<bool MX8> struct Elem;
template<> struct Elem<false> {
   static constexpr int EMAX = 2, WORDS = 1;
   __device__ static __forceinline__ void encode8(const float* v, uint32_t* w) { w[0] = e2m1_encode8(v); }
   __device__ static __forceinline__ void decode8(const uint32_t* w, float* v)
   {
      uint32_t h[4];
      e2m1_decode8(w[0], h);
#pragma unroll
      for(int i = 0; i < 4; ++i) {
         const float2 f = half2_f(h[i]);
         v[2 * i] = f.x;
         v[2 * i + 1] = f.y;
      }
   }
};
template<> struct Elem<true> {
   static constexpr int EMAX = 8, WORDS = 2;
   __device__ static __forceinline__ void encode8(const float* v, uint32_t* w)
   {
      w[0] = e4m3_encode4(v);
      w[1] = e4m3_encode4(v + 4);
   }
   __device__ static __forceinline__ void decode8(const uint32_t* w, float* v)
   {
      uint32_t h[4];
      e4m3_decode4(w[0], h);
      e4m3_decode4(w[1], h + 2);
#pragma unroll
      for(int i = 0; i < 4; ++i) {
         const float2 f = half2_f(h[i]);
         v[2 * i] = f.x;
         v[2 * i + 1] = f.y;
      }
   }
};

// block of 32 spread over four neighbouring lanes, eight values each: the
// block's scale byte, in all four
template<int EMAX> __device__ __forceinline__ uint32_t block_scale4(const float* v)
{
   uint32_t m = 0;
#pragma unroll
   for(int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
   m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
   m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
   return scale_byte<EMAX>(m);
}

}  // namespace mx
}  // namespace fufft
