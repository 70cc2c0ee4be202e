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

#include <type_traits>

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
// tiled tensor map with unit element strides and zero fill; FUFFT_ERR_UNSUPPORTED where the driver refuses it
fufft_status encode_tmap(CUtensorMap* tm, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                         const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle);
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

// 32-byte transfers (p 32-byte aligned)
__device__ __forceinline__ void load32(const void* p, uint32_t* w)
{
   asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w)
{
   asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                :: "l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// |x| as bits: they order like the values, an infinity above every number and
// a NaN above an infinity, so an integer maximum keeps both
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// |x| as bits of the largest of N values as they lie in memory, three words an
// instruction; of 16-bit values two maxima, in the halves of a word.  The
// signed maximum is the largest of those without a sign bit, the unsigned one
// the largest of those with it (if there are any): no bit has to be masked on
// the way.  fp32 has an instruction for the maximum of magnitudes that keeps NaN.
template<class T, int N> __device__ __forceinline__ uint32_t max_words(const uint32_t* w)
{
   static_assert(N % 2 == 0, "the first, pairs, the last");
   if constexpr(sizeof(T) == 4) {
      float m = __uint_as_float(w[0]);
#pragma unroll
      for(int i = 1; i + 1 < N; i += 2)
         asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(__uint_as_float(w[i])), "f"(__uint_as_float(w[i + 1])));
      asm("max.NaN.abs.f32 %0, %0, %1, %1;" : "+f"(m) : "f"(__uint_as_float(w[N - 1])));
      return __float_as_uint(m) & 0x7fffffffu;
   } else {
      uint32_t p = w[0], n = w[0];
#pragma unroll
      for(int i = 1; i + 1 < N; i += 2) {
         p = __vimax3_s16x2(p, w[i], w[i + 1]);
         n = __vimax3_u16x2(n, w[i], w[i + 1]);
      }
      p = __vimax3_s16x2(p, p, w[N - 1]);
      n = __vimax3_u16x2(n, n, w[N - 1]);
      return __vimax3_s16x2(p, p, n & 0x7fff7fffu);
   }
}
// the two values of w, each times its power of two.  A bfloat16 holds every
// power of two that scale_inverse returns, and one mixed fma widens and
// multiplies a half, exactly; minus zero is what keeps the sign of a zero
template<class T> __device__ __forceinline__ void scaled_pair(uint32_t w, float2 factor, float* a, float* b)
{
   if constexpr(std::is_same<T, __nv_bfloat16>::value) {
      asm("{\n\t.reg .b16 lo, hi, f0, f1, z;\n\tmov.b32 {lo, hi}, %2;\n\tmov.b32 {z, f0}, %3;\n\tmov.b32 {z, f1}, %4;\n\t"
          "fma.rn.f32.bf16 %0, lo, f0, %5;\n\tfma.rn.f32.bf16 %1, hi, f1, %5;\n\t}"
          : "=f"(*a), "=f"(*b) : "r"(w), "r"(__float_as_uint(factor.x)), "r"(__float_as_uint(factor.y)), "f"(-0.0f));
   } else {
      const float2 f = fmul2(unpack2<T>(w), factor);
      *a = f.x;
      *b = f.y;
   }
}

// Sixteen consecutive values as they lie in memory: half a block, the unit of
// the format kernels (two neighbouring lanes a block).
constexpr int HALF = 16;
template<class T> struct Half {
   static constexpr int WORDS = HALF * (int)sizeof(T) / 4;
   uint32_t w[WORDS];
   // all sixteen, p on 32 bytes
   __device__ __forceinline__ void load(const T* p)
   {
#pragma unroll
      for(int i = 0; i < WORDS / 8; ++i) load32(reinterpret_cast<const uint8_t*>(p) + 32 * i, w + 8 * i);
   }
   __device__ __forceinline__ void store(T* p) const
   {
#pragma unroll
      for(int i = 0; i < WORDS / 8; ++i) store32(reinterpret_cast<uint8_t*>(p) + 32 * i, w + 8 * i);
   }
   // the first `count`, anywhere; zeros after them
   __device__ __forceinline__ void load_some(const T* p, int count)
   {
#pragma unroll
      for(int i = 0; i < WORDS; ++i) {
         if constexpr(sizeof(T) == 4) {
            w[i] = i < count ? __float_as_uint(p[i]) : 0u;
         } else {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
            w[i] = (2 * i < count ? (uint32_t)q[2 * i] : 0u) | (2 * i + 1 < count ? (uint32_t)q[2 * i + 1] << 16 : 0u);
         }
      }
   }
   __device__ __forceinline__ void store_some(T* p, int count) const
   {
#pragma unroll
      for(int i = 0; i < WORDS; ++i) {
         if constexpr(sizeof(T) == 4) {
            if(i < count) p[i] = __uint_as_float(w[i]);
         } else {
            uint16_t* q = reinterpret_cast<uint16_t*>(p);
            if(2 * i < count) q[2 * i] = (uint16_t)w[i];
            if(2 * i + 1 < count) q[2 * i + 1] = (uint16_t)(w[i] >> 16);
         }
      }
   }
   __device__ __forceinline__ void zero()
   {
#pragma unroll
      for(int i = 0; i < WORDS; ++i) w[i] = 0;
   }
   // maximum of abs_bits
   __device__ __forceinline__ uint32_t max_bits() const
   {
      const uint32_t m = max_words<T, WORDS>(w);
      if constexpr(sizeof(T) == 4) return m;
      else return abs_bits(unpack2<T>(max(m >> 16, m & 0xffffu)).x);
   }
   // the values times a power of two
   __device__ __forceinline__ void scaled(float factor, float* v) const
   {
#pragma unroll
      for(int i = 0; i < HALF / 2; ++i) {
         if constexpr(sizeof(T) == 4) {
            const float2 f = fmul2(make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1])), make_float2(factor, factor));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
         } else {
            scaled_pair<T>(w[i], make_float2(factor, factor), v + 2 * i, v + 2 * i + 1);
         }
      }
   }
   __device__ __forceinline__ void set(const float* v)
   {
#pragma unroll
      for(int i = 0; i < WORDS; ++i) {
         if constexpr(sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
         else w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
      }
   }
};

// scale byte of a block from the maximum of abs_bits
template<int EMAX> __device__ __forceinline__ uint32_t scale_byte(uint32_t max_bits)
{
   const int e = (int)(max_bits >> 23);
   return e == 255 ? 255u : (uint32_t)max(e - EMAX, 0);
}
// 2^(127 - s) (s <= 252, or a NaN block's, for which any will do)
__device__ __forceinline__ float scale_inverse(uint32_t s) { return __uint_as_float((254u - s) << 23); }
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

// the two element formats; sixteen codes are WORDS words
template<bool MX8> struct Elem;
template<> struct Elem<false> {
   static constexpr int EMAX = 2, WORDS = 2;
   __device__ static __forceinline__ void encode(const float* v, uint32_t* w)
   {
      w[0] = e2m1_encode8(v);
      w[1] = e2m1_encode8(v + 8);
   }
   __device__ static __forceinline__ void halves(const uint32_t* w, uint32_t* h)
   {
      e2m1_decode8(w[0], h);
      e2m1_decode8(w[1], h + 4);
   }
};
template<> struct Elem<true> {
   static constexpr int EMAX = 8, WORDS = 4;
   __device__ static __forceinline__ void encode(const float* v, uint32_t* w)
   {
#pragma unroll
      for(int i = 0; i < 4; ++i) w[i] = e4m3_encode4(v + 4 * i);
   }
   __device__ static __forceinline__ void halves(const uint32_t* w, uint32_t* h)
   {
#pragma unroll
      for(int i = 0; i < 4; ++i) e4m3_decode4(w[i], h + 2 * i);
   }
};
// sixteen codes -> values times `scale`
template<bool MX8> __device__ __forceinline__ void decode(const uint32_t* w, float scale, float* v)
{
   uint32_t h[8];
   Elem<MX8>::halves(w, h);
#pragma unroll
   for(int i = 0; i < 8; ++i) {
      const float2 f = fmul2(half2_f(h[i]), make_float2(scale, scale));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
   }
}
// 8 (MX4) or 16 (MX8) bytes of codes
template<int WORDS> __device__ __forceinline__ void load_codes(const uint8_t* p, uint32_t* w)
{
   if constexpr(WORDS == 4) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
   } else {
      const uint2 q = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = q.x; w[1] = q.y;
   }
}
template<int WORDS> __device__ __forceinline__ void store_codes(uint8_t* p, const uint32_t* w)
{
   if constexpr(WORDS == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
   else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

// A block in two neighbouring lanes, sixteen values each (all 32 lanes take
// part): its scale byte, and the lane's codes.
template<bool MX8, class T> __device__ __forceinline__ uint32_t encode_pair(const Half<T>& h, uint32_t* w)
{
   uint32_t m = h.max_bits();
   m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
   const uint32_t s = scale_byte<Elem<MX8>::EMAX>(m);
   const float inv = scale_inverse(s);
   float v[HALF];
   h.scaled(inv, v);
   Elem<MX8>::encode(v, w);
   if(s == 255u) {   // zero codes under a NaN scale
#pragma unroll
      for(int i = 0; i < Elem<MX8>::WORDS; ++i) w[i] = 0;
   }
   return s;
}

}  // namespace mx
}  // namespace fufft
