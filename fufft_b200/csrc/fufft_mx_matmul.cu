// fufft_mx_matmul.cu -- product of two 4-bit microscaled matrices,
// out[m][n] = sum_k a[m][k] b[n][k] + bias[n], summed in fp32.
#include "fufft_internal.cuh"
#include "fufft_mx.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace mx {

struct MatmulArgs {
   const uint8_t *a, *a_scale, *b, *b_scale;
   const float* bias;
   void* out;
   long long m, n, k, out_stride;
};

// 64 x 64 outputs per CTA, 4 x 4 per thread, one block of 32 k at a time
template<class T>
__global__ void __launch_bounds__(256) matmul_kernel(MatmulArgs g)
{
   __shared__ float as[BLOCK][65], bs[BLOCK][65];
   const long long tiles_n = ceil_div(g.n, 64);
   const long long m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
   const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
   const int line = threadIdx.x >> 2, part = threadIdx.x & 3;
   float acc[4][4] = {};
   for(long long k0 = 0; k0 < g.k; k0 += BLOCK) {
#pragma unroll
      for(int side = 0; side < 2; ++side) {
         const long long row = (side ? n0 : m0) + line, rows = side ? g.n : g.m;
         const uint8_t* codes = side ? g.b : g.a;
         const uint8_t* scales = side ? g.b_scale : g.a_scale;
         float v[8] = {};
         if(row < rows) {
            const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + row * mx4_pitch(g.k) + k0 / 2 + part * 4);
            const long long tile = (row / TILE_ROWS) * mx4_scale_tiles(g.k) + k0 / 128;
            const float s = scale_value(scales[tile * TILE_BYTES + tile_word((int)(row % TILE_ROWS)) + (k0 / BLOCK) % 4]);
            Elem<false>::decode8(&q, v);
#pragma unroll
            for(int i = 0; i < 8; ++i) v[i] *= s;
         }
#pragma unroll
         for(int i = 0; i < 8; ++i) (side ? bs : as)[part * 8 + i][line] = v[i];
      }
      __syncthreads();
#pragma unroll 8
      for(int k = 0; k < BLOCK; ++k) {
         float a[4], b[4];
#pragma unroll
         for(int i = 0; i < 4; ++i) {
            a[i] = as[k][ty * 4 + i];
            b[i] = bs[k][tx * 4 + i];
         }
#pragma unroll
         for(int i = 0; i < 4; ++i)
#pragma unroll
            for(int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
      }
      __syncthreads();
   }
#pragma unroll
   for(int i = 0; i < 4; ++i)
#pragma unroll
      for(int j = 0; j < 4; ++j) {
         const long long m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
         if(m < g.m && n < g.n)
            static_cast<T*>(g.out)[m * g.out_stride + n] = from_f<T>(acc[i][j] + (g.bias ? g.bias[n] : 0.0f));
      }
}

}  // namespace mx
}  // namespace fufft

extern "C" {

fufft_status fufft_mx4_matmul(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                              const uint8_t* b_scales, const float* bias, void* out, fufft_dtype dtype, int64_t m,
                              int64_t n, int64_t k, int64_t out_stride, fufft_stream_t stream)
{
   constexpr int64_t MAX = 1ll << 30;
   if(dtype < FUFFT_F32 || dtype > FUFFT_BF16) return FUFFT_ERR_INVALID_ARG;
   if(m < 0 || n < 0 || k < 0 || m > MAX || n > MAX || k > MAX) return FUFFT_ERR_INVALID_SIZE;
   if(m == 0 || n == 0) return FUFFT_OK;
   if(mx::ceil_div(m, 64) > 0x7fffffffll / mx::ceil_div(n, 64)) return FUFFT_ERR_INVALID_SIZE;
   if(!out || (k && (!a_codes || !a_scales || !b_codes || !b_scales)) || (m > 1 && out_stride < n)) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(a_codes, 16) || !aligned(a_scales, 16) || !aligned(b_codes, 16) || !aligned(b_scales, 16) ||
      !aligned(bias, 4) || !aligned(out, dtype == FUFFT_F32 ? 4 : 2))
      return FUFFT_ERR_MISALIGNED;
   mx::MatmulArgs g{a_codes, a_scales, b_codes, b_scales, bias, out, m, n, k, out_stride};
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   const unsigned grid = (unsigned)(mx::ceil_div(m, 64) * mx::ceil_div(n, 64));
   switch(dtype) {
   case FUFFT_F32: mx::matmul_kernel<float><<<grid, 256, 0, st>>>(g); break;
   case FUFFT_F16: mx::matmul_kernel<__half><<<grid, 256, 0, st>>>(g); break;
   default: mx::matmul_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(g); break;
   }
   count_launch();
   return check(cudaGetLastError());
}

}  // extern "C"
