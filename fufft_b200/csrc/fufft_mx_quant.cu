// fufft_mx_quant.cu -- 4-bit microscaled matrices: quantisation along the
// rows, along the columns, or both from one read, and the way back.
#include "fufft_internal.cuh"
#include "fufft_mx.cuh"
#include "fufft_tc.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace mx {

// Rows: one warp per (row, 256 columns); a lane holds eight columns, four
// lanes a block, sixteen lanes the four blocks of one scale word.  Columns
// beyond `cols` are zeros.
template<class T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, long long rows, long long cols,
                                                            long long row_stride, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales, bool vec)
{
   tc::let_next_start();
   const int lane = threadIdx.x & 31;
   const long long chunks = mx4_pitch(cols) / (K_PAD / 2);
   const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
   if(w >= rows * chunks) return;
   const long long row = w / chunks, chunk = w % chunks, c0 = chunk * K_PAD + lane * 8;
   float v[8];
   const int count = (int)max(0ll, min(8ll, cols - c0));
   load8(x + row * row_stride + c0, vec && count == 8, count, v);
   const uint32_t s = block_scale4<2>(v);
   const float inv = scale_inverse(s);
#pragma unroll
   for(int i = 0; i < 8; ++i) v[i] = s == 255u ? 0.0f : v[i] * inv;
   *reinterpret_cast<uint32_t*>(codes + row * mx4_pitch(cols) + chunk * (K_PAD / 2) + lane * 4) = e2m1_encode8(v);
   uint32_t word = s << (8 * ((lane >> 2) & 3));
   word |= __shfl_xor_sync(0xffffffffu, word, 4);
   word |= __shfl_xor_sync(0xffffffffu, word, 8);
   if((lane & 15) == 0) {
      const long long tile = (row / TILE_ROWS) * mx4_scale_tiles(cols) + chunk * 2 + (lane >> 4);
      *reinterpret_cast<uint32_t*>(scales + tile * TILE_BYTES + tile_word((int)(row % TILE_ROWS))) = word;
   }
}

// Columns (and rows, where asked): a CTA holds a tile of 128 x 128 values in
// shared memory, a thread encodes whole blocks of 32: lane = row for the row
// blocks, lane = column for the column blocks; with an odd pitch both walk
// the tile without bank conflicts.
constexpr int QT = 128;
constexpr int QT_PITCH = QT + 1;

__device__ __forceinline__ void encode_block(const float* t, int step, uint8_t* code_at, uint32_t* scale)
{
   float v[BLOCK];
   uint32_t m = 0;
#pragma unroll
   for(int i = 0; i < BLOCK; ++i) {
      v[i] = t[i * step];
      m = max(m, abs_bits(v[i]));
   }
   const uint32_t s = scale_byte<2>(m);
   const float inv = scale_inverse(s);
#pragma unroll
   for(int i = 0; i < BLOCK; ++i) v[i] = s == 255u ? 0.0f : v[i] * inv;
   *reinterpret_cast<uint4*>(code_at) =
      make_uint4(e2m1_encode8(v), e2m1_encode8(v + 8), e2m1_encode8(v + 16), e2m1_encode8(v + 24));
   *scale = s;
}

template<class T>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const T* __restrict__ x, long long rows, long long cols,
                                                            long long row_stride, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales, uint8_t* __restrict__ codes_t,
                                                            uint8_t* __restrict__ scales_t, bool vec)
{
   extern __shared__ float tile[];
   const long long ct = mx4_scale_tiles(cols), r0 = (blockIdx.x / ct) * QT, c0 = (blockIdx.x % ct) * QT;
   for(int i = threadIdx.x; i < QT * (QT / 8); i += 256) {
      const int r = i / (QT / 8), c = i % (QT / 8) * 8;
      float v[8];
      const int count = r0 + r < rows ? (int)max(0ll, min(8ll, cols - c0 - c)) : 0;
      load8(x + (r0 + r) * row_stride + c0 + c, vec && count == 8, count, v);
#pragma unroll
      for(int k = 0; k < 8; ++k) tile[r * QT_PITCH + c + k] = v[k];
   }
   __syncthreads();
   const int line = threadIdx.x & (QT - 1);
#pragma unroll
   for(int h = 0; h < 2; ++h) {
      const int b = (threadIdx.x >> 7) + 2 * h;   // block of the line
      uint32_t s;
      if(codes && r0 + line < rows) {
         encode_block(tile + line * QT_PITCH + b * BLOCK, 1,
                      codes + (r0 + line) * mx4_pitch(cols) + (c0 + b * BLOCK) / 2, &s);
         scales[(r0 / TILE_ROWS * ct + c0 / QT) * TILE_BYTES + tile_word(line) + b] = (uint8_t)s;
      }
      if(codes_t && c0 + line < cols) {
         encode_block(tile + b * BLOCK * QT_PITCH + line, QT_PITCH,
                      codes_t + (c0 + line) * mx4_pitch(rows) + (r0 + b * BLOCK) / 2, &s);
         scales_t[(c0 / TILE_ROWS * mx4_scale_tiles(rows) + r0 / QT) * TILE_BYTES + tile_word(line) + b] = (uint8_t)s;
      }
   }
}

template<class T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, long long rows,
                                                         long long cols, T* __restrict__ out, long long row_stride,
                                                         bool vec)
{
   const int lane = threadIdx.x & 31;
   const long long chunks = mx4_pitch(cols) / (K_PAD / 2);
   const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
   if(w >= rows * chunks) return;
   const long long row = w / chunks, chunk = w % chunks, c0 = chunk * K_PAD + lane * 8;
   const int count = (int)max(0ll, min(8ll, cols - c0));
   if(count == 0) return;
   const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + row * mx4_pitch(cols) + c0 / 2);
   const long long tile = (row / TILE_ROWS) * mx4_scale_tiles(cols) + chunk * 2 + (lane >> 4);
   const float s = scale_value(scales[tile * TILE_BYTES + tile_word((int)(row % TILE_ROWS)) + ((lane >> 2) & 3)]);
   float v[8];
   Elem<false>::decode8(&q, v);
#pragma unroll
   for(int i = 0; i < 8; ++i) v[i] *= s;
   store8(out + row * row_stride + c0, vec && count == 8, count, v);
}

template<class T>
fufft_status quantize(const void* x, long long rows, long long cols, long long row_stride, uint8_t* codes,
                      uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, cudaStream_t st)
{
   const T* p = static_cast<const T*>(x);
   const bool vec = aligned(x, 16) && (row_stride * (long long)sizeof(T)) % 16 == 0;
   if(!codes_t) {
      const long long warps = rows * (mx4_pitch(cols) / (K_PAD / 2));
      quantize_rows_kernel<T><<<(unsigned)ceil_div(warps, 8), 256, 0, st>>>(p, rows, cols, row_stride, codes, scales, vec);
   } else {
      constexpr int SMEM = QT * QT_PITCH * (int)sizeof(float);
      static std::atomic<uint64_t> configured{0};
      fufft_status s = allow_smem(quantize_tile_kernel<T>, SMEM, configured);
      if(s != FUFFT_OK) return s;
      const long long tiles = mx4_scale_tiles(rows) * mx4_scale_tiles(cols);
      quantize_tile_kernel<T><<<(unsigned)tiles, 256, SMEM, st>>>(p, rows, cols, row_stride, codes, scales, codes_t,
                                                                  scales_t, vec);
   }
   count_launch();
   return check(cudaGetLastError());
}

template<class T>
fufft_status dequantize(const uint8_t* codes, const uint8_t* scales, long long rows, long long cols, void* out,
                        long long row_stride, cudaStream_t st)
{
   const bool vec = aligned(out, 16) && (row_stride * (long long)sizeof(T)) % 16 == 0;
   const long long warps = rows * (mx4_pitch(cols) / (K_PAD / 2));
   dequantize_kernel<T><<<(unsigned)ceil_div(warps, 8), 256, 0, st>>>(codes, scales, rows, cols, static_cast<T*>(out),
                                                                     row_stride, vec);
   count_launch();
   return check(cudaGetLastError());
}

constexpr long long MAX_DIM = 1ll << 30;
constexpr long long MAX_ELEMENTS = 1ll << 38;   // keeps every grid below 2^31 blocks

}  // namespace mx
}  // namespace fufft

extern "C" {

size_t fufft_mx4_codes_bytes(int64_t rows, int64_t cols)
{
   return rows < 0 || cols < 0 || rows > mx::MAX_DIM || cols > mx::MAX_DIM ? 0 : (size_t)(rows * mx::mx4_pitch(cols));
}

size_t fufft_mx4_scales_bytes(int64_t rows, int64_t cols)
{
   if(rows < 0 || cols < 0 || rows > mx::MAX_DIM || cols > mx::MAX_DIM) return 0;
   return (size_t)(mx::ceil_div(rows, mx::TILE_ROWS) * mx::mx4_scale_tiles(cols) * mx::TILE_BYTES);
}

fufft_status fufft_mx4_quantize(const void* x, fufft_dtype dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                uint8_t* codes, uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t,
                                fufft_stream_t stream)
{
   if(dtype < FUFFT_F32 || dtype > FUFFT_BF16) return FUFFT_ERR_INVALID_ARG;
   if(rows < 0 || cols < 0 || rows > mx::MAX_DIM || cols > mx::MAX_DIM) return FUFFT_ERR_INVALID_SIZE;
   if(rows == 0 || cols == 0) return FUFFT_OK;
   if(rows > mx::MAX_ELEMENTS / (mx::mx4_pitch(cols) * 2)) return FUFFT_ERR_INVALID_SIZE;
   if(!x || (!codes && !codes_t) || !codes != !scales || !codes_t != !scales_t) return FUFFT_ERR_INVALID_ARG;
   if(row_stride < cols && rows > 1) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(x, dtype == FUFFT_F32 ? 4 : 2) || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(codes_t, 16) ||
      !aligned(scales_t, 16))
      return FUFFT_ERR_MISALIGNED;
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return mx::quantize<float>(x, rows, cols, row_stride, codes, scales, codes_t, scales_t, st);
   case FUFFT_F16: return mx::quantize<__half>(x, rows, cols, row_stride, codes, scales, codes_t, scales_t, st);
   default: return mx::quantize<__nv_bfloat16>(x, rows, cols, row_stride, codes, scales, codes_t, scales_t, st);
   }
}

fufft_status fufft_mx4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* out,
                                  fufft_dtype dtype, int64_t row_stride, fufft_stream_t stream)
{
   if(dtype < FUFFT_F32 || dtype > FUFFT_BF16) return FUFFT_ERR_INVALID_ARG;
   if(rows < 0 || cols < 0 || rows > mx::MAX_DIM || cols > mx::MAX_DIM) return FUFFT_ERR_INVALID_SIZE;
   if(rows == 0 || cols == 0) return FUFFT_OK;
   if(rows > mx::MAX_ELEMENTS / (mx::mx4_pitch(cols) * 2)) return FUFFT_ERR_INVALID_SIZE;
   if(!codes || !scales || !out || (row_stride < cols && rows > 1)) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(out, dtype == FUFFT_F32 ? 4 : 2) || !aligned(codes, 16) || !aligned(scales, 16)) return FUFFT_ERR_MISALIGNED;
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return mx::dequantize<float>(codes, scales, rows, cols, out, row_stride, st);
   case FUFFT_F16: return mx::dequantize<__half>(codes, scales, rows, cols, out, row_stride, st);
   default: return mx::dequantize<__nv_bfloat16>(codes, scales, rows, cols, out, row_stride, st);
   }
}

}  // extern "C"
