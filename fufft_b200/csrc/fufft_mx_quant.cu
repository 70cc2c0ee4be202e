// fufft_mx_quant.cu -- 4-bit microscaled matrices: quantisation along the
// rows, along the columns, or both from one read, and the way back.
#include <cudaTypedefs.h>

#include <mutex>

#include "fufft_internal.cuh"
#include "fufft_mx.cuh"
#include "fufft_tc.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace host {
fufft_status encode_tmap(CUtensorMap* tm, CUtensorMapDataType type, int rank, const void* base, const cuuint64_t* dims,
                         const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle)
{
   static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
   static std::once_flag once;
   std::call_once(once, [] {
      void* p = nullptr;
      cudaDriverEntryPointQueryResult q;
      if(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
         q == cudaDriverEntryPointSuccess)
         fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
   });
   if(!fn) return FUFFT_ERR_UNSUPPORTED;
   const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
   const CUresult r = fn(tm, type, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
   return r == CUDA_SUCCESS ? FUFFT_OK : FUFFT_ERR_UNSUPPORTED;
}
}  // namespace host
namespace mx {

// Alignment of the rows of a matrix: whole 32-byte transfers, or any.
template<class T> bool rows_on_32(const void* p, long long row_stride)
{
   return aligned(p, 32) && row_stride * (long long)sizeof(T) % 32 == 0;
}

// Rows: a warp takes U x 512 columns of a row, a lane sixteen of each, two
// lanes a block, eight lanes the four blocks of a scale word.  Columns beyond
// `cols` are zeros.  Bound by reading x and writing the codes (16384^2 bf16 98
// us; its bytes at the rate of a plain copy, half of which are writes, 104;
// 8192^2 bf16 27, fp32 46).
constexpr int SPAN = 32 * HALF;   // columns of a warp's pass
constexpr int STAGE = SPAN + SPAN / HALF;

// sixteen consecutive values a lane out of 512 that a warp reads side by
// side: rows on odd addresses go through shared memory
template<class T> __device__ __forceinline__ void load_unaligned(const T* p, int count, float* stage, int lane, Half<T>& h)
{
   __syncwarp();
#pragma unroll
   for(int i = 0; i < HALF; ++i) {
      const int e = i * 32 + lane;
      stage[e + e / HALF] = e < count ? to_f(p[e]) : 0.0f;
   }
   __syncwarp();
   float v[HALF];
#pragma unroll
   for(int i = 0; i < HALF; ++i) v[i] = stage[lane * (HALF + 1) + i];
   h.set(v);
}

template<class T, int U>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, unsigned rows, long long cols,
                                                            long long row_stride, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales, bool on_32)
{
   tc::let_next_start();
   __shared__ float stage[8][STAGE];
   const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
   const long long pitch = mx4_pitch(cols);
   const unsigned per = (unsigned)ceil_div(pitch * 2, U * SPAN), w = blockIdx.x * 8 + warp;
   const unsigned row = w / per;
   if(row >= rows) return;
   const long long c0 = (long long)(w % per) * (U * SPAN);
   const T* at = x + row * row_stride + c0;
   Half<T> h[U];
#pragma unroll
   for(int u = 0; u < U; ++u) {
      const int left = (int)max(0ll, min((long long)SPAN, cols - c0 - u * SPAN));
      const int mine = max(0, min(HALF, left - lane * HALF));
      if(!on_32) load_unaligned(at + u * SPAN, left, stage[warp], lane, h[u]);
      else if(mine == HALF) h[u].load(at + u * SPAN + lane * HALF);
      else h[u].load_some(at + u * SPAN + lane * HALF, mine);
   }
   // The last tile's rows that are not there have zeros for scales: dealt to those that are, eight lanes a tile.  Rows
   // 32 apart are neighbours in a tile.
   const unsigned tile_rows = min(rows - row / TILE_ROWS * TILE_ROWS, (unsigned)TILE_ROWS);
   if(tile_rows < TILE_ROWS)
      for(int u = 0; u < U; ++u) {
         const long long col = c0 + u * SPAN + lane * HALF;
         if(col >= pitch * 2) break;
         uint8_t* words = scales + ((long long)(row / TILE_ROWS) * (pitch / 64) + col / 128) * TILE_BYTES;
         const unsigned in = row % TILE_ROWS, step = min(tile_rows, 32u);
         for(unsigned r = in % 32 + step * (lane & 7); in < 32 && r < 32; r += step * 8) {
            uint32_t* line = reinterpret_cast<uint32_t*>(words + r * 16);
            if(r >= tile_rows) *reinterpret_cast<uint4*>(line) = make_uint4(0, 0, 0, 0);
            else
               for(int k = 1; k < 4; ++k)
                  if(r + 32 * k >= tile_rows) line[k] = 0u;
         }
      }
#pragma unroll
   for(int u = 0; u < U; ++u) {
      uint32_t c[2];
      const uint32_t s = encode_pair<false>(h[u], c);
      uint32_t word = s << (8 * ((lane >> 1) & 3));
      word |= __shfl_xor_sync(0xffffffffu, word, 2);
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      const long long col = c0 + u * SPAN + lane * HALF;
      if(col >= pitch * 2) continue;
      store_codes<2>(codes + row * pitch + col / 2, c);
      if((lane & 7) == 0) {
         const long long tile = (long long)(row / TILE_ROWS) * (pitch / 64) + col / 128;
         *reinterpret_cast<uint32_t*>(scales + tile * TILE_BYTES + tile_word((int)(row % TILE_ROWS))) = word;
      }
   }
}

// Columns (and rows, where asked): a CTA takes a tile of 128 x 128 values
// through shared memory, as they came.  Row blocks are encoded from the
// registers of the load, eight lanes a row; column blocks from the tile, four
// lanes the four blocks of a column, so that a column's 64 bytes of codes leave
// side by side.  Within a row the four-word groups of a lane stand 8 groups
// apart, next to the other lanes' groups (place, word_at), and every 32 rows
// are skewed by 8 words: both the stores of the rows and the loads of 8 words
// x 4 blocks fall on 32 banks.
// Bound by the reads and writes with fp32 (8192^2 both ways 61 us, floor 52; two
// CTAs an SM, whose registers hold a block: 65 before the maxima took abs values
// unmasked, then three 78), by the ALU and the phases of a tile with bfloat16
// (40 us, floor 31; four CTAs the same; 46 while halves were widened by masks
// and shifts and zeroed one by one, then two 55).
constexpr int QT = 128;
template<class T> struct Tile {
   static constexpr int PITCH = QT * (int)sizeof(T) / 4 + 4;         // words; rows stay on 16 bytes
   static constexpr int BYTES = (QT * PITCH + 3 * 8) * 4;
   static constexpr int PER = 4 / (int)sizeof(T);                     // columns of a word
   static constexpr int GROUPS = Half<T>::WORDS / 4;                  // of a lane
   __device__ static __forceinline__ int at(int row, int place) { return row * PITCH + (row >> 5) * 8 + place; }
   __device__ static __forceinline__ int place(int word)
   {
      const int g = word >> 2;
      return (g % GROUPS * 8 + g / GROUPS) * 4 + (word & 3);
   }
   __device__ static __forceinline__ int word_at(int place)
   {
      const int p = place >> 2;
      return ((p & 7) * GROUPS + (p >> 3)) * 4 + (place & 3);
   }
};

// 32 values over the block's scale -> its sixteen bytes of codes, zeros under a NaN scale
__device__ __forceinline__ uint4 encode_block(uint32_t s, const float* v)
{
   const uint4 q = make_uint4(e2m1_encode8(v), e2m1_encode8(v + 8), e2m1_encode8(v + 16), e2m1_encode8(v + 24));
   return s == 255u ? make_uint4(0, 0, 0, 0) : q;
}

// a tile's scales of rows that are not there, where some are and some are not
__device__ __forceinline__ void clear_words(uint8_t* words, long long there)
{
   if(there <= 0 || there >= TILE_ROWS) return;
   for(int r = (int)there + threadIdx.x; r < TILE_ROWS; r += blockDim.x) *reinterpret_cast<uint32_t*>(words + tile_word(r)) = 0u;
}

template<class T, bool ROWS>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 2 : 3) quantize_tile_kernel(const T* __restrict__ x, long long rows, long long cols,
                                                               long long row_stride, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales, uint8_t* __restrict__ codes_t,
                                                               uint8_t* __restrict__ scales_t, bool on_32)
{
   using Q = Tile<T>;
   extern __shared__ uint4 dynamic[];
   uint32_t* tile = reinterpret_cast<uint32_t*>(dynamic);
   const unsigned ct = (unsigned)mx4_scale_tiles(cols);
   const long long r0 = (long long)(blockIdx.x / ct) * QT, c0 = (long long)(blockIdx.x % ct) * QT;
   const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
   Half<T> h[4];
   if(on_32) {
#pragma unroll
      for(int u = 0; u < 4; ++u) {
         const int r = warp * 16 + u * 4 + (lane >> 3), c = (lane & 7) * HALF;
         const int mine = r0 + r < rows ? (int)max(0ll, min((long long)HALF, cols - c0 - c)) : 0;
         const T* at = x + (r0 + r) * row_stride + c0 + c;
         if(mine == HALF) h[u].load(at);
         else h[u].load_some(at, mine);
      }
   } else {
      // a row at a time, side by side, into the tile; then as above from there
      T* cells = reinterpret_cast<T*>(tile);
      for(int k = 0; k < 16; ++k) {
         const int r = warp * 16 + k;
#pragma unroll
         for(int i = 0; i < QT / 32; ++i) {
            const int c = i * 32 + lane;
            cells[Q::at(r, Q::place(c / Q::PER)) * Q::PER + c % Q::PER] = r0 + r < rows && c0 + c < cols ? x[(r0 + r) * row_stride + c0 + c] : from_f<T>(0.0f);
         }
      }
      __syncwarp();
#pragma unroll
      for(int u = 0; u < 4; ++u) {
         const int r = warp * 16 + u * 4 + (lane >> 3);
#pragma unroll
         for(int i = 0; i < Half<T>::WORDS; ++i) h[u].w[i] = tile[Q::at(r, Q::place((lane & 7) * Half<T>::WORDS + i))];
      }
      __syncwarp();
   }
#pragma unroll
   for(int u = 0; u < 4; ++u) {
      const int r = warp * 16 + u * 4 + (lane >> 3), c = (lane & 7) * HALF;
      if(on_32)
#pragma unroll
         for(int i = 0; i < Half<T>::WORDS / 4; ++i)
            *reinterpret_cast<uint4*>(tile + Q::at(r, (i * 8 + (lane & 7)) * 4)) =
               make_uint4(h[u].w[4 * i], h[u].w[4 * i + 1], h[u].w[4 * i + 2], h[u].w[4 * i + 3]);
      if constexpr(ROWS) {
         uint32_t q[2];
         const uint32_t s = encode_pair<false>(h[u], q);
         uint32_t word = s << (8 * ((lane >> 1) & 3));
         word |= __shfl_xor_sync(0xffffffffu, word, 2);
         word |= __shfl_xor_sync(0xffffffffu, word, 4);
         if(r0 + r < rows) {
            store_codes<2>(codes + (r0 + r) * mx4_pitch(cols) + (c0 + c) / 2, q);
            if((lane & 7) == 0)
               *reinterpret_cast<uint32_t*>(scales + (r0 / TILE_ROWS * ct + c0 / QT) * TILE_BYTES + tile_word(r)) = word;
         }
      }
   }
   if constexpr(ROWS) clear_words(scales + (r0 / TILE_ROWS * ct + c0 / QT) * TILE_BYTES, rows - r0);
   __syncthreads();
   const int b = lane & 3;
   uint8_t* scale_tile = scales_t + (c0 / TILE_ROWS * mx4_scale_tiles(rows) + r0 / QT) * TILE_BYTES;
#pragma unroll
   for(int k = 0; k < QT / Q::PER / 64; ++k) {
      const int place = k * 64 + warp * 8 + (lane >> 2), column = Q::word_at(place) * Q::PER;   // one column or two
      uint32_t raw[BLOCK];
#pragma unroll
      for(int i = 0; i < BLOCK; ++i) raw[i] = tile[Q::at(b * BLOCK + i, place)];
      const uint32_t most = max_words<T, BLOCK>(raw);
      uint32_t s[Q::PER];
      uint4 q[Q::PER];
      float v[BLOCK];
      if constexpr(Q::PER == 1) {
         s[0] = scale_byte<2>(most);
         const float inv = scale_inverse(s[0]);
#pragma unroll
         for(int i = 0; i < BLOCK; i += 2) {
            const float2 f = fmul2(make_float2(__uint_as_float(raw[i]), __uint_as_float(raw[i + 1])), make_float2(inv, inv));
            v[i] = f.x;
            v[i + 1] = f.y;
         }
         q[0] = encode_block(s[0], v);
      } else {
         // both columns are widened in one go
         const float2 top = unpack2<T>(most);
         s[0] = scale_byte<2>(abs_bits(top.x));
         s[1] = scale_byte<2>(abs_bits(top.y));
         const float2 inv = make_float2(scale_inverse(s[0]), scale_inverse(s[1]));
         float v1[BLOCK];
#pragma unroll
         for(int i = 0; i < BLOCK; ++i) {
            scaled_pair<T>(raw[i], inv, v + i, v1 + i);
         }
         q[0] = encode_block(s[0], v);
         q[1] = encode_block(s[1], v1);
      }
#pragma unroll
      for(int e = 0; e < Q::PER; ++e) {
         uint32_t scale_word = s[e] << (8 * b);
         scale_word |= __shfl_xor_sync(0xffffffffu, scale_word, 1);
         scale_word |= __shfl_xor_sync(0xffffffffu, scale_word, 2);
         const int c = column + e;
         if(c0 + c < cols) {
            *reinterpret_cast<uint4*>(codes_t + (c0 + c) * mx4_pitch(rows) + r0 / 2 + b * 16) = q[e];
            if(b == 0) *reinterpret_cast<uint32_t*>(scale_tile + tile_word(c)) = scale_word;
         }
      }
   }
   clear_words(scale_tile, cols - c0);
}

template<class T, int U>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ codes,
                                                         const uint8_t* __restrict__ scales, unsigned rows, long long cols,
                                                         T* __restrict__ out, long long row_stride, bool on_32)
{
   __shared__ float stage[8][STAGE];
   const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
   const long long pitch = mx4_pitch(cols);
   const unsigned per = (unsigned)ceil_div(cols, U * SPAN), w = blockIdx.x * 8 + warp;
   const unsigned row = w / per;
   if(row >= rows) return;
   const long long c0 = (long long)(w % per) * (U * SPAN);
   const uint8_t* tiles = scales + (long long)(row / TILE_ROWS) * (pitch / 64) * TILE_BYTES + tile_word((int)(row % TILE_ROWS));
   uint32_t q[U][2], s[U];
#pragma unroll
   for(int u = 0; u < U; ++u) {
      const long long col = c0 + u * SPAN + lane * HALF;
      q[u][0] = q[u][1] = s[u] = 0;
      if(col < cols) {
         load_codes<2>(codes + row * pitch + col / 2, q[u]);
         s[u] = __ldg(tiles + col / 128 * TILE_BYTES + ((lane >> 1) & 3));
      }
   }
#pragma unroll
   for(int u = 0; u < U; ++u) {
      float v[HALF];
      decode<false>(q[u], scale_value(s[u]), v);
      T* at = out + row * row_stride + c0 + u * SPAN;
      const int left = (int)max(0ll, min((long long)SPAN, cols - c0 - u * SPAN)), mine = left - lane * HALF;
      if(on_32) {
         Half<T> h;
         h.set(v);
         if(mine >= HALF) h.store(at + lane * HALF);
         else h.store_some(at + lane * HALF, mine);
      } else {
         __syncwarp();
#pragma unroll
         for(int i = 0; i < HALF; ++i) stage[warp][lane * (HALF + 1) + i] = v[i];
         __syncwarp();
#pragma unroll
         for(int i = 0; i < HALF; ++i) {
            const int e = i * 32 + lane;
            if(e < left) at[e] = from_f<T>(stage[warp][e + e / HALF]);
         }
      }
   }
}

// four passes a warp in flight where rows have them and the card stays full;
// else one (bf16, one / four: 16 x 4096 2.1 / 2.7 us, 16384^2 112 / 98)
bool four_passes(long long rows, long long spans) { return spans >= 4 && rows * spans >= 32 * 148; }

template<class T>
fufft_status quantize(const void* x, long long rows, long long cols, long long row_stride, uint8_t* codes,
                      uint8_t* scales, uint8_t* codes_t, uint8_t* scales_t, cudaStream_t st)
{
   const T* p = static_cast<const T*>(x);
   const bool on_32 = rows_on_32<T>(x, row_stride);
   if(!codes_t) {
      const long long spans = ceil_div(mx4_pitch(cols) * 2, SPAN);
      if(four_passes(rows, spans))
         quantize_rows_kernel<T, 4><<<(unsigned)ceil_div(rows * ceil_div(spans, 4), 8), 256, 0, st>>>(p, (unsigned)rows, cols, row_stride, codes, scales, on_32);
      else
         quantize_rows_kernel<T, 1><<<(unsigned)ceil_div(rows * spans, 8), 256, 0, st>>>(p, (unsigned)rows, cols, row_stride, codes, scales, on_32);
   } else {
      static std::atomic<uint64_t> configured[2]{};
      fufft_status s = codes ? allow_smem(quantize_tile_kernel<T, true>, Tile<T>::BYTES, configured[1])
                             : allow_smem(quantize_tile_kernel<T, false>, Tile<T>::BYTES, configured[0]);
      if(s != FUFFT_OK) return s;
      const unsigned tiles = (unsigned)(mx4_scale_tiles(rows) * mx4_scale_tiles(cols));
      if(codes)
         quantize_tile_kernel<T, true><<<tiles, 256, Tile<T>::BYTES, st>>>(p, rows, cols, row_stride, codes, scales, codes_t, scales_t, on_32);
      else
         quantize_tile_kernel<T, false><<<tiles, 256, Tile<T>::BYTES, st>>>(p, rows, cols, row_stride, codes, scales, codes_t, scales_t, on_32);
   }
   count_launch();
   return check(cudaGetLastError());
}

template<class T>
fufft_status dequantize(const uint8_t* codes, const uint8_t* scales, long long rows, long long cols, void* out,
                        long long row_stride, cudaStream_t st)
{
   const bool on_32 = rows_on_32<T>(out, row_stride);
   const long long spans = ceil_div(cols, SPAN);
   if(four_passes(rows, spans))
      dequantize_kernel<T, 4><<<(unsigned)ceil_div(rows * ceil_div(spans, 4), 8), 256, 0, st>>>(codes, scales, (unsigned)rows, cols, static_cast<T*>(out), row_stride, on_32);
   else
      dequantize_kernel<T, 1><<<(unsigned)ceil_div(rows * spans, 8), 256, 0, st>>>(codes, scales, (unsigned)rows, cols, static_cast<T*>(out), row_stride, on_32);
   count_launch();
   return check(cudaGetLastError());
}

constexpr long long MAX_DIM = 1ll << 30;
constexpr long long MAX_ELEMENTS = 1ll << 38;   // keeps grids and warp indices below 2^31

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
