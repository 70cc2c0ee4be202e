// fufft_cache.cu -- the paged sequence cache in microscaled formats: tokens
// quantised as they are written, read back token by token or channel by
// channel (zero padded: the rows the FFT convolution takes).
#include "fufft_cache.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace cache {

// sequence of token t in a ragged run (cu[b] <= t < cu[b + 1]), or -1
__device__ __forceinline__ int find_sequence(const int32_t* cu, int batch, long long t)
{
   if(t < cu[0] || t >= cu[batch]) return -1;
   int lo = 0, hi = batch - 1;
   while(lo < hi) {   // the last b with cu[b] <= t: an empty sequence never wins over the one after it
      const int mid = (lo + hi + 1) >> 1;
      if(cu[mid] <= t) lo = mid;
      else hi = mid - 1;
   }
   return lo;
}

// a thread holds eight channels of a token, four neighbouring threads a block
template<class T, bool MX8>
__global__ void __launch_bounds__(256) append_kernel(const T* __restrict__ x, long long row_stride, Pages p,
                                                     const int32_t* __restrict__ cu, const int32_t* __restrict__ starts,
                                                     long long tokens, int channels, bool vec)
{
   using E = mx::Elem<MX8>;
   const int per = channels / 8;
   const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
   const bool live = g < tokens * per;
   const long long t = live ? g / per : 0;
   const int c = live ? (int)(g % per) * 8 : 0;
   float v[8];
   mx::load8(x + t * row_stride + c, vec, 8, v);
   const uint32_t s = mx::block_scale4<E::EMAX>(v);
   const float inv = mx::scale_inverse(s);
#pragma unroll
   for(int i = 0; i < 8; ++i) v[i] = s == 255u ? 0.0f : v[i] * inv;
   uint32_t w[E::WORDS];
   E::encode8(v, w);
   if(!live) return;
   const int b = find_sequence(cu, p.batch, t);
   if(b < 0) return;
   const long long slot = p.slot(b, (long long)starts[b] + (t - cu[b]));
   if(slot < 0) return;
   uint32_t* at = reinterpret_cast<uint32_t*>(p.codes + slot * (long long)per * (4 * E::WORDS)) + (c / 8) * E::WORDS;
   if constexpr(MX8) *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
   else *at = w[0];
   if((threadIdx.x & 3) == 0) p.scales[slot * (channels / mx::BLOCK) + c / mx::BLOCK] = (uint8_t)s;
}

template<class T, bool MX8>
__global__ void __launch_bounds__(256) read_kernel(T* __restrict__ out, long long row_stride, Pages p,
                                                   const int32_t* __restrict__ cu, const int32_t* __restrict__ starts,
                                                   long long tokens, int channels, bool vec)
{
   using E = mx::Elem<MX8>;
   const int per = channels / 8;
   const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
   if(g >= tokens * per) return;
   const long long t = g / per;
   const int c = (int)(g % per) * 8;
   float v[8] = {};
   const int b = find_sequence(cu, p.batch, t);
   const long long slot = b < 0 ? -1 : p.slot(b, (long long)starts[b] + (t - cu[b]));
   if(slot >= 0) p.load8<MX8>(slot, c, channels, v);
   mx::store8(out + t * row_stride + c, vec, 8, v);
}

// a CTA turns 64 positions x 64 channels around in shared memory
constexpr int RT = 64;
template<class T, bool MX8>
__global__ void __launch_bounds__(256) read_channels_kernel(T* __restrict__ out, Pages p,
                                                            const int32_t* __restrict__ starts,
                                                            const int32_t* __restrict__ counts, long long n, int channels)
{
   __shared__ float tile[RT][RT + 1];
   const long long tiles_n = (n + RT - 1) / RT, tiles_c = (channels + RT - 1) / RT;
   const long long id = blockIdx.x;
   const int b = (int)(id / (tiles_n * tiles_c));
   const int c0 = (int)(id / tiles_n % tiles_c) * RT;
   const long long i0 = id % tiles_n * RT;
   const long long count = counts[b];
#pragma unroll
   for(int k = 0; k < RT * RT / 8 / 256; ++k) {
      const int e = threadIdx.x + 256 * k, r = e / (RT / 8), c = e % (RT / 8) * 8;
      float v[8] = {};
      if(i0 + r < count && c0 + c < channels) {
         const long long slot = p.slot(b, (long long)starts[b] + i0 + r);
         if(slot >= 0) p.load8<MX8>(slot, c0 + c, channels, v);
      }
#pragma unroll
      for(int i = 0; i < 8; ++i) tile[r][c + i] = v[i];
   }
   __syncthreads();
   for(int e = threadIdx.x; e < RT * RT; e += 256) {
      const int c = e / RT, r = e % RT;
      if(c0 + c < channels && i0 + r < n) out[((long long)b * channels + c0 + c) * n + i0 + r] = mx::from_f<T>(tile[r][c]);
   }
}

template<class T>
fufft_status append(const fufft_cache* c, const void* x, long long row_stride, const int32_t* cu, const int32_t* starts,
                    long long tokens, cudaStream_t st)
{
   const T* xp = static_cast<const T*>(x);
   const bool vec = aligned(x, 16) && (row_stride * (long long)sizeof(T)) % 16 == 0;
   const unsigned grid = (unsigned)mx::ceil_div(tokens * (c->channels / 8), 256);
   if(c->kind == FUFFT_CACHE_MX8) append_kernel<T, true><<<grid, 256, 0, st>>>(xp, row_stride, Pages(c), cu, starts, tokens, c->channels, vec);
   else append_kernel<T, false><<<grid, 256, 0, st>>>(xp, row_stride, Pages(c), cu, starts, tokens, c->channels, vec);
   count_launch();
   return check(cudaGetLastError());
}

template<class T>
fufft_status read(const fufft_cache* c, void* out, long long row_stride, const int32_t* cu, const int32_t* starts,
                  long long tokens, cudaStream_t st)
{
   T* op = static_cast<T*>(out);
   const bool vec = aligned(out, 16) && (row_stride * (long long)sizeof(T)) % 16 == 0;
   const unsigned grid = (unsigned)mx::ceil_div(tokens * (c->channels / 8), 256);
   if(c->kind == FUFFT_CACHE_MX8) read_kernel<T, true><<<grid, 256, 0, st>>>(op, row_stride, Pages(c), cu, starts, tokens, c->channels, vec);
   else read_kernel<T, false><<<grid, 256, 0, st>>>(op, row_stride, Pages(c), cu, starts, tokens, c->channels, vec);
   count_launch();
   return check(cudaGetLastError());
}

template<class T>
fufft_status read_channels(const fufft_cache* c, void* out, long long n, const int32_t* starts, const int32_t* counts,
                           cudaStream_t st)
{
   T* op = static_cast<T*>(out);
   const unsigned grid = (unsigned)(mx::ceil_div(n, RT) * mx::ceil_div(c->channels, RT) * c->batch);
   if(c->kind == FUFFT_CACHE_MX8) read_channels_kernel<T, true><<<grid, 256, 0, st>>>(op, Pages(c), starts, counts, n, c->channels);
   else read_channels_kernel<T, false><<<grid, 256, 0, st>>>(op, Pages(c), starts, counts, n, c->channels);
   count_launch();
   return check(cudaGetLastError());
}

fufft_status check_cache(const fufft_cache* c)
{
   if(!c) return FUFFT_ERR_INVALID_ARG;
   if(c->kind != FUFFT_CACHE_MX4 && c->kind != FUFFT_CACHE_MX8) return FUFFT_ERR_INVALID_ARG;
   if(c->channels <= 0 || c->channels % mx::BLOCK || c->channels > MAX_CHANNELS || c->page_size <= 0 || c->pages < 0 ||
      c->max_pages < 0)
      return FUFFT_ERR_INVALID_SIZE;
   if((long long)c->pages * c->page_size > 0x7fffffffll) return FUFFT_ERR_INVALID_SIZE;   // a row index is 32 bits
   if(c->batch < 0 || c->batch > MAX_BATCH) return FUFFT_ERR_INVALID_BATCH;
   if(c->batch == 0) return FUFFT_OK;
   if(c->table_stride < c->max_pages) return FUFFT_ERR_INVALID_ARG;
   if(c->pages && (!c->codes || !c->scales)) return FUFFT_ERR_INVALID_ARG;
   if(c->max_pages && !c->page_table) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(c->codes, 16) || !aligned(c->scales, 16) || !aligned(c->page_table, 4)) return FUFFT_ERR_MISALIGNED;
   return FUFFT_OK;
}

}  // namespace cache
}  // namespace fufft

namespace {
bool bad_dtype(fufft_dtype d) { return d < FUFFT_F32 || d > FUFFT_BF16; }
unsigned dtype_align(fufft_dtype d) { return d == FUFFT_F32 ? 4 : 2; }
}  // namespace

extern "C" {

fufft_status fufft_cache_append(const fufft_cache* c, const void* x, fufft_dtype dtype, int64_t row_stride,
                                const int32_t* cu, const int32_t* starts, int64_t tokens, fufft_stream_t stream)
{
   fufft_status s = cache::check_cache(c);
   if(s != FUFFT_OK) return s;
   if(bad_dtype(dtype)) return FUFFT_ERR_INVALID_ARG;
   if(tokens < 0 || tokens > cache::MAX_TOKENS) return FUFFT_ERR_INVALID_SIZE;
   if(tokens == 0 || c->batch == 0) return FUFFT_OK;
   if(!x || !cu || !starts || (row_stride < c->channels && tokens > 1)) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(x, dtype_align(dtype)) || !aligned(cu, 4) || !aligned(starts, 4)) return FUFFT_ERR_MISALIGNED;
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return cache::append<float>(c, x, row_stride, cu, starts, tokens, st);
   case FUFFT_F16: return cache::append<__half>(c, x, row_stride, cu, starts, tokens, st);
   default: return cache::append<__nv_bfloat16>(c, x, row_stride, cu, starts, tokens, st);
   }
}

fufft_status fufft_cache_read(const fufft_cache* c, void* out, fufft_dtype dtype, int64_t row_stride, const int32_t* cu,
                              const int32_t* starts, int64_t tokens, fufft_stream_t stream)
{
   fufft_status s = cache::check_cache(c);
   if(s != FUFFT_OK) return s;
   if(bad_dtype(dtype)) return FUFFT_ERR_INVALID_ARG;
   if(tokens < 0 || tokens > cache::MAX_TOKENS) return FUFFT_ERR_INVALID_SIZE;
   if(tokens == 0 || c->batch == 0) return FUFFT_OK;
   if(!out || !cu || !starts || (row_stride < c->channels && tokens > 1)) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(out, dtype_align(dtype)) || !aligned(cu, 4) || !aligned(starts, 4)) return FUFFT_ERR_MISALIGNED;
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return cache::read<float>(c, out, row_stride, cu, starts, tokens, st);
   case FUFFT_F16: return cache::read<__half>(c, out, row_stride, cu, starts, tokens, st);
   default: return cache::read<__nv_bfloat16>(c, out, row_stride, cu, starts, tokens, st);
   }
}

fufft_status fufft_cache_read_channels(const fufft_cache* c, void* out, fufft_dtype dtype, int64_t n,
                                       const int32_t* starts, const int32_t* counts, fufft_stream_t stream)
{
   fufft_status s = cache::check_cache(c);
   if(s != FUFFT_OK) return s;
   if(bad_dtype(dtype)) return FUFFT_ERR_INVALID_ARG;
   if(n < 0 || n > cache::MAX_TOKENS) return FUFFT_ERR_INVALID_SIZE;
   if(n == 0 || c->batch == 0) return FUFFT_OK;
   if(mx::ceil_div(n, cache::RT) * mx::ceil_div(c->channels, cache::RT) > 0x7fffffffll / c->batch) return FUFFT_ERR_INVALID_SIZE;
   if(!out || !starts || !counts) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(out, dtype_align(dtype)) || !aligned(starts, 4) || !aligned(counts, 4)) return FUFFT_ERR_MISALIGNED;
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return cache::read_channels<float>(c, out, n, starts, counts, st);
   case FUFFT_F16: return cache::read_channels<__half>(c, out, n, starts, counts, st);
   default: return cache::read_channels<__nv_bfloat16>(c, out, n, starts, counts, st);
   }
}

}  // extern "C"
