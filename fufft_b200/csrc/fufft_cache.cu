// fufft_cache.cu -- the paged sequence cache in microscaled formats: tokens
// quantised as they are written, read back token by token or channel by
// channel (zero padded: the rows the FFT convolution takes).
#include <algorithm>

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

// A CTA takes `per` tokens: their places are looked up once, by a thread each,
// then its threads walk over the tokens' halves of blocks (16 channels, two
// neighbouring lanes a block), a token after the other.  Bound by reading one
// side and writing the other (65536 x 4096 bf16, MX4: append 106 us, read 109,
// floor 104).
constexpr int MAX_PER = 64;
constexpr int THREADS = 256;

struct Walk {   // over [tokens][units], THREADS at a time, without a division a step
   unsigned units, dt, du, t, u;
   __device__ __forceinline__ explicit Walk(unsigned units_)
      : units(units_), dt(THREADS / units_), du(THREADS % units_), t(threadIdx.x / units_), u(threadIdx.x % units_)
   {
   }
   __device__ __forceinline__ void step()
   {
      t += dt;
      u += du;
      if(u >= units) {
         u -= units;
         ++t;
      }
   }
};

// tokens t0 .. t0 + n - 1: rows of the flattened pages, -1 without one
__device__ __forceinline__ void look_up(const Pages& p, const int32_t* cu, const int32_t* starts, long long t0, int n,
                                        int* rows)
{
   if(threadIdx.x < n) {
      const long long t = t0 + threadIdx.x;
      const int b = find_sequence(cu, p.batch, t);
      rows[threadIdx.x] = b < 0 ? -1 : p.slot(b, (long long)starts[b] + (t - cu[b]));
   }
   __syncthreads();
}

// four steps' loads, then four steps' stores
constexpr int U = 4;

template<class T, bool MX8>
__global__ void __launch_bounds__(THREADS) append_kernel(const T* __restrict__ x, long long row_stride, Pages p,
                                                         const int32_t* __restrict__ cu, const int32_t* __restrict__ starts,
                                                         long long tokens, int per, int units, bool on_32)
{
   using E = mx::Elem<MX8>;
   __shared__ int rows[MAX_PER];
   const long long t0 = (long long)blockIdx.x * per;
   const int n = (int)min((long long)per, tokens - t0);
   look_up(p, cu, starts, t0, n, rows);
   x += t0 * row_stride;
   Walk w(units);
   // whole warps go round together: a block's two lanes meet in a shuffle
   const unsigned rounds = ((unsigned)(n * units) + THREADS * U - 1) / (THREADS * U);
   for(unsigned r = 0; r < rounds; ++r) {
      mx::Half<T> h[U];
      unsigned t[U], u[U];
#pragma unroll
      for(int k = 0; k < U; ++k, w.step()) {
         t[k] = w.t;
         u[k] = w.u;
         const T* at = x + t[k] * row_stride + u[k] * mx::HALF;
         if(t[k] >= (unsigned)n) h[k].zero();
         else if(on_32) h[k].load(at);
         else h[k].load_some(at, mx::HALF);
      }
#pragma unroll
      for(int k = 0; k < U; ++k) {
         uint32_t q[E::WORDS];
         const uint32_t s = mx::encode_pair<MX8>(h[k], q);
         const int row = t[k] < (unsigned)n ? rows[t[k]] : -1;
         if(row < 0) continue;
         mx::store_codes<E::WORDS>(p.codes + ((long long)row * units + u[k]) * (4 * E::WORDS), q);
         if((u[k] & 1) == 0) p.scales[((long long)row * units + u[k]) / 2] = (uint8_t)s;
      }
   }
}

template<class T, bool MX8>
__global__ void __launch_bounds__(THREADS) read_kernel(T* __restrict__ out, long long row_stride, Pages p,
                                                       const int32_t* __restrict__ cu, const int32_t* __restrict__ starts,
                                                       long long tokens, int per, int units, bool on_32)
{
   using E = mx::Elem<MX8>;
   __shared__ int rows[MAX_PER];
   const long long t0 = (long long)blockIdx.x * per;
   const int n = (int)min((long long)per, tokens - t0);
   look_up(p, cu, starts, t0, n, rows);
   out += t0 * row_stride;
   Walk w(units);
   while(w.t < (unsigned)n) {
      uint32_t q[U][E::WORDS], s[U];
      unsigned t[U], u[U];
#pragma unroll
      for(int k = 0; k < U; ++k, w.step()) {
         t[k] = w.t;
         u[k] = w.u;
         const int row = t[k] < (unsigned)n ? rows[t[k]] : -1;
#pragma unroll
         for(int i = 0; i < E::WORDS; ++i) q[k][i] = 0;
         s[k] = 0;
         if(row >= 0) {
            mx::load_codes<E::WORDS>(p.codes + ((long long)row * units + u[k]) * (4 * E::WORDS), q[k]);
            s[k] = __ldg(p.scales + ((long long)row * units + u[k]) / 2);
         }
      }
#pragma unroll
      for(int k = 0; k < U; ++k) {
         if(t[k] >= (unsigned)n) continue;
         float v[mx::HALF];
         mx::decode<MX8>(q[k], mx::scale_value(s[k]), v);
         mx::Half<T> h;
         h.set(v);
         T* at = out + t[k] * row_stride + u[k] * mx::HALF;
         if(on_32) h.store(at);
         else h.store_some(at, mx::HALF);
      }
   }
}

// A CTA turns 128 positions x 64 channels around in shared memory: a lane
// brings sixteen channels of a position, a group of lanes takes a channel's
// positions out, 16 bytes each.  The tile is skewed by 8 words per 16
// channels: the lanes of a warp, 8 positions x 4 groups of channels, store
// into 32 banks.  Bound by writing the rows, padding and all (8 x 4096 x 16384
// fp32 from 8192 tokens MX4: 433 us, floor 349; MX8 449, floor 370, and 489 with
// loads under conditions).
constexpr int RN = 128, RC = 64, RPITCH = RN + 4;
template<class T, bool MX8>
__global__ void __launch_bounds__(THREADS) read_channels_kernel(T* __restrict__ out, Pages p,
                                                                const int32_t* __restrict__ starts,
                                                                const int32_t* __restrict__ counts, long long n,
                                                                int channels, unsigned tiles_n, unsigned tiles_c, bool on_16)
{
   using E = mx::Elem<MX8>;
   constexpr int W = 16 / (int)sizeof(T);   // positions of a store
   __shared__ int rows[RN];
   __shared__ __align__(16) float tile[RC * RPITCH + 3 * 8];
   const unsigned id = blockIdx.x, rest = id / tiles_n;
   const int b = (int)(rest / tiles_c), c0 = (int)(rest % tiles_c) * RC;
   const long long i0 = (long long)(id % tiles_n) * RN;
   const long long count = min((long long)counts[b], n);
   const bool any = i0 < count && p.pages > 0;
   if(any) {
      if(threadIdx.x < RN) {
         const long long i = i0 + threadIdx.x;
         rows[threadIdx.x] = i < count ? p.slot(b, (long long)starts[b] + i) : -1;
      }
      __syncthreads();
      uint32_t q[2][E::WORDS], s[2];
      bool there[2];
#pragma unroll
      for(int k = 0; k < 2; ++k) {
         const int r = k * 64 + (threadIdx.x >> 2), c = c0 + (threadIdx.x & 3) * mx::HALF;
         there[k] = c < channels && rows[r] >= 0;
         // loads without a condition, the first row's where there is none: what a branch may or may not have loaded
         // is waited for where the branch ends
         const long long row = there[k] ? rows[r] : 0, at = there[k] ? c : 0;
         mx::load_codes<E::WORDS>(p.codes + (row * (channels / mx::HALF) + at / mx::HALF) * (4 * E::WORDS), q[k]);
         s[k] = __ldg(p.scales + row * (channels / mx::BLOCK) + at / mx::BLOCK);
      }
#pragma unroll
      for(int k = 0; k < 2; ++k) {
         const int r = k * 64 + (threadIdx.x >> 2), g = threadIdx.x & 3;
         float v[mx::HALF];
         mx::decode<MX8>(q[k], mx::scale_value(s[k]), v);
#pragma unroll
         for(int i = 0; i < mx::HALF; ++i) tile[(g * mx::HALF + i) * RPITCH + g * 8 + r] = there[k] ? v[i] : 0.0f;
      }
      __syncthreads();
   }
   for(int e = threadIdx.x; e < RC * (RN / W); e += THREADS) {
      const int c = e / (RN / W), r = e % (RN / W) * W;
      if(c0 + c >= channels || i0 + r >= n) continue;
      float v[W];
#pragma unroll
      for(int i = 0; i < W / 4; ++i) {
         const float4 f = any ? *reinterpret_cast<const float4*>(tile + c * RPITCH + (c >> 4) * 8 + r + 4 * i)
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
         v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
      }
      T* at = out + ((long long)b * channels + c0 + c) * n + i0 + r;
      if(on_16 && i0 + r + W <= n) {
         if constexpr(sizeof(T) == 4) *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
         else *reinterpret_cast<uint4*>(at) = make_uint4(mx::pack2<T>(v[0], v[1]), mx::pack2<T>(v[2], v[3]),
                                                         mx::pack2<T>(v[4], v[5]), mx::pack2<T>(v[6], v[7]));
      } else {
#pragma unroll
         for(int i = 0; i < W; ++i)
            if(i0 + r + i < n) at[i] = mx::from_f<T>(v[i]);
      }
   }
}

// tokens of a CTA: 32 K values, but two CTAs per SM before that
int tokens_per_cta(const fufft_cache* c, long long tokens)
{
   int dev = 0, sms = 148;
   if(cudaGetDevice(&dev) == cudaSuccess) sms = sm_count(dev);
   long long per = std::max(1, 32768 / c->channels);
   per = std::min<long long>(per, mx::ceil_div(tokens, 2 * sms));
   return (int)std::min<long long>(per, MAX_PER);
}

template<class T>
fufft_status append(const fufft_cache* c, const void* x, long long row_stride, const int32_t* cu, const int32_t* starts,
                    long long tokens, cudaStream_t st)
{
   const T* xp = static_cast<const T*>(x);
   const bool on_32 = aligned(x, 32) && row_stride * (long long)sizeof(T) % 32 == 0;
   const int per = tokens_per_cta(c, tokens), units = c->channels / mx::HALF;
   const unsigned grid = (unsigned)mx::ceil_div(tokens, per);
   if(c->kind == FUFFT_CACHE_MX8) append_kernel<T, true><<<grid, THREADS, 0, st>>>(xp, row_stride, Pages(c), cu, starts, tokens, per, units, on_32);
   else append_kernel<T, false><<<grid, THREADS, 0, st>>>(xp, row_stride, Pages(c), cu, starts, tokens, per, units, on_32);
   count_launch();
   return check(cudaGetLastError());
}

template<class T>
fufft_status read(const fufft_cache* c, void* out, long long row_stride, const int32_t* cu, const int32_t* starts,
                  long long tokens, cudaStream_t st)
{
   T* op = static_cast<T*>(out);
   const bool on_32 = aligned(out, 32) && row_stride * (long long)sizeof(T) % 32 == 0;
   const int per = tokens_per_cta(c, tokens), units = c->channels / mx::HALF;
   const unsigned grid = (unsigned)mx::ceil_div(tokens, per);
   if(c->kind == FUFFT_CACHE_MX8) read_kernel<T, true><<<grid, THREADS, 0, st>>>(op, row_stride, Pages(c), cu, starts, tokens, per, units, on_32);
   else read_kernel<T, false><<<grid, THREADS, 0, st>>>(op, row_stride, Pages(c), cu, starts, tokens, per, units, on_32);
   count_launch();
   return check(cudaGetLastError());
}

template<class T>
fufft_status read_channels(const fufft_cache* c, void* out, long long n, const int32_t* starts, const int32_t* counts,
                           cudaStream_t st)
{
   T* op = static_cast<T*>(out);
   const unsigned tn = (unsigned)mx::ceil_div(n, RN), tc = (unsigned)mx::ceil_div(c->channels, RC);
   const unsigned grid = tn * tc * (unsigned)c->batch;
   const bool on_16 = aligned(out, 16) && n * (long long)sizeof(T) % 16 == 0;
   if(c->kind == FUFFT_CACHE_MX8) read_channels_kernel<T, true><<<grid, THREADS, 0, st>>>(op, Pages(c), starts, counts, n, c->channels, tn, tc, on_16);
   else read_channels_kernel<T, false><<<grid, THREADS, 0, st>>>(op, Pages(c), starts, counts, n, c->channels, tn, tc, on_16);
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
   if(tokens == 0) return FUFFT_OK;
   if(!out || !cu || (!starts && c->batch) || (row_stride < c->channels && tokens > 1)) return FUFFT_ERR_INVALID_ARG;
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
   if(mx::ceil_div(n, cache::RN) * mx::ceil_div(c->channels, cache::RC) > 0x7fffffffll / c->batch) return FUFFT_ERR_INVALID_SIZE;
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
