// fufft_cache_conv.cu -- one new output of a causal convolution per sequence,
// from the cached inputs:
//   y[b][c] = gate[b][c] * sum_{j < min(len_b, L)} taps[j][head(c)] * x[b][len_b - 1 - j][c]
// with head(c) = c / (channels / heads).
#include "fufft_cache.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace cache {

struct ConvStep {
   const int32_t* lengths;
   const void* taps;
   long long taps_stride;
   int n_taps, group;        // group = channels per head
   int channels;
   const void* gate;
   long long gate_stride;
   void* out;
   long long out_stride;
   float* partial;           // [splits][batch][channels], or null with one split
   int chunk;                // lags per split
};

template<class TT> __device__ __forceinline__ void load_taps8(const ConvStep& a, long long j, int c, float* h)
{
   const TT* row = static_cast<const TT*>(a.taps) + j * a.taps_stride;
#pragma unroll
   for(int i = 0; i < 8; ++i) h[i] = mx::to_f(row[(c + i) / a.group]);
}

template<class T> __device__ __forceinline__ void finish8(const ConvStep& a, int b, int c, float* y)
{
#pragma unroll
   for(int i = 0; i < 8; ++i) {
      if(a.gate) y[i] *= mx::to_f(static_cast<const T*>(a.gate)[b * a.gate_stride + c + i]);
      static_cast<T*>(a.out)[b * a.out_stride + c + i] = mx::from_f<T>(y[i]);
   }
}

// a warp holds 256 channels, the eight warps of a CTA take the lags in turn
template<class T, class TT, bool MX8>
__global__ void __launch_bounds__(256) conv_step_kernel(Pages p, ConvStep a)
{
   __shared__ float sum[8][256];
   const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
   const int c = blockIdx.x * 256 + lane * 8, b = blockIdx.z;
   const long long len = a.lengths[b];
   const long long j0 = (long long)blockIdx.y * a.chunk;
   const long long j1 = min(min(j0 + a.chunk, len), (long long)a.n_taps);
   float y[8] = {};
   if(c < a.channels)
      for(long long j = j0 + warp; j < j1; j += 8) {
         const long long slot = p.slot(b, len - 1 - j);
         if(slot < 0) continue;
         float v[8], h[8];
         p.load8<MX8>(slot, c, a.channels, v);
         load_taps8<TT>(a, j, c, h);
#pragma unroll
         for(int i = 0; i < 8; ++i) y[i] = fmaf(v[i], h[i], y[i]);
      }
#pragma unroll
   for(int i = 0; i < 8; ++i) sum[warp][lane * 8 + i] = y[i];
   __syncthreads();
   if(warp == 0 && c < a.channels) {
#pragma unroll
      for(int w = 1; w < 8; ++w)
#pragma unroll
         for(int i = 0; i < 8; ++i) y[i] += sum[w][lane * 8 + i];
      if(a.partial) {
         float* at = a.partial + ((long long)blockIdx.y * p.batch + b) * a.channels + c;
#pragma unroll
         for(int i = 0; i < 8; ++i) at[i] = y[i];
      } else {
         finish8<T>(a, b, c, y);
      }
   }
}

// joins the splits in their order
template<class T>
__global__ void __launch_bounds__(256) conv_join_kernel(ConvStep a, int batch, int splits)
{
   const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
   const int per = a.channels / 8;
   if(g >= (long long)batch * per) return;
   const int b = (int)(g / per), c = (int)(g % per) * 8;
   float y[8] = {};
   for(int s = 0; s < splits; ++s)
#pragma unroll
      for(int i = 0; i < 8; ++i) y[i] += a.partial[((long long)s * batch + b) * a.channels + c + i];
   finish8<T>(a, b, c, y);
}

// lags per split: enough CTAs for four per SM, 64 lags at least
struct Plan {
   int chunk, splits;
};
Plan plan(long long lags, int channels, int batch, int sms)
{
   const long long rows = mx::ceil_div(channels, 256) * batch;
   const long long want = mx::ceil_div(4ll * sms, rows > 0 ? rows : 1);
   long long chunk = mx::ceil_div(lags > 0 ? lags : 1, want);
   chunk = mx::ceil_div(chunk < 64 ? 64 : chunk, 8) * 8;
   return {(int)chunk, (int)mx::ceil_div(lags > 0 ? lags : 1, chunk)};
}

template<class T, class TT>
fufft_status run(const fufft_cache* c, const ConvStep& a, int splits, cudaStream_t st)
{
   const dim3 grid((unsigned)mx::ceil_div(c->channels, 256), (unsigned)splits, (unsigned)c->batch);
   if(c->kind == FUFFT_CACHE_MX8) conv_step_kernel<T, TT, true><<<grid, 256, 0, st>>>(Pages(c), a);
   else conv_step_kernel<T, TT, false><<<grid, 256, 0, st>>>(Pages(c), a);
   count_launch();
   fufft_status s = check(cudaGetLastError());
   if(s != FUFFT_OK || splits == 1) return s;
   conv_join_kernel<T><<<(unsigned)mx::ceil_div((long long)c->batch * (c->channels / 8), 256), 256, 0, st>>>(a, c->batch, splits);
   count_launch();
   return check(cudaGetLastError());
}

long long lags_of(const fufft_cache* c, int64_t n_taps)
{
   const long long held = (long long)c->max_pages * c->page_size;
   return held < n_taps ? held : n_taps;
}

}  // namespace cache
}  // namespace fufft

extern "C" {

size_t fufft_cache_conv_workspace(const fufft_cache* c, int64_t n_taps)
{
   if(cache::check_cache(c) != FUFFT_OK || n_taps < 0 || n_taps > cache::MAX_TOKENS || c->batch == 0) return 0;
   int dev = 0;
   if(cudaGetDevice(&dev) != cudaSuccess) return 0;
   const cache::Plan p = cache::plan(cache::lags_of(c, n_taps), c->channels, c->batch, sm_count(dev));
   return p.splits == 1 ? 0 : (size_t)p.splits * c->batch * c->channels * sizeof(float);
}

fufft_status fufft_cache_conv(const fufft_cache* c, const int32_t* lengths, const void* taps, fufft_dtype taps_dtype,
                              int64_t n_taps, int heads, int64_t taps_stride, const void* gate, int64_t gate_stride,
                              void* out, fufft_dtype dtype, int64_t out_stride, void* workspace, size_t workspace_bytes,
                              fufft_stream_t stream)
{
   fufft_status s = cache::check_cache(c);
   if(s != FUFFT_OK) return s;
   if(dtype < FUFFT_F32 || dtype > FUFFT_BF16 || (taps_dtype != FUFFT_F32 && taps_dtype != FUFFT_BF16)) return FUFFT_ERR_INVALID_ARG;
   if(n_taps < 0 || n_taps > cache::MAX_TOKENS || heads <= 0 || c->channels % heads) return FUFFT_ERR_INVALID_SIZE;
   if(c->batch == 0) return FUFFT_OK;
   if(c->batch > 65535) return FUFFT_ERR_INVALID_BATCH;
   if(!lengths || !out || (n_taps && !taps)) return FUFFT_ERR_INVALID_ARG;
   if((n_taps > 1 && taps_stride < heads) || (c->batch > 1 && (out_stride < c->channels || (gate && gate_stride < c->channels))))
      return FUFFT_ERR_INVALID_ARG;
   if(!aligned(lengths, 4) || !aligned(taps, taps_dtype == FUFFT_F32 ? 4 : 2) || !aligned(out, dtype == FUFFT_F32 ? 4 : 2) ||
      !aligned(gate, dtype == FUFFT_F32 ? 4 : 2) || !aligned(workspace, 16))
      return FUFFT_ERR_MISALIGNED;
   int dev = 0;
   if((s = check(cudaGetDevice(&dev))) != FUFFT_OK) return s;
   const cache::Plan p = cache::plan(cache::lags_of(c, n_taps), c->channels, c->batch, sm_count(dev));
   const size_t need = p.splits == 1 ? 0 : (size_t)p.splits * c->batch * c->channels * sizeof(float);
   if(workspace_bytes < need || (need && !workspace)) return FUFFT_ERR_INVALID_ARG;
   cache::ConvStep a{};
   a.lengths = lengths;
   a.taps = taps;
   a.taps_stride = taps_stride;
   a.n_taps = (int)n_taps;
   a.group = c->channels / heads;
   a.channels = c->channels;
   a.gate = gate;
   a.gate_stride = gate_stride;
   a.out = out;
   a.out_stride = out_stride;
   a.partial = need ? static_cast<float*>(workspace) : nullptr;
   a.chunk = p.chunk;
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   const bool wide = taps_dtype == FUFFT_F32;
   switch(dtype) {
   case FUFFT_F32: return wide ? cache::run<float, float>(c, a, p.splits, st) : cache::run<float, __nv_bfloat16>(c, a, p.splits, st);
   case FUFFT_F16: return wide ? cache::run<__half, float>(c, a, p.splits, st) : cache::run<__half, __nv_bfloat16>(c, a, p.splits, st);
   default: return wide ? cache::run<__nv_bfloat16, float>(c, a, p.splits, st) : cache::run<__nv_bfloat16, __nv_bfloat16>(c, a, p.splits, st);
   }
}

}  // extern "C"
