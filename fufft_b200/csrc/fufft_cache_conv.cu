// fufft_cache_conv.cu -- one new output of a causal convolution per sequence,
// from the cached inputs:
//   y[b][c] = gate[b][c] * sum_{j < min(len_b, L)} taps[j][head(c)] * x[b][len_b - 1 - j][c]
// with head(c) = c / (channels / heads).
#include <algorithm>

#include "fufft_cache.cuh"
#include "fufft_tc.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace cache {

constexpr int CH = 16;        // channels per thread: one 8-byte (MX4) or 16-byte (MX8) load a token
constexpr int TILE = 256;     // lags whose cache rows are looked up together, at most
constexpr int THREADS = 256;

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
   fufft_dtype dtype;
   bool vec_taps;            // rows of taps start on 16 bytes
   float* partial;           // [outer][batch][channels], or null with outer == 1
   int lanes, slots;         // threads side by side on the channels; lags in turn
   int split, outer, tile;   // CTAs of a cluster and clusters along the lags; lags per tile
};

// taps of one lag as they lie in memory
enum class Taps { CHANNEL, HEAD, GATHER };   // one per channel / one for all 16 / any
template<class TT, Taps MODE> struct TapRow {
   static constexpr int WORDS = MODE == Taps::HEAD ? 1 : CH * (int)sizeof(TT) / 4;
   uint32_t w[WORDS];
   __device__ __forceinline__ void load(const ConvStep& a, long long j, int c)
   {
      const TT* row = static_cast<const TT*>(a.taps) + j * a.taps_stride;
      if constexpr(MODE == Taps::HEAD) {
         w[0] = __float_as_uint(mx::to_f(row[c / a.group]));
      } else if constexpr(MODE == Taps::CHANNEL) {
#pragma unroll
         for(int i = 0; i < WORDS / 4; ++i) {
            const uint4 q = __ldg(reinterpret_cast<const uint4*>(row + c) + i);
            w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
         }
      } else if constexpr(sizeof(TT) == 4) {
#pragma unroll
         for(int i = 0; i < CH; ++i) w[i] = __float_as_uint(row[(c + i) / a.group]);
      } else {
#pragma unroll
         for(int i = 0; i < CH / 2; ++i)
            w[i] = mx::pack2<__nv_bfloat16>(mx::to_f(row[(c + 2 * i) / a.group]), mx::to_f(row[(c + 2 * i + 1) / a.group]));
      }
   }
   __device__ __forceinline__ float2 pair(int i) const
   {
      if constexpr(MODE == Taps::HEAD) return make_float2(__uint_as_float(w[0]), __uint_as_float(w[0]));
      else if constexpr(sizeof(TT) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
      else return mx::unpack2<__nv_bfloat16>(w[i]);
   }
};

__device__ __forceinline__ float2 ffma2(float2 a, float2 b, float2 c)
{
   float2 r;
   asm("{\n\t.reg .b64 ra, rb, rc, rr;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
       "fma.rn.f32x2 rr, ra, rb, rc;\n\tmov.b64 {%0, %1}, rr;\n\t}"
       : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
   return r;
}

// sixteen stored values
template<bool MX8> struct Codes {
   uint32_t w[MX8 ? 4 : 2];
   __device__ __forceinline__ void load(const uint8_t* at)
   {
      if constexpr(MX8) {
         const uint4 q = __ldg(reinterpret_cast<const uint4*>(at));
         w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
      } else {
         const uint2 q = __ldg(reinterpret_cast<const uint2*>(at));
         w[0] = q.x; w[1] = q.y;
      }
   }
   __device__ __forceinline__ void halves(uint32_t* h) const
   {
      if constexpr(MX8) {
#pragma unroll
         for(int i = 0; i < 4; ++i) mx::e4m3_decode4(w[i], h + 2 * i);
      } else {
         mx::e2m1_decode8(w[0], h);
         mx::e2m1_decode8(w[1], h + 4);
      }
   }
};

template<class T> __device__ __forceinline__ void finish(const ConvStep& a, int b, int c, float y)
{
   if(a.gate) y *= mx::to_f(static_cast<const T*>(a.gate)[b * a.gate_stride + c]);
   static_cast<T*>(a.out)[b * a.out_stride + c] = mx::from_f<T>(y);
}
__device__ __forceinline__ void finish(const ConvStep& a, int b, int c, float y)
{
   if(a.dtype == FUFFT_F32) finish<float>(a, b, c, y);
   else if(a.dtype == FUFFT_F16) finish<__half>(a, b, c, y);
   else finish<__nv_bfloat16>(a, b, c, y);
}

// A CTA: a.lanes x 16 channels of NB sequences, a.slots lags at a time; the
// same taps serve the NB sequences, which stand at different positions of
// their pages but at the same lag.  Per stored value: half a conversion, one
// widening, half a product of scale and tap, half a sum (packed pairs).
// CTAs of a cluster take tiles of lags in turn and join through distributed
// shared memory, in rank order.
template<bool MX8, class TT, Taps MODE, int NB>
__global__ void __launch_bounds__(THREADS, 2) conv_step_kernel(Pages p, ConvStep a)
{
   constexpr int U = NB == 4 ? (MX8 ? 1 : 2) : NB == 2 ? 2 : (sizeof(TT) == 4 && MODE != Taps::HEAD ? 2 : 4);   // lags in flight
   __shared__ int rows[NB][TILE];
   extern __shared__ float4 dynamic[];
   float* joined = reinterpret_cast<float*>(dynamic);   // [NB][slots][lanes * CH]
   const int rank = a.split > 1 ? (int)tc::cluster_rank() : 0;
   const int worker = blockIdx.x, workers = a.split * a.outer;
   const int slot = threadIdx.x / a.lanes, lane = threadIdx.x % a.lanes;
   const int c0 = blockIdx.y * a.lanes * CH, c = c0 + lane * CH, b0 = blockIdx.z * NB;
   const bool active = slot < a.slots && c < a.channels;
   const long long row_bytes = MX8 ? a.channels : a.channels / 2;
   const uint8_t* codes = p.codes + (MX8 ? c : c / 2);
   const uint8_t* scales = p.scales + c / mx::BLOCK;
   const int row_scales = a.channels / mx::BLOCK;

   int len[NB], longest = 0;
#pragma unroll
   for(int s = 0; s < NB; ++s) {
      len[s] = b0 + s < p.batch ? a.lengths[b0 + s] : 0;
      longest = max(longest, len[s]);
   }
   longest = min(longest, a.n_taps);
   float2 acc[NB][CH / 2];
#pragma unroll
   for(int s = 0; s < NB; ++s)
#pragma unroll
      for(int i = 0; i < CH / 2; ++i) acc[s][i] = make_float2(0.0f, 0.0f);

   for(long long j0 = (long long)worker * a.tile; j0 < longest; j0 += (long long)workers * a.tile) {
      const int count = (int)min((long long)a.tile, longest - j0);
      __syncthreads();
      for(int e = threadIdx.x; e < count; e += THREADS)
#pragma unroll
         for(int s = 0; s < NB; ++s) rows[s][e] = len[s] > j0 + e ? (int)p.slot(b0 + s, len[s] - 1 - (j0 + e)) : -1;
      __syncthreads();
      if(!active) continue;
      for(int j = slot; j < count; j += a.slots * U) {
         Codes<MX8> q[U][NB];
         uint32_t sc[U][NB];
         TapRow<TT, MODE> h[U];
#pragma unroll
         for(int u = 0; u < U; ++u) {
            const int ju = j + u * a.slots;
            if(ju < count) h[u].load(a, j0 + ju, c);
#pragma unroll
            for(int s = 0; s < NB; ++s) {
               const int row = ju < count ? rows[s][ju] : -1;
               sc[u][s] = 256;   // nothing there
               if(row >= 0) {
                  q[u][s].load(codes + row * row_bytes);
                  sc[u][s] = __ldg(scales + (long long)row * row_scales);
               }
            }
         }
#pragma unroll
         for(int u = 0; u < U; ++u)
#pragma unroll
            for(int s = 0; s < NB; ++s) {
               if(sc[u][s] > 255) continue;
               const float scale = mx::scale_value(sc[u][s]);
               uint32_t v[CH / 2];
               q[u][s].halves(v);
#pragma unroll
               for(int i = 0; i < CH / 2; ++i)
                  acc[s][i] = ffma2(mx::half2_f(v[i]), fmul2(h[u].pair(i), make_float2(scale, scale)), acc[s][i]);
            }
      }
   }

   // the slots of this CTA, in their order
   const int width = a.lanes * CH, pitch = a.slots * width;
#pragma unroll
   for(int s = 0; s < NB; ++s)
      if(slot < a.slots)
#pragma unroll
         for(int i = 0; i < CH / 4; ++i)
            *reinterpret_cast<float4*>(joined + s * pitch + (slot * a.lanes + lane) * CH + 4 * i) =
               make_float4(acc[s][2 * i].x, acc[s][2 * i].y, acc[s][2 * i + 1].x, acc[s][2 * i + 1].y);
   __syncthreads();
   for(int e = threadIdx.x; e < NB * width; e += THREADS) {
      float* at = joined + e / width * pitch + e % width;
      float y = *at;
      for(int k = 1; k < a.slots; ++k) y += at[k * width];
      *at = y;
   }
   // the CTAs of the cluster, in their order
   if(a.split > 1) tc::cluster_sync();
   else __syncthreads();
   for(int e = threadIdx.x + rank * THREADS; e < NB * width; e += THREADS * a.split) {
      const int s = e / width, i = e % width;
      if(b0 + s >= p.batch || c0 + i >= a.channels) continue;
      const float* at = joined + s * pitch + i;
      float y = *at;
      if(a.split > 1) {
         y = 0.0f;
         for(int r = 0; r < a.split; ++r) y += tc::load_peer(tc::peer_smem(at, r));
      }
      if(a.partial) a.partial[((long long)(worker / a.split) * p.batch + b0 + s) * a.channels + c0 + i] = y;
      else finish(a, b0 + s, c0 + i, y);
   }
   if(a.split > 1) tc::cluster_sync();   // nobody leaves while its sums are being read
}

// joins the clusters in their order
__global__ void __launch_bounds__(256) conv_join_kernel(ConvStep a, int batch)
{
   const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
   if(g >= (long long)batch * a.channels) return;
   float y = 0.0f;
   for(int k = 0; k < a.outer; ++k) y += a.partial[(long long)k * batch * a.channels + g];
   finish(a, (int)(g / a.channels), (int)(g % a.channels), y);
}

// How the work is laid out, from the sizes alone.
struct Plan {
   int nb, lanes, chunks, slots, split, outer, tile;
};
Plan plan(long long lags, int channels, int batch, int sms)
{
   Plan p;
   lags = lags > 0 ? lags : 1;
   p.nb = batch >= 3 ? 4 : batch;
   const int units = channels / CH;
   const long long groups = mx::ceil_div(batch, p.nb);
   // clusters along the lags while a CTA keeps 32 of them
   p.split = 1;
   while(p.split < 8 && lags >= 64ll * p.split) p.split *= 2;
   // channels in as few chunks as give four CTAs per SM, a chunk not below 256 channels
   p.chunks = (int)mx::ceil_div(units, THREADS);
   while(p.chunks * groups * p.split < 4ll * sms && mx::ceil_div(units, p.chunks * 2) >= 16) p.chunks *= 2;
   p.lanes = (int)mx::ceil_div(units, p.chunks);
   p.slots = THREADS / p.lanes;
   p.outer = 1;
   while(p.chunks * groups * p.split * p.outer < 2ll * sms && lags >= 2048ll * p.split * p.outer) p.outer *= 2;
   p.tile = (int)std::min<long long>(TILE, mx::ceil_div(lags, (long long)p.split * p.outer));
   return p;
}

template<bool MX8, class TT, Taps MODE, int NB>
fufft_status launch(const fufft_cache* c, const ConvStep& a, const Plan& p, cudaStream_t st)
{
   auto kern = conv_step_kernel<MX8, TT, MODE, NB>;
   static std::atomic<uint64_t> configured{0};
   fufft_status s = allow_smem(kern, NB * THREADS * CH * (int)sizeof(float), configured);
   if(s != FUFFT_OK) return s;
   cudaLaunchConfig_t cfg = {};
   cfg.gridDim = dim3((unsigned)(p.split * p.outer), (unsigned)p.chunks, (unsigned)mx::ceil_div(c->batch, NB));
   cfg.blockDim = dim3(THREADS);
   cfg.dynamicSmemBytes = (size_t)NB * p.slots * p.lanes * CH * sizeof(float);
   cfg.stream = st;
   cudaLaunchAttribute at[1];
   at[0].id = cudaLaunchAttributeClusterDimension;
   at[0].val.clusterDim.x = (unsigned)p.split;
   at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
   cfg.attrs = at;
   cfg.numAttrs = 1;
   if((s = check(cudaLaunchKernelEx(&cfg, kern, Pages(c), a))) != FUFFT_OK) return s;
   count_launch();
   if(p.outer > 1) {
      conv_join_kernel<<<(unsigned)mx::ceil_div((long long)c->batch * c->channels, 256), 256, 0, st>>>(a, c->batch);
      count_launch();
   }
   return check(cudaGetLastError());
}
template<bool MX8, class TT, Taps MODE>
fufft_status launch(const fufft_cache* c, const ConvStep& a, const Plan& p, cudaStream_t st)
{
   return p.nb == 4 ? launch<MX8, TT, MODE, 4>(c, a, p, st)
                    : p.nb == 2 ? launch<MX8, TT, MODE, 2>(c, a, p, st) : launch<MX8, TT, MODE, 1>(c, a, p, st);
}
template<bool MX8, class TT>
fufft_status launch(const fufft_cache* c, const ConvStep& a, const Plan& p, cudaStream_t st)
{
   if(a.group == 1 && a.vec_taps) return launch<MX8, TT, Taps::CHANNEL>(c, a, p, st);
   if(a.group % CH == 0) return launch<MX8, TT, Taps::HEAD>(c, a, p, st);
   return launch<MX8, TT, Taps::GATHER>(c, a, p, st);
}

long long lags_of(const fufft_cache* c, int64_t n_taps)
{
   const long long held = (long long)c->max_pages * c->page_size;
   return held < n_taps ? held : n_taps;
}

size_t workspace(const Plan& p, const fufft_cache* c)
{
   return p.outer == 1 ? 0 : (size_t)p.outer * c->batch * c->channels * sizeof(float);
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
   return cache::workspace(p, c);
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
   const size_t need = cache::workspace(p, c);
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
   a.dtype = dtype;
   a.vec_taps = aligned(taps, 16) && taps_stride * (taps_dtype == FUFFT_F32 ? 4 : 2) % 16 == 0;
   a.partial = need ? static_cast<float*>(workspace) : nullptr;
   a.lanes = p.lanes;
   a.slots = p.slots;
   a.split = p.split;
   a.outer = p.outer;
   a.tile = p.tile;
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   if(c->kind == FUFFT_CACHE_MX8)
      return taps_dtype == FUFFT_F32 ? cache::launch<true, float>(c, a, p, st) : cache::launch<true, __nv_bfloat16>(c, a, p, st);
   return taps_dtype == FUFFT_F32 ? cache::launch<false, float>(c, a, p, st) : cache::launch<false, __nv_bfloat16>(c, a, p, st);
}

}  // extern "C"
