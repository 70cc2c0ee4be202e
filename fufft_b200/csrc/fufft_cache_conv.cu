// fufft_cache_conv.cu -- one new output of a causal convolution per sequence,
// from the cached inputs:
//   y[b][c] = gate[b][c] * sum_{j < min(len_b, L)} taps[j][head(c)] * x[b][len_b - 1 - j][c]
// with head(c) = c / (channels / heads).
#include <algorithm>
#include <type_traits>

#include "fufft_cache.cuh"
#include "fufft_tc.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace cache {

constexpr int CH = 16;        // channels per thread: one 8-byte (MX4) or 16-byte (MX8) load a token
constexpr int TILE = 1024;    // lags whose cache rows are looked up together, at most (1 x 16384 x 32 MX4: 8.8 us, with 256 10.3)
constexpr int THREADS = 256;
constexpr int MAX_SPLIT = 8;    // CTAs of a portable cluster

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

// x times scale, halves widened: exact
__device__ __forceinline__ float2 widen_scaled(uint32_t x, uint32_t scale)
{
   float2 r;
   asm("{\n\t.reg .b16 a, b, c, d;\n\tmov.b32 {a, b}, %2;\n\tmov.b32 {c, d}, %3;\n\t"
       "fma.rn.f32.f16 %0, a, c, %4;\n\tfma.rn.f32.f16 %1, b, c, %4;\n\t}"
       : "=f"(r.x), "=f"(r.y) : "r"(x), "r"(scale), "f"(0.0f));
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

// a thread's sums, to [sequence][slot][lanes x 16] in shared memory
template<int NB>
__device__ __forceinline__ void park(float* joined, const float2 (&acc)[NB][CH / 2], int slot, int lane, int slots, int lanes)
{
#pragma unroll
   for(int s = 0; s < NB; ++s)
#pragma unroll
      for(int i = 0; i < CH / 4; ++i)
         *reinterpret_cast<float4*>(joined + ((s * slots + slot) * lanes + lane) * CH + 4 * i) =
            make_float4(acc[s][2 * i].x, acc[s][2 * i].y, acc[s][2 * i + 1].x, acc[s][2 * i + 1].y);
}

// Adds the slots of this CTA in their order, then the CTAs of its cluster in
// theirs (through distributed shared memory, a part of the results each), and
// writes the results, or the cluster's part of them where there are several
// (rows `part`, one a sequence).
template<int NB>
__device__ __forceinline__ void join(float* joined, const ConvStep& a, const Pages& p, int width, int slots, int threads,
                                     int rank, int b0, int c0, long long part)
{
   __syncthreads();
   for(int e = threadIdx.x; e < NB * width; e += threads) {
      float* at = joined + e / width * (slots * width) + e % width;
      float y = *at;
      for(int k = 1; k < slots; ++k) y += at[k * width];
      *at = y;
   }
   if(a.split > 1) tc::cluster_sync();
   else __syncthreads();
   for(int e = threadIdx.x + rank * threads; e < NB * width; e += threads * a.split) {
      const int s = e / width, i = e % width;
      if(b0 + s >= p.batch || c0 + i >= a.channels) continue;
      const float* at = joined + s * (slots * width) + i;
      float y = *at;
      if(a.split > 1) {
         float v[MAX_SPLIT];
#pragma unroll
         for(int r = 0; r < MAX_SPLIT; ++r) v[r] = r < a.split ? tc::load_peer(tc::peer_smem(at, r)) : 0.0f;
         y = 0.0f;
#pragma unroll
         for(int r = 0; r < MAX_SPLIT; ++r) y += v[r];
      }
      if(a.partial) a.partial[(part + s) * a.channels + c0 + i] = y;
      else finish(a, b0 + s, c0 + i, y);
   }
   if(a.split > 1) tc::cluster_sync();   // nobody leaves while its sums are being read
}

// A CTA: a.lanes x 16 channels of NB sequences, a.slots lags at a time; the
// same taps serve the NB sequences, which stand at different positions of
// their pages but at the same lag.  A value is scaled before it meets the tap:
// a stored value is a number of 32 bits, exactly, where a scale of 2^124 times
// a tap need not be.  One exact fma widens and scales it where the scale is a
// half-precision number, two operations where a scale of the thread's batch is
// not (5 x 5000 x 2112 MX4, 3001 taps of 22 heads: 12.7 us, 14.8 if all took
// two); half a packed fma adds it times its tap.  The variants whose taps are
// gathered spill, up to 250 bytes with four sequences and fp32 taps.
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
         for(int s = 0; s < NB; ++s) rows[s][e] = len[s] > j0 + e ? p.slot(b0 + s, len[s] - 1 - (j0 + e)) : -1;
      __syncthreads();
      if(!active) continue;
      for(int j = slot; j < count; j += a.slots * U) {
         Codes<MX8> q[U][NB];
         uint32_t sc[U][NB];
         uint32_t there = 0;   // which of them are
         TapRow<TT, MODE> h[U];
         // loads without a condition, the first row's where there is none: what a branch may or may not have loaded
         // is waited for where the branch ends
#pragma unroll
         for(int u = 0; u < U; ++u) {
            const int ju = min(j + u * a.slots, count - 1);
            h[u].load(a, j0 + ju, c);
#pragma unroll
            for(int s = 0; s < NB; ++s) {
               const int row = rows[s][ju];
               there |= (row >= 0 && j + u * a.slots < count ? 1u : 0u) << (u * NB + s);
               q[u][s].load(codes + max(row, 0) * row_bytes);
               sc[u][s] = __ldg(scales + (long long)max(row, 0) * row_scales);
            }
         }
         uint32_t widest = 0;   // below 30: all scales are 2^-14 .. 2^15, normal halves
#pragma unroll
         for(int u = 0; u < U; ++u)
#pragma unroll
            for(int s = 0; s < NB; ++s) widest = max(widest, sc[u][s] - 113u);
         const auto sum = [&](auto halves) {
#pragma unroll
            for(int u = 0; u < U; ++u)
#pragma unroll
               for(int s = 0; s < NB; ++s) {
                  if(!(there >> (u * NB + s) & 1)) continue;
                  uint32_t v[CH / 2];
                  q[u][s].halves(v);
                  if constexpr(halves.value) {
                     const uint32_t scale = (sc[u][s] - 112u) << 10;
#pragma unroll
                     for(int i = 0; i < CH / 2; ++i) acc[s][i] = ffma2(widen_scaled(v[i], scale), h[u].pair(i), acc[s][i]);
                  } else {
                     const float scale = mx::scale_value(sc[u][s]);
#pragma unroll
                     for(int i = 0; i < CH / 2; ++i)
                        acc[s][i] = ffma2(fmul2(mx::half2_f(v[i]), make_float2(scale, scale)), h[u].pair(i), acc[s][i]);
                  }
               }
         };
         if(widest < 30u) sum(std::true_type());
         else sum(std::false_type());
      }
   }

   if(slot < a.slots) park<NB>(joined, acc, slot, lane, a.slots, a.lanes);
   join<NB>(joined, a, p, a.lanes * CH, a.slots, THREADS, rank, b0, c0, (long long)(blockIdx.x / a.split) * p.batch + b0);
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

// ---------------------------------------------------------------------------
// The same through a ring of stages in shared memory, where rows are long
// enough to be copied one by one: what bounds the step is then reading the
// cache, with three instructions a value left to issue meanwhile.  A stage is
// `lags` lags of NS sequences: their rows of codes (tensor copies that gather
// four rows each; a row that is not there is one outside the tensor, and reads
// as zeros), the taps (one tensor copy, 16-byte chunks permuted so that the
// lanes' wide loads fall on different banks) and the scales, with the taps that
// heads share.  A warp fills each slot of the ring; it asks for the pages and
// the scales a stage ahead.  Eight warps sum: a thread keeps 16 channels of the
// NS sequences, so a tap is widened once for all of them.
//
// Two ways to sum a value.  Where every scale of the stage is a half-precision
// number (2^-24 .. 2^15), an exact fma widens the half x and scales it, one
// instruction on both halves of the FMA pipe, and half a packed fma adds it
// times its tap: twice as fast as the general way, whose widening and packed
// product and sum all go to one half of the pipe (B200, a loop of them alone:
// 29 values a clock and SM, 49 this way).  Where rows are missing, each row is
// asked for first (16 sequences of 16384 to 32768, one empty, x 2048 MX4: 171
// us; 201 where such stages took the general way).
// 16 x 32768 x 2048 MX4, bf16 taps: 199 us, floor 107 (a scale of zero in one
// token of 64 takes every stage the general way: 228); taps that heads share
// 208, MX8 259.  The sums alone, without a ring to wait for, 165 (130 with taps
// that heads share, which are read and widened once a block).  Sixteen warps of eight channels a thread: the sums
// alone 171, with the ring 212.
// ---------------------------------------------------------------------------
namespace pipe {
constexpr int CONSUMERS = 8, PRODUCERS = 4, THREADS = (CONSUMERS + PRODUCERS) * 32;   // warps that sum; that fill
constexpr int MAX_PAIRS = 256;                                                         // rows of a stage
constexpr int MAX_STAGES = PRODUCERS;

struct Args {
   ConvStep a;
   unsigned int* status;
   int lags, stages, stage_bytes, codes_at, scales_at;   // of a stage: lags; offsets of its parts (taps at 0)
   int row_bytes;                                        // of the CTA's chunk
   int tap_bytes;                                        // of a lag's taps in the chunk
   int pool;                                             // CTAs of a chunk that the lags are dealt to, or 0
   bool quads;                                           // four blocks' scales at once
};

// Long histories of unequal lengths: the stages of all groups of NS sequences
// are dealt to `pool` CTAs, each of one group, by one warp, to
// starts[group] .. starts[group + 1] - 1: with q the least number for which
// sum ceil(stages of a group / q) does not exceed the pool, a group of t
// stages gets ceil(t / q) CTAs.  pool is at least twice the groups.
constexpr int MAX_GROUPS = 128;
__device__ __forceinline__ int upper_bound(const int* starts, int groups, int worker)   // the group of a CTA; `groups` beyond the last
{
   int lo = 0, hi = groups;
   while(lo < hi) {
      const int mid = (lo + hi) / 2;
      if(starts[mid + 1] > worker) hi = mid;
      else lo = mid + 1;
   }
   return lo;
}
template<int NS> __device__ __noinline__ void deal(const int32_t* lengths, int batch, int n_taps, int lags, int pool, int lane, int* starts)
{
   const int groups = (batch + NS - 1) / NS;
   int t[MAX_GROUPS / 32];
   long long total = 0;
#pragma unroll
   for(int k = 0; k < MAX_GROUPS / 32; ++k) {
      int longest = 0;
      for(int s = 0; s < NS; ++s) {
         const int b = (k * 32 + lane) * NS + s;
         if(b < batch) longest = max(longest, lengths[b]);
      }
      t[k] = (int)(((unsigned)min(longest, n_taps) + lags - 1) / (unsigned)lags);
      total += t[k];
   }
#pragma unroll
   for(int d = 16; d; d /= 2) total += __shfl_xor_sync(0xffffffffu, total, d);
   int lo = max(1, (int)((total + pool - 1) / pool)), hi = max(1, (int)((total + pool - groups - 1) / (pool - groups)));
   while(lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      int need = 0;
#pragma unroll
      for(int k = 0; k < MAX_GROUPS / 32; ++k) need += (t[k] + mid - 1) / mid;
      if((int)__reduce_add_sync(0xffffffffu, need) <= pool) hi = mid;
      else lo = mid + 1;
   }
   int before = 0;
   if(lane == 0) starts[0] = 0;
#pragma unroll
   for(int k = 0; k < MAX_GROUPS / 32; ++k) {
      int sum = (t[k] + lo - 1) / lo;
#pragma unroll
      for(int d = 1; d < 32; d *= 2) {
         const int other = __shfl_up_sync(0xffffffffu, sum, d);
         if(lane >= d) sum += other;
      }
      if(k * 32 + lane < groups) starts[k * 32 + lane + 1] = before + sum;
      before += __shfl_sync(0xffffffffu, sum, 31);
   }
}

// a CTA's share: its first sequence, its number among the CTAs of the group
// and theirs, the longest history within the taps, its stages
struct Share {
   int b0, worker, workers, longest, n;
};
// the length of sequence lane % NS of a group
template<int NS> __device__ __forceinline__ int b_length(const ConvStep& a, const Pages& p, int b0, int lane)
{
   return b0 + lane % NS < p.batch ? max(a.lengths[b0 + lane % NS], 0) : 0;
}

// joins the CTAs of a sequence's group, in their order
template<int NS>
__global__ void __launch_bounds__(256) join_dealt_kernel(ConvStep a, int batch, int lags, int pool)
{
   __shared__ int starts[MAX_GROUPS + 1];
   if(threadIdx.x < 32) deal<NS>(a.lengths, batch, a.n_taps, lags, pool, threadIdx.x, starts);
   __syncthreads();
   const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
   if(i >= (long long)batch * a.channels) return;
   const int b = (int)(i / a.channels), c = (int)(i % a.channels);
   float y = 0.0f;
   for(int w = starts[b / NS]; w < starts[b / NS + 1]; ++w) y += a.partial[((long long)w * NS + b % NS) * a.channels + c];
   finish(a, b, c, y);
}

__device__ __forceinline__ void load_taps(const CUtensorMap* tm, void* dst, int x, int y, int z, uint64_t* bar)
{
   asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                :: "r"(smem_u32(dst)), "l"(tm), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)) : "memory");
}
// four rows of a 2-D map whose box is one row high, side by side; x a multiple of 16 bytes
__device__ __forceinline__ void gather4(const CUtensorMap* tm, void* dst, int x, int4 r, uint64_t* bar)
{
   asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
                :: "r"(smem_u32(dst)), "l"(tm), "r"(x), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "r"(smem_u32(bar)) : "memory");
}
// A scale as a stage holds it: the half-precision number in the low half, its byte in bits 16 .. 23.
constexpr uint32_t NO_HALF = 1u << 31, NO_ROW = 1u << 30;
__device__ __forceinline__ uint32_t scale_entry(uint32_t s)
{
   const int e = (int)s - 127;
   const uint32_t half = e > 15 || e < -24 ? 0u : e >= -14 ? (uint32_t)(e + 15) << 10 : 1u << (e + 24);
   return half | s << 16 | (half ? 0u : NO_HALF);
}

// Cache rows of the pairs (lag, sequence) of a stage, pair = lag * NS +
// sequence; -1 without one.  For the first 64 the page table is asked a stage
// ahead of the use.  Loads that are ahead of their use have no condition (a
// lane without a pair reads any entry): what a branch may or may not have
// loaded is waited for where the branch ends.
template<int NS> struct Rows {
   static constexpr int AHEAD = 2;
   int page[AHEAD], in[AHEAD];
   __device__ __forceinline__ void ask(const Pages& p, int b0, int len, int lane, int pairs, long long j0)
   {
#pragma unroll
      for(int k = 0; k < AHEAD; ++k) {
         const int pair = k * 32 + lane;   // a lane's sequence, lane % NS, is the same throughout
         const long long pos = len - 1 - (j0 + pair / NS);
         const unsigned at = (unsigned)max(0ll, pos) / (unsigned)p.page_size;
         const bool there = pair < pairs && pos >= 0 && at < (unsigned)p.max_pages;
         in[k] = there ? (int)((unsigned)pos - at * (unsigned)p.page_size) : -1;
         page[k] = __ldg(p.table + (there ? (b0 + lane % NS) * p.table_stride + at : 0));
      }
   }
   __device__ __forceinline__ void settle(const Pages& p, int b0, int len, int lane, int pairs, int filled, long long j0, int* rows) const
   {
      __syncwarp();
#pragma unroll
      for(int k = 0; k < AHEAD; ++k)
         if(k * 32 + lane < filled) rows[k * 32 + lane] = in[k] < 0 ? -1 : p.row(page[k], in[k]);
      for(int pair = AHEAD * 32 + lane; pair < filled; pair += 32) {
         const long long j = j0 + pair / NS;
         rows[pair] = pair < pairs && j < len ? p.slot(b0 + lane % NS, len - 1 - j) : -1;
      }
      __syncwarp();
   }
};

// The scales of a stage, [pair][block]: a lane takes W blocks of a row, BATCH
// rows at a time.  The first batch is loaded a stage ahead, and put into place
// when the slot is free.
template<int W, int BATCH> struct Scales {
   int each, at_once, mine, b0;   // 2^each lanes a row, rows at a time, this lane's row and its first block
   uint32_t raw[BATCH];
   int row[BATCH];
   __device__ __forceinline__ Scales(int blocks, int lane)
   {
      const int across = blocks / W;
      each = across <= 1 ? 0 : min(5, 32 - __clz(across - 1));
      at_once = 32 >> each;
      mine = lane >> each;
      b0 = (lane & ((1 << each) - 1)) * W;
   }
   __device__ __forceinline__ void load(const int* rows, const uint8_t* scales, int row_scales, int first, int b, int blocks, int pairs)
   {
#pragma unroll
      for(int k = 0; k < BATCH; ++k) {
         const int pair = first + k * at_once + mine;
         row[k] = pair < pairs && b < blocks ? rows[pair] : -2;
         const uint8_t* at = scales + (row[k] < 0 ? 0 : (long long)row[k] * row_scales + b);   // no condition: nothing to wait for
         if constexpr(W == 4) raw[k] = __ldg(reinterpret_cast<const unsigned int*>(at));
         else raw[k] = __ldg(at);
      }
   }
   // the entries' flags
   __device__ __forceinline__ uint32_t store(const uint32_t* entry, uint32_t* out, int first, int b, int blocks) const
   {
      uint32_t seen = 0;
#pragma unroll
      for(int k = 0; k < BATCH; ++k) {
         if(row[k] == -2) continue;
         uint32_t* to = out + (first + k * at_once + mine) * blocks + b;
         if constexpr(W == 4) {
            uint4 e = make_uint4(NO_ROW, NO_ROW, NO_ROW, NO_ROW);
            if(row[k] >= 0) e = make_uint4(entry[raw[k] & 255], entry[raw[k] >> 8 & 255], entry[raw[k] >> 16 & 255], entry[raw[k] >> 24]);
            seen |= e.x | e.y | e.z | e.w;
            *reinterpret_cast<uint4*>(to) = e;
         } else {
            const uint32_t e = row[k] >= 0 ? entry[raw[k]] : NO_ROW;
            seen |= e;
            *to = e;
         }
      }
      return seen;
   }
   // what the first batch has left
   __device__ __forceinline__ uint32_t rest(const int* rows, const uint32_t* entry, const uint8_t* scales, int row_scales, uint32_t* out,
                                            int blocks, int pairs)
   {
      uint32_t seen = 0;
      for(int base = 0; base < blocks; base += W << each)
         for(int first = base ? 0 : BATCH * at_once; first < pairs; first += BATCH * at_once) {
            load(rows, scales, row_scales, first, base + b0, blocks, pairs);
            seen |= store(entry, out, first, base + b0, blocks);
         }
      return seen;
   }
};

// The taps of a stage that blocks share, [lag][block], as numbers; sixteen loads under way.
template<class TT>
__device__ __forceinline__ void stage_taps(const TT* taps, long long stride, int c0, int group, float* out, int pitch, int blocks,
                                           int lags, int lane)
{
   const int each = blocks <= 1 ? 0 : min(5, 32 - __clz(blocks - 1)), at_once = 32 >> each, mine = lane >> each;
   for(int b = lane & ((1 << each) - 1); b < blocks; b += 1 << each) {
      const int head = (c0 + b * mx::BLOCK) / group;
      for(int first = mine; first < lags; first += 16 * at_once) {
         TT t[16];
#pragma unroll
         for(int k = 0; k < 16; ++k)
            if(first + k * at_once < lags) t[k] = taps[(first + k * at_once) * stride + head];
#pragma unroll
         for(int k = 0; k < 16; ++k)
            if(first + k * at_once < lags) out[(first + k * at_once) * pitch + b] = mx::to_f(t[k]);
      }
   }
}

// What a consumer does with its lags of a stage.  FAST: every scale a half; ALL: every row there too.
enum class Sum { ALL, FAST, ANY };
template<bool MX8, class TT, bool HEAD, int NB> struct Lag {   // what a thread reads of one lag
   uint32_t q[NB][MX8 ? 4 : 2], e[NB], t[HEAD ? 1 : CH * sizeof(TT) / 4];
   __device__ __forceinline__ void load(const uint8_t* at, uint32_t off, const uint8_t* codes, int row, const uint32_t* scales, int blocks)
   {
#pragma unroll
      for(int s = 0; s < NB; ++s) {
         e[s] = scales[s * blocks];
         if constexpr(MX8) {
            const uint4 x = *reinterpret_cast<const uint4*>(codes + s * row);
            q[s][0] = x.x; q[s][1] = x.y; q[s][2] = x.z; q[s][3] = x.w;
         } else {
            const uint2 x = *reinterpret_cast<const uint2*>(codes + s * row);
            q[s][0] = x.x; q[s][1] = x.y;
         }
      }
      if constexpr(HEAD) {
         t[0] = *reinterpret_cast<const uint32_t*>(at + off);
      } else {
         const uint32_t flip = (off >> 3) & 0x70;
#pragma unroll
         for(int k = 0; k < (int)(CH * sizeof(TT) / 16); ++k) {
            const uint4 x = *reinterpret_cast<const uint4*>(at + ((off + 16 * k) ^ flip));
            t[4 * k] = x.x; t[4 * k + 1] = x.y; t[4 * k + 2] = x.z; t[4 * k + 3] = x.w;
         }
      }
   }
   __device__ __forceinline__ float2 tap(int k) const
   {
      if constexpr(HEAD) return make_float2(__uint_as_float(t[0]), __uint_as_float(t[0]));
      else if constexpr(sizeof(TT) == 4) return make_float2(__uint_as_float(t[2 * k]), __uint_as_float(t[2 * k + 1]));
      else return mx::unpack2<__nv_bfloat16>(t[k]);
   }
   template<Sum HOW> __device__ __forceinline__ void sum(float2 (&acc)[NB][CH / 2]) const
   {
      float2 w[HEAD ? 1 : CH / 2];
#pragma unroll
      for(int k = 0; k < (HEAD ? 1 : CH / 2); ++k) w[k] = tap(k);
#pragma unroll
      for(int s = 0; s < NB; ++s) {
         if constexpr(HOW != Sum::ALL)
            if(e[s] & NO_ROW) continue;   // nothing, whatever the tap is
         uint32_t v[CH / 2];
         mx::Elem<MX8>::halves(q[s], v);
         if constexpr(HOW != Sum::ANY) {
#pragma unroll
            for(int k = 0; k < CH / 2; ++k) acc[s][k] = ffma2(widen_scaled(v[k], e[s]), w[HEAD ? 0 : k], acc[s][k]);
         } else {
            const float scale = mx::scale_value(e[s] >> 16 & 255);
#pragma unroll
            for(int k = 0; k < CH / 2; ++k) acc[s][k] = ffma2(fmul2(mx::half2_f(v[k]), make_float2(scale, scale)), w[HEAD ? 0 : k], acc[s][k]);
         }
      }
   }
};
// Where a thread's first lag lies in a stage, and its steps from lag to lag.
struct Path {
   uint32_t tap, tap_step;
   int codes, codes_step, row, scales, scales_step, blocks, slot, slots;
};
template<bool MX8, class TT, bool HEAD, int NB, Sum HOW>
__device__ __forceinline__ void sum_stage(const uint8_t* at, const Path& w, int count, float2 (&acc)[NB][CH / 2])
{
   using L = Lag<MX8, TT, HEAD, NB>;
   uint32_t tap = w.tap;
   const uint8_t* codes = at + w.codes;
   const uint32_t* scales = reinterpret_cast<const uint32_t*>(at + w.scales);
#pragma unroll 1
   for(int l = w.slot; l < count; l += w.slots, tap += w.tap_step, codes += w.codes_step, scales += w.scales_step) {
      L one;
      one.load(at, tap, codes, w.row, scales, w.blocks);
      one.template sum<HOW>(acc);
   }
}

template<class TT, bool HEAD, int NS, int W>
__device__ __forceinline__ void fill(const CUtensorMap* codes_map, const CUtensorMap* taps_map, const Pages& p, const Args& g, uint8_t* ring,
                                     uint64_t* full, uint64_t* empty, uint32_t* flags, const uint32_t* entry, int* found, int st,
                                     const Share share, int mine, int c0, int x, int blocks, int lane)
{
   const ConvStep& a = g.a;
   uint8_t* at = ring + st * g.stage_bytes;
   uint32_t* out = reinterpret_cast<uint32_t*>(at + g.scales_at);
   const uint8_t* scales = p.scales + c0 / mx::BLOCK;
   const int row_scales = a.channels / mx::BLOCK;
   Scales<W, HEAD ? 16 : 8> sc(blocks, lane);
   uint32_t phase = 1;
   bool ok = true;
   const auto first = [&](long long i) { return (share.worker + i * share.workers) * g.lags; };   // lag of stage i
   const auto held = [&](long long j0) { return (int)max(0ll, min((long long)g.lags, share.longest - j0)); };
   Rows<NS> next;
   const auto ask = [&](long long j0) { next.ask(p, share.b0, mine, lane, held(j0) * NS, j0); };
   // the rows of the stage whose pages were asked for, and its scales; the pages of the one after it
   const auto look_ahead = [&](long long i) {
      const long long j0 = first(i);
      next.settle(p, share.b0, mine, lane, held(j0) * NS, g.lags * NS, j0, found);
      sc.load(found, scales, row_scales, 0, sc.b0, blocks, held(j0) * NS);
      ask(first(i + g.stages));
   };
   ask(first(st));
   look_ahead(st);
   for(int i = st; i < share.n; i += g.stages, phase ^= 1) {
      const long long j0 = first(i);
      const int count = held(j0);
      if(!(ok = mbar_wait(empty + st, phase, g.status))) break;
      if(tc::elect()) {
         mbar_expect_tx(full + st, g.lags * (NS * g.row_bytes + (HEAD ? 0 : g.tap_bytes)));
         if(!HEAD) load_taps(taps_map, at, 0, c0 / (128 / (int)sizeof(TT)), (int)j0, full + st);
      }
      __syncwarp();
      for(int pair = lane * 4; pair < g.lags * NS; pair += 128)
         gather4(codes_map, at + g.codes_at + pair * g.row_bytes, x, *reinterpret_cast<const int4*>(found + pair), full + st);
      __syncwarp();
      uint32_t seen = sc.store(entry, out, 0, sc.b0, blocks);
      seen |= sc.rest(found, entry, scales, row_scales, out, blocks, count * NS);
      seen = __reduce_or_sync(0xffffffffu, seen) & (NO_HALF | NO_ROW);
      if constexpr(HEAD)
         stage_taps(static_cast<const TT*>(a.taps) + j0 * a.taps_stride, a.taps_stride, c0, a.group, reinterpret_cast<float*>(at),
                    g.tap_bytes / 4, blocks, count, lane);
      if(lane == 0) flags[st] = seen | (uint32_t)count;
      __syncwarp();
      if(lane == 0) tc::arrive_own(full + st);
      look_ahead((long long)i + g.stages);
   }
   if(!ok) {   // a wait gave up: time for the copies under way to land
      const uint64_t t0 = globaltimer_ns();
      while(globaltimer_ns() - t0 < 2000000ull) {}
   }
}

// TT: of the taps; HEAD: shared by blocks of 32 channels; NS sequences a CTA
template<bool MX8, class TT, bool HEAD, int NS>
__global__ void __launch_bounds__(THREADS, 1) conv_pipe_kernel(const __grid_constant__ CUtensorMap codes_map,
                                                               const __grid_constant__ CUtensorMap taps_map, Pages p, Args g)
{
   extern __shared__ uint8_t raw[];
   uint8_t* ring = reinterpret_cast<uint8_t*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
   __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES];
   __shared__ uint32_t flags[MAX_STAGES], entry[256];   // lags of a stage, with NO_HALF and NO_ROW where one of its scales has it
   __shared__ __align__(16) int rows[PRODUCERS][MAX_PAIRS];
   __shared__ int starts[MAX_GROUPS + 1];
   __shared__ Share share;
   const ConvStep& a = g.a;
   const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
   const int rank = a.split > 1 ? (int)tc::cluster_rank() : 0;
   const int c0 = blockIdx.y * a.lanes * CH;
   const int units = min(a.lanes, a.channels / CH - (int)blockIdx.y * a.lanes), blocks = units / 2;
   if(threadIdx.x == 0) {
      for(int s = 0; s < g.stages; ++s) {
         mbar_init(full + s, 2);
         mbar_init(empty + s, CONSUMERS);
      }
      fence_mbar_init();
      prefetch_tmap(&codes_map);
      if(!HEAD) prefetch_tmap(&taps_map);
   }
   if(threadIdx.x < 256) entry[threadIdx.x] = scale_entry(threadIdx.x);
   if(warp == CONSUMERS) {   // what this CTA does
      Share w{(int)blockIdx.z * NS, (int)blockIdx.x, a.split, 0, 0};
      if(g.pool) {
         const int groups = (p.batch + NS - 1) / NS;
         deal<NS>(a.lengths, p.batch, a.n_taps, g.lags, g.pool, lane, starts);
         __syncwarp();
         const int group = upper_bound(starts, groups, w.worker);
         if(group < groups) {
            w.b0 = group * NS;
            w.workers = starts[group + 1] - starts[group];
            w.worker -= starts[group];
         } else {
            w.b0 = -1;
         }
      }
      if(w.b0 >= 0) {
         const int mine = b_length<NS>(a, p, w.b0, lane);
         w.longest = min((int)__reduce_max_sync(0xffffffffu, (unsigned)mine), a.n_taps);
         const int tiles = (int)(((long long)w.longest + g.lags - 1) / g.lags);
         w.n = tiles > w.worker ? (tiles - 1 - w.worker) / w.workers + 1 : 0;
      }
      if(lane == 0) share = w;
   }
   __syncthreads();
   if(share.b0 < 0) return;   // nothing left for this CTA

   float2 acc[NS][CH / 2];
#pragma unroll
   for(int s = 0; s < NS; ++s)
#pragma unroll
      for(int i = 0; i < CH / 2; ++i) acc[s][i] = make_float2(0.0f, 0.0f);
   const int slots = a.slots, unit = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
   const bool sums = warp < CONSUMERS && slot < slots && unit < units;

   if(warp >= CONSUMERS) {
      // Finding a stage's rows, issuing its copies and reading its scales take a warp as long as several stages
      // take the sums, so several warps fill.  A slot of the ring is one warp's alone: a second one could wait
      // for the slot's next phase while the first still waits for this one, and take this one's parity for it.
      const int st = warp - CONSUMERS, x = (MX8 ? c0 : c0 / 2) / 4;
      if(st < g.stages) {
         const int mine = b_length<NS>(a, p, share.b0, lane);
         if(g.quads) fill<TT, HEAD, NS, 4>(&codes_map, &taps_map, p, g, ring, full, empty, flags, entry, rows[st], st, share, mine, c0, x, blocks, lane);
         else fill<TT, HEAD, NS, 1>(&codes_map, &taps_map, p, g, ring, full, empty, flags, entry, rows[st], st, share, mine, c0, x, blocks, lane);
      }
   } else {
      Path w;
      w.slot = slot;
      w.slots = slots;
      w.blocks = blocks;
      w.row = g.row_bytes;
      w.tap = slot * g.tap_bytes + (HEAD ? unit / 2 * 4 : unit * (CH * (int)sizeof(TT)));
      w.tap_step = slots * g.tap_bytes;
      w.codes = g.codes_at + slot * NS * g.row_bytes + unit * (MX8 ? CH : CH / 2);
      w.codes_step = slots * NS * g.row_bytes;
      w.scales = g.scales_at + (slot * NS * blocks + unit / 2) * 4;
      w.scales_step = slots * NS * blocks;
      int st = 0;
      uint32_t phase = 0;
      const uint8_t* at = ring;
      for(int i = 0, n = share.n; i < n; ++i) {
         if(!mbar_wait(full + st, phase, g.status)) break;
         const uint32_t f = flags[st];
         const int count = f & 0xffff;
         if(sums) {
            if(f <= 0xffff) sum_stage<MX8, TT, HEAD, NS, Sum::ALL>(at, w, count, acc);
            else if(!(f & NO_HALF)) sum_stage<MX8, TT, HEAD, NS, Sum::FAST>(at, w, count, acc);
            else sum_stage<MX8, TT, HEAD, NS, Sum::ANY>(at, w, count, acc);
         }
         __syncwarp();
         if(lane == 0) tc::arrive_own(empty + st);
         at += g.stage_bytes;
         if(++st == g.stages) {
            st = 0;
            phase ^= 1;
            at = ring;
         }
      }
   }
   __syncthreads();   // the ring is done with: every stage that was filled has been waited for
   float* joined = reinterpret_cast<float*>(ring);
   if(warp < CONSUMERS && slot < slots) park<NS>(joined, acc, slot, unit, slots, a.lanes);
   join<NS>(joined, a, p, a.lanes * CH, slots, THREADS, rank, share.b0, c0, (long long)blockIdx.x * NS);
}

struct Plan {
   int ns, lanes, chunks, slots, split, pool, lags, stages;
   int row_bytes, tap_bytes, codes_at, scales_at, stage_bytes;
   size_t partials(int channels) const { return (size_t)pool * ns * channels * sizeof(float); }
};
constexpr int SMEM = 200 * 1024;

// false: not this way.  tap_size: bytes of a tap, 0 where heads share them
bool plan(long long lags, bool mx8, int channels, int batch, int tap_size, int sms, Plan* p)
{
   constexpr int grain = 4;   // units of a chunk: 128 bytes of taps, and of four rows of codes
   const int units = channels / CH;
   if(units % grain || units * (mx8 ? CH : CH / 2) < 256 || lags < 64) return false;
   p->ns = batch > 2 ? 4 : batch;
   const long long groups = mx::ceil_div(batch, p->ns);
   // A cluster of eight joins short histories in the same launch; long ones
   // are dealt to as many CTAs as the card takes at once, and joined by a
   // second launch (MX4 x 2048, one sequence of 32768 and 15 of 100: an equal
   // share for each group 194 us, dealt 73).
   const double value = mx8 ? 33.0 / 32 : 17.0 / 32;
   const bool small = (double)lags * channels * (batch * value + tap_size) < 64.0 * (1 << 20);
   // scales that have to be read byte by byte are worth it for long histories only (us, ring / direct: 5 ragged to
   // 5000 x 2112 MX4, 3001 taps of 22 heads 53.2 / 13.0; 1 x 5000 x 2112, a filter a channel 16.4 / 12.1; 4 x 2000 x 1088 MX8
   // 23.0 / 16.4)
   if(small && channels % 128) return false;
   const auto lay = [&](int chunks) {
      p->lanes = (int)mx::ceil_div(mx::ceil_div(units, chunks), grain) * grain;
      p->chunks = (int)mx::ceil_div(units, p->lanes);
      const int most = small ? MAX_SPLIT : groups > MAX_GROUPS ? 1 : (int)mx::ceil_div(lags, 256);
      int w = (int)std::max<long long>(1, std::min<long long>(most, sms / (p->chunks * groups)));
      if(small)
         while(w & (w - 1)) w &= w - 1;   // clusters of 1, 2, 4 or 8
      p->split = small ? w : 1;
      p->pool = small || w == 1 ? 0 : (int)std::min<long long>(most * groups, sms / p->chunks);
      p->row_bytes = p->lanes * (mx8 ? CH : CH / 2);
      p->tap_bytes = tap_size ? p->lanes * CH * tap_size : p->lanes / 2 * 4;
      const int per_lag = p->tap_bytes + p->ns * (p->row_bytes + p->lanes / 2 * 4);
      p->lags = 8;
      // the scales of a stage are loaded in batches, one after the other where they are read byte by byte
      const int rows = channels % 128 == 0 && p->lanes % 8 == 0 ? MAX_PAIRS : 64;
      while(p->lags < 64 && p->lags * 2 * per_lag <= 44 * 1024 && p->lags * 2 * p->ns <= rows && lags >= (long long)p->lags * 4 * w)
         p->lags *= 2;
      p->slots = std::min(p->lags, CONSUMERS * 32 / p->lanes);
      p->codes_at = (int)mx::ceil_div(p->lags * p->tap_bytes, 128) * 128;
      p->scales_at = p->codes_at + p->lags * p->ns * p->row_bytes;
      p->stage_bytes = (int)mx::ceil_div(p->lags * per_lag + 128, 1024) * 1024;
      p->stages = std::min(MAX_STAGES, SMEM / p->stage_bytes);
      return p->pool ? (long long)p->chunks * p->pool : p->chunks * groups * w;   // CTAs
   };
   // chunks of 1024 channels, or of fewer where the card would not be full or the ring not four stages long
   int chunks = (int)mx::ceil_div(units, 64);
   while((lay(chunks) < sms * 3 / 4 || p->stages < 4) && units / (chunks * 2) >= 2 * grain) chunks *= 2;
   lay(chunks);
   return p->stages >= 3;
}

size_t smem_of(const Plan& p)
{
   const size_t ring = (size_t)p.stages * p.stage_bytes, sums = (size_t)p.ns * p.slots * p.lanes * CH * sizeof(float);
   return std::max(ring, sums) + 1024;
}

template<bool MX8, class TT, bool HEAD, int NS>
fufft_status launch(const fufft_cache* c, const Args& g, const CUtensorMap& cm, const CUtensorMap& tm, const Plan& p, cudaStream_t st)
{
   auto kern = conv_pipe_kernel<MX8, TT, HEAD, NS>;
   static std::atomic<uint64_t> configured{0};
   fufft_status s = allow_smem(kern, SMEM + 1024, configured);
   if(s != FUFFT_OK) return s;
   cudaLaunchConfig_t cfg = {};
   cfg.gridDim = dim3((unsigned)(p.pool ? p.pool : p.split), (unsigned)p.chunks, p.pool ? 1u : (unsigned)mx::ceil_div(c->batch, NS));
   cfg.blockDim = dim3(THREADS);
   cfg.dynamicSmemBytes = smem_of(p);
   cfg.stream = st;
   cudaLaunchAttribute at[1];
   at[0].id = cudaLaunchAttributeClusterDimension;
   at[0].val.clusterDim.x = (unsigned)p.split;
   at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
   cfg.attrs = at;
   cfg.numAttrs = 1;
   if((s = check(cudaLaunchKernelEx(&cfg, kern, cm, tm, Pages(c), g))) != FUFFT_OK) return s;
   count_launch();
   if(!p.pool) return FUFFT_OK;
   join_dealt_kernel<NS><<<(unsigned)mx::ceil_div((long long)c->batch * c->channels, 256), 256, 0, st>>>(g.a, c->batch, p.lags, p.pool);
   count_launch();
   return check(cudaGetLastError());
}
template<bool MX8, class TT, bool HEAD>
fufft_status launch(const fufft_cache* c, const Args& g, const CUtensorMap& cm, const CUtensorMap& tm, const Plan& p, cudaStream_t st)
{
   return p.ns == 4 ? launch<MX8, TT, HEAD, 4>(c, g, cm, tm, p, st)
                    : p.ns == 2 ? launch<MX8, TT, HEAD, 2>(c, g, cm, tm, p, st) : launch<MX8, TT, HEAD, 1>(c, g, cm, tm, p, st);
}
template<bool MX8, class TT>
fufft_status launch(const fufft_cache* c, const Args& g, bool shared, const CUtensorMap& cm, const CUtensorMap& tm, const Plan& p,
                    cudaStream_t st)
{
   return shared ? launch<MX8, TT, true>(c, g, cm, tm, p, st) : launch<MX8, TT, false>(c, g, cm, tm, p, st);
}

// taps as [lag][128 bytes][...]: boxes of a stage's lags and a chunk's channels, the 16-byte chunks of the
// 128-byte rows permuted; lags beyond the last read as zeros
fufft_status taps_tmap(CUtensorMap* tm, const ConvStep& a, int tap_size, const Plan& p)
{
   cuuint64_t dims[3] = {(cuuint64_t)(128 / tap_size), (cuuint64_t)(a.channels * tap_size / 128), (cuuint64_t)a.n_taps};
   cuuint64_t strides[2] = {128, (cuuint64_t)a.taps_stride * tap_size};
   cuuint32_t box[3] = {(cuuint32_t)(128 / tap_size), (cuuint32_t)(p.tap_bytes / 128), (cuuint32_t)p.lags};
   return encode_tmap(tm, tap_size == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, a.taps, dims,
                      strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// the cache's rows of codes, a box of one row's chunk
fufft_status codes_tmap(CUtensorMap* tm, const fufft_cache* c, const Plan& p)
{
   const long long row = c->kind == FUFFT_CACHE_MX8 ? c->channels : c->channels / 2;
   const cuuint64_t dims[2] = {(cuuint64_t)row / 4, (cuuint64_t)c->pages * c->page_size}, strides[1] = {(cuuint64_t)row};
   const cuuint32_t box[2] = {(cuuint32_t)p.row_bytes / 4, 1};
   return encode_tmap(tm, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, c->codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}
}  // namespace pipe

// How the work is laid out, from the sizes alone.
struct Plan {
   int nb, lanes, chunks, slots, split, outer, tile;
};
Plan plan(long long lags, int channels, int batch, int sms)
{
   Plan p;
   lags = lags > 0 ? lags : 1;
   const int units = channels / CH;
   // clusters along the lags while a CTA keeps 32 of them
   p.split = 1;
   while(p.split < MAX_SPLIT && lags >= 64ll * p.split) p.split *= 2;
   // Channels in as few chunks as give four CTAs per SM, a chunk not below 256 channels; fewer sequences that share
   // their taps where that leaves SMs without a pair of CTAs.
   for(p.nb = batch > 2 ? 4 : batch;; p.nb /= 2) {
      const long long groups = mx::ceil_div(batch, p.nb);
      p.chunks = (int)mx::ceil_div(units, THREADS);
      while(p.chunks * groups * p.split < 4ll * sms && mx::ceil_div(units, p.chunks * 2) >= 16) p.chunks *= 2;
      p.lanes = (int)mx::ceil_div(units, p.chunks);
      p.chunks = (int)mx::ceil_div(units, p.lanes);
      p.slots = THREADS / p.lanes;
      p.outer = 1;
      while(p.chunks * groups * p.split * p.outer < 2ll * sms && lags >= 2048ll * p.split * p.outer) p.outer *= 2;
      if(p.nb == 1 || p.chunks * groups * p.split * p.outer >= 2ll * sms) break;
   }
   // the same number of tiles for every CTA
   const long long workers = (long long)p.split * p.outer, tiles = mx::ceil_div(lags, workers * TILE);
   p.tile = (int)mx::ceil_div(lags, workers * tiles);
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
   return FUFFT_OK;
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

// bytes of the partial results of `outer` clusters
size_t partials(int outer, const fufft_cache* c)
{
   return outer == 1 ? 0 : (size_t)outer * c->batch * c->channels * sizeof(float);
}

fufft_status join_clusters(const ConvStep& a, int batch, cudaStream_t st)
{
   conv_join_kernel<<<(unsigned)mx::ceil_div((long long)batch * a.channels, 256), 256, 0, st>>>(a, batch);
   count_launch();
   return check(cudaGetLastError());
}

}  // namespace cache
}  // namespace fufft

extern "C" {

size_t fufft_cache_conv_workspace(const fufft_cache* c, int64_t n_taps)
{
   if(cache::check_cache(c) != FUFFT_OK || n_taps < 0 || n_taps > cache::MAX_TOKENS || c->batch == 0) return 0;
   int dev = 0;
   if(cudaGetDevice(&dev) != cudaSuccess) return 0;
   const long long lags = cache::lags_of(c, n_taps);
   const int sms = sm_count(dev);
   size_t need = cache::partials(cache::plan(lags, c->channels, c->batch, sms).outer, c);
   cache::pipe::Plan p;   // whichever way the taps will lie
   for(int tap_size : {0, 2, 4})
      if(cache::pipe::plan(lags, c->kind == FUFFT_CACHE_MX8, c->channels, c->batch, tap_size, sms, &p)) need = std::max(need, p.partials(c->channels));
   return need;
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
   cache::ConvStep a{};
   a.lengths = lengths;
   a.taps = taps;
   a.taps_stride = taps_stride;
   a.n_taps = c->pages > 0 ? (int)n_taps : 0;   // without a page there is no row
   a.group = c->channels / heads;
   a.channels = c->channels;
   a.gate = gate;
   a.gate_stride = gate_stride;
   a.out = out;
   a.out_stride = out_stride;
   a.dtype = dtype;
   const int tap_size = taps_dtype == FUFFT_F32 ? 4 : 2;
   a.vec_taps = aligned(taps, 16) && taps_stride * tap_size % 16 == 0;
   const bool mx8 = c->kind == FUFFT_CACHE_MX8;
   const long long lags = cache::lags_of(c, n_taps);
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);

   // long rows, taps that a tensor copy takes or that whole blocks share: the ring
   cache::pipe::Plan pp;
   const bool shared = a.group % mx::BLOCK == 0;
   if((shared || (a.group == 1 && a.vec_taps)) &&
      c->pages > 0 && cache::pipe::plan(lags, mx8, c->channels, c->batch, shared ? 0 : tap_size, sm_count(dev), &pp)) {
      const size_t need = pp.partials(c->channels);
      if(workspace_bytes < need || (need && !workspace)) return FUFFT_ERR_INVALID_ARG;
      DeviceCtx ctx;
      if((s = device_ctx(&ctx)) != FUFFT_OK) return s;
      a.partial = need ? static_cast<float*>(workspace) : nullptr;
      a.lanes = pp.lanes;
      a.slots = pp.slots;
      a.split = pp.split;
      CUtensorMap tm{}, cm;
      if((s = cache::pipe::codes_tmap(&cm, c, pp)) != FUFFT_OK) return s;
      if(!shared && (s = cache::pipe::taps_tmap(&tm, a, tap_size, pp)) != FUFFT_OK) return s;
      const cache::pipe::Args g{a, ctx.status, pp.lags, pp.stages, pp.stage_bytes, pp.codes_at, pp.scales_at, pp.row_bytes, pp.tap_bytes, pp.pool,
                                c->channels % 128 == 0 && pp.lanes % 8 == 0};
      if(mx8) s = tap_size == 4 ? cache::pipe::launch<true, float>(c, g, shared, cm, tm, pp, st) : cache::pipe::launch<true, __nv_bfloat16>(c, g, shared, cm, tm, pp, st);
      else s = tap_size == 4 ? cache::pipe::launch<false, float>(c, g, shared, cm, tm, pp, st) : cache::pipe::launch<false, __nv_bfloat16>(c, g, shared, cm, tm, pp, st);
      return s;
   }
   const cache::Plan p = cache::plan(lags, c->channels, c->batch, sm_count(dev));
   const size_t need = cache::partials(p.outer, c);
   if(workspace_bytes < need || (need && !workspace)) return FUFFT_ERR_INVALID_ARG;
   a.partial = need ? static_cast<float*>(workspace) : nullptr;
   a.lanes = p.lanes;
   a.slots = p.slots;
   a.split = p.split;
   a.outer = p.outer;
   a.tile = p.tile;
   if(mx8) s = tap_size == 4 ? cache::launch<true, float>(c, a, p, st) : cache::launch<true, __nv_bfloat16>(c, a, p, st);
   else s = tap_size == 4 ? cache::launch<false, float>(c, a, p, st) : cache::launch<false, __nv_bfloat16>(c, a, p, st);
   return s != FUFFT_OK || p.outer == 1 ? s : cache::join_clusters(a, c->batch, st);
}

}  // extern "C"
