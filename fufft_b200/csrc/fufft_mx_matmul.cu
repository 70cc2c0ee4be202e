// fufft_mx_matmul.cu -- product of two 4-bit microscaled matrices,
// out[m][n] = sum_k a[m][k] b[n][k] + bias[n], on the tensor cores
// (tcgen05 kind::mxf4: E2M1 products under E8M0 scales, fp32 sums in tensor
// memory).
#include <algorithm>
#include <type_traits>

#include "fufft_internal.cuh"
#include "fufft_mx.cuh"
#include "fufft_tc.cuh"

using namespace fufft;
using namespace fufft::host;

namespace fufft {
namespace mx {

struct MatmulArgs {
   const uint8_t *p_scale, *q_scale;
   const float* bias;
   void* out;
   unsigned int* status;
   long long p_rows, q_rows, out_stride;
   int chunks;               // 256-column chunks of the summed axis
   int tiles_p, split;
};

// ---------------------------------------------------------------------------
// Few outputs (one token up to a small batch): the CTA's 128 tensor-memory
// lanes are 128 rows of b, its BN columns rows of a, so that a single token
// still streams b at full width, and CTAs of a cluster take parts of the
// summed axis and join their sums through distributed shared memory, in rank
// order.  Bound by reading b's codes and scales once.
//
// Rows that are not quantised yet (Raw<X>, four at most) are quantised on the
// way: two warps that have nothing else to do put each stage's 256 columns
// into the layout that the copies would have left, in every CTA that needs
// them.  It saves a launch on the host (15.5 -> 9.6 us a call) and costs the
// GPU nothing (us, inside / before: one token 4096 x 4096 5.8 / 6.7, 8192 x
// 8192 8.1 / 8.7); sixteen rows would take the two warps longer than the
// product (8192 x 8192 18.2 / 8.8).
// ---------------------------------------------------------------------------
struct Packed {};              // a comes in codes and scales
template<class X> struct Raw {};   // a comes as rows of X
struct RawArgs {
   const void* x;
   long long stride, cols;
   bool on_32;
};

constexpr int MAX_SPLIT = 8;         // CTAs of a portable cluster
template<int BN> struct Split {
   static constexpr int SF_Q = (BN + 127) / 128;                     // scale tiles of the columns
   static constexpr int P_BYTES = 128 * 128, Q_BYTES = BN * 128, SF_BYTES = 1024;
   static constexpr int STAGE = P_BYTES + Q_BYTES + SF_BYTES * (1 + SF_Q);
   static constexpr int STAGES = BN <= 16 ? 5 : BN <= 64 ? 4 : 3;
   static constexpr int SF_COLS = 8 + 8 * SF_Q;                      // tensor-memory columns of a stage's scales
   static constexpr int NEED = BN + STAGES * SF_COLS;
   static constexpr int TMEM = NEED <= 128 ? 128 : NEED <= 256 ? 256 : 512;
   static constexpr int PITCH = 132;                                 // of a partial column, in floats
   static constexpr int JOIN = BN * PITCH * 4;
   static constexpr int BODY = STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN;
   static constexpr int SMEM = BODY + 1024 + 128;
   static_assert(STAGE % 1024 == 0, "the 128-byte swizzle repeats every 1024 bytes");
};

// The unquantised rows, by 64 threads: a thread takes half a block of a stage,
// two neighbouring lanes a block.  Four stages' loads are under way ahead of
// the one that is encoded.
template<class X> struct Turn {
   Half<X> h;
   __device__ __forceinline__ void load(const RawArgs& r, int rows, int row, long long col)
   {
      const int count = row < rows ? (int)max(0ll, min((long long)HALF, r.cols - col)) : 0;
      const X* at = static_cast<const X*>(r.x) + row * r.stride + col;
      if(r.on_32 && count == HALF) h.load(at);
      else h.load_some(at, count);
   }
   __device__ __forceinline__ void store(uint8_t* codes, uint8_t* scales, int row, int half) const
   {
      uint32_t q[2];
      const uint32_t s = encode_pair<false>(h, q);
      // 128-byte rows whose 16-byte chunks are permuted by the row, as the copies' swizzle leaves them
      *reinterpret_cast<uint2*>(codes + row * 128 + ((half >> 1 ^ (row & 7)) << 4) + (half & 1) * 8) = make_uint2(q[0], q[1]);
      if((half & 1) == 0) scales[(half >> 3) * TILE_BYTES + tile_word(row) + (half >> 1 & 3)] = (uint8_t)s;
   }
};
template<class A> struct RowType { using type = float; };
template<class X> struct RowType<Raw<X>> { using type = X; };

template<class T, int BN, class A>
__global__ void __launch_bounds__(128) matmul_split_kernel(const __grid_constant__ CUtensorMap tp,
                                                           const __grid_constant__ CUtensorMap tq, MatmulArgs g, RawArgs x)
{
   using C = Split<BN>;
   constexpr bool PACKED = std::is_same_v<A, Packed>;
   static_assert(PACKED || BN == 16, "four rows at most are quantised here");
   extern __shared__ uint8_t raw[];
   uint8_t* body = reinterpret_cast<uint8_t*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
   uint64_t* full = reinterpret_cast<uint64_t*>(body + C::BODY);
   uint64_t* empty = full + C::STAGES;
   uint64_t* done = empty + C::STAGES;
   uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);

   const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
   const int rank = g.split > 1 ? (int)tc::cluster_rank() : 0;
   const long long tile = blockIdx.x / g.split;
   const int p0 = (int)(tile % g.tiles_p) * 128;
   const long long q0 = tile / g.tiles_p * BN;
   const int per = (g.chunks + g.split - 1) / g.split;
   const int k0 = min(rank * per, g.chunks), k1 = min(k0 + per, g.chunks), n = k1 - k0;

   if(threadIdx.x == 0) {
      for(int s = 0; s < C::STAGES; ++s) {
         mbar_init(full + s, PACKED ? 1 : 3);
         mbar_init(empty + s, 1);
      }
      mbar_init(done, 1);
      fence_mbar_init();
      if(n > 0) {   // with nothing to sum there are no maps
         prefetch_tmap(&tp);
         prefetch_tmap(&tq);
      }
   }
   if(warp == 2) tc::tmem_alloc<C::TMEM>(tmem_at);
   tc::fence_before_sync();
   __syncthreads();
   tc::fence_after_sync();
   const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);

   if(warp == 0) {
      // copies: both operands' 256 columns and their scales, one stage each
      const long long q_tile_last = ceil_div(g.q_rows, TILE_ROWS) - 1;
      const uint8_t* p_scale = g.p_scale + ((long long)(p0 / TILE_ROWS) * g.chunks + k0) * C::SF_BYTES;
      const uint8_t* q_scale = g.q_scale + (q0 / TILE_ROWS * g.chunks + k0) * C::SF_BYTES;
      auto load_p = [&](int i, int s) {
         mbar_expect_tx(full + s, PACKED ? C::STAGE : C::P_BYTES + C::SF_BYTES);
         tma_load_2d(body + s * C::STAGE, &tp, (k0 + i) * 128, p0, full + s);
         bulk_g2s(body + s * C::STAGE + C::P_BYTES + C::Q_BYTES, p_scale + (long long)i * C::SF_BYTES, C::SF_BYTES, full + s);
      };
      auto load_q = [&](int i, int s) {
         uint8_t* at = body + s * C::STAGE + C::P_BYTES;
         tma_load_2d(at, &tq, (k0 + i) * 128, (int)q0, full + s);
#pragma unroll
         for(int h = 0; h < C::SF_Q; ++h)
            bulk_g2s(at + C::Q_BYTES + (1 + h) * C::SF_BYTES,
                     q_scale + (min((long long)h, q_tile_last - q0 / TILE_ROWS) * g.chunks + i) * C::SF_BYTES, C::SF_BYTES, full + s);
      };
      // b's first stages are under way before a's quantisation, the kernel before, has ended
      const int ahead = min(n, C::STAGES);
      if(tc::elect())
         for(int i = 0; i < ahead; ++i) load_p(i, i);
      if constexpr(PACKED) {
         tc::wait_for_previous();
         if(tc::elect())
            for(int i = 0; i < ahead; ++i) load_q(i, i);
      }
      __syncwarp();
      int issued = ahead, s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for(int i = ahead; i < n; ++i) {
         if(!mbar_wait(empty + s, phase, g.status)) {
            ok = false;
            break;
         }
         if(tc::elect()) {
            load_p(i, s);
            if(PACKED) load_q(i, s);
         }
         __syncwarp();
         issued = i + 1;
         if(++s == C::STAGES) {
            s = 0;
            phase ^= 1;
         }
      }
      // after a wait that gave up: no copy may still be landing when the CTA ends
      if(!ok)
         for(int i = max(0, issued - C::STAGES); i < issued; ++i) mbar_wait(full + i % C::STAGES, i / C::STAGES & 1, g.status);
   } else if(warp == 1 && n > 0) {
      const uint32_t q_col = (uint32_t)(q0 % TILE_ROWS / 32);       // this tile's first scale column of its row tile
      const uint64_t rows0 = tc::rows_desc(smem_u32(body)), scales0 = tc::scales_desc(smem_u32(body) + C::P_BYTES + C::Q_BYTES);
      int s = 0;
      uint32_t phase = 0;
      for(int i = 0; i < n; ++i) {
         if(!mbar_wait(full + s, phase, g.status)) break;
         tc::fence_after_sync();
         const uint64_t rows = rows0 + (uint32_t)(s * (C::STAGE >> 4)), sf = scales0 + (uint32_t)(s * (C::STAGE >> 4));
         const uint32_t col = tmem + BN + s * C::SF_COLS;
         if(tc::elect()) {
#pragma unroll
            for(int t = 0; t < 2; ++t) {
               tc::copy_scales(col + t * 4, sf + t * (TILE_BYTES >> 4));
#pragma unroll
               for(int h = 0; h < C::SF_Q; ++h)
                  tc::copy_scales(col + 8 + (t * C::SF_Q + h) * 4, sf + (((1 + h) * C::SF_BYTES + t * TILE_BYTES) >> 4));
            }
#pragma unroll
            for(int k = 0; k < 4; ++k)
               tc::mma_mxf4(tmem, rows + k * 2, rows + ((C::P_BYTES + k * 32) >> 4), tc::mxf4_idesc(128, BN, (k & 1) * 2),
                            col + (k >> 1) * 4, col + 8 + (k >> 1) * C::SF_Q * 4 + q_col, i > 0 || k > 0);
            tc::commit(empty + s);
         }
         __syncwarp();
         if(++s == C::STAGES) {
            s = 0;
            phase ^= 1;
         }
      }
      if(tc::elect()) tc::commit(done);
   } else if(!PACKED && warp >= 2) {
      const int row = threadIdx.x >> 4 & 3, half = threadIdx.x & 15;
      const long long col = (long long)k0 * K_PAD + half * HALF;
      Turn<typename RowType<A>::type> ahead[4];
#pragma unroll
      for(int q = 0; q < 4; ++q)
         if(q < n) ahead[q].load(x, (int)g.q_rows, row, col + (long long)q * K_PAD);
      int s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for(int i = 0; i < n && ok; i += 4) {
#pragma unroll
         for(int q = 0; q < 4; ++q) {
            if(i + q >= n || !(ok = mbar_wait(empty + s, phase, g.status))) break;
            uint8_t* at = body + s * C::STAGE + C::P_BYTES;
            ahead[q].store(at, at + C::Q_BYTES + C::SF_BYTES, row, half);
            if(i + q + 4 < n) ahead[q].load(x, (int)g.q_rows, row, col + (long long)(i + q + 4) * K_PAD);
            fence_proxy_async_smem();
            __syncwarp();
            if(lane == 0) tc::arrive_own(full + s);
            if(++s == C::STAGES) {
               s = 0;
               phase ^= 1;
            }
         }
      }
   }
   __syncwarp();
   bool ok = n == 0 || mbar_wait(done, 0, g.status);
   tc::fence_after_sync();
   // lane = row p0 + 32 warp + lane of b, column j = row q0 + j of a
   const uint32_t mine = tmem + ((uint32_t)warp << 21);
   const int line = warp * 32 + lane;
   T* out = static_cast<T*>(g.out);
   if(g.split == 1) {
      const long long row = p0 + line;
      const float bias = g.bias && row < g.p_rows ? g.bias[row] : 0.0f;
#pragma unroll
      for(int j0 = 0; j0 < BN; j0 += 16) {
         float v[16];
         tc::tmem_load16(mine + j0, v);
         tc::tmem_load_wait();
#pragma unroll
         for(int j = 0; j < 16; ++j)
            if(ok && row < g.p_rows && q0 + j0 + j < g.q_rows)
               out[(q0 + j0 + j) * g.out_stride + row] = from_f<T>((n ? v[j] : 0.0f) + bias);
      }
   } else {
      float* part = reinterpret_cast<float*>(body);   // every copy has landed and been used: `done`
#pragma unroll
      for(int j0 = 0; j0 < BN; j0 += 16) {
         float v[16];
         tc::tmem_load16(mine + j0, v);
         tc::tmem_load_wait();
#pragma unroll
         for(int j = 0; j < 16; ++j) part[(j0 + j) * C::PITCH + line] = n && ok ? v[j] : 0.0f;
      }
      tc::cluster_sync();
      // a warp takes a column, a lane four rows of b: the ranks' sums are loaded side by side, added in order
      const int rows = (int)min((long long)BN, g.q_rows - q0);
      const long long row = p0 + lane * 4;
      for(int j = rank * 4 + warp; j < rows; j += g.split * 4) {
         float4 v[MAX_SPLIT];
#pragma unroll
         for(int r = 0; r < MAX_SPLIT; ++r)
            if(r < g.split) v[r] = tc::load_peer4(tc::peer_smem(part + j * C::PITCH + lane * 4, r));
         float4 sum = v[0];
#pragma unroll
         for(int r = 1; r < MAX_SPLIT; ++r)
            if(r < g.split) {
               sum.x += v[r].x;
               sum.y += v[r].y;
               sum.z += v[r].z;
               sum.w += v[r].w;
            }
         const float y[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
         for(int x = 0; x < 4; ++x)
            if(row + x < g.p_rows) out[(q0 + j) * g.out_stride + row + x] = from_f<T>(y[x] + (g.bias ? g.bias[row + x] : 0.0f));
      }
      tc::cluster_sync();   // nobody leaves while its sums are being read
   }
   tc::fence_before_sync();
   __syncthreads();
   if(warp == 2) tc::tmem_free<C::TMEM>(tmem);
}

// ---------------------------------------------------------------------------
// Many outputs: pairs of CTAs, 256 rows of one operand by BN of the other a
// tile, each CTA holding half of both; a pair walks over tiles.  One warp
// copies, one issues, eight bring the finished sums out.  The 256 rows
// (tensor-memory lanes) are a's, and a warp hands tiles of 32 rows x 128 bytes
// to tensor copies, where the rows of the result start on 16 bytes (8192 x
// 4096 x 256 bf16, all of it storing: stores of whole sectors from the lanes
// 29.6 us, tensor copies 14.3, no stores at all 10.5); else the 256 rows are b's (SWAP), and
// the lanes of a warp store side by side, aligned or not.
// ---------------------------------------------------------------------------
template<int BN_, int ACC_> struct Pair {
   static constexpr int BN = BN_, ACC = ACC_;                        // columns of a tile; accumulators
   static constexpr int STAGES = 5;
   static constexpr int A_BYTES = 128 * 128, B_BYTES = BN / 2 * 128, SF_BYTES = 1024;
   static constexpr int STAGE = A_BYTES + B_BYTES + 3 * SF_BYTES;    // scales: 128 rows of a, 256 rows of b
   static constexpr int SF_COLS = 24;
   static constexpr int SF_AT = ACC * BN;
   static constexpr int TMEM = 512;
   static constexpr int THREADS = 320, EPILOGUE = 8, OUT = 32 * 128;  // bytes of a warp's tile on its way out
   static constexpr int SMEM = STAGES * STAGE + EPILOGUE * OUT + 1024 + 256;
   static constexpr int COLS = 128;                                  // a warp brings out 32 x 128, or what is left of BN
   static constexpr int GROUP = 8;                                   // row tiles that are walked together
   static_assert(STAGE % 1024 == 0 && SF_AT + STAGES * SF_COLS <= TMEM && BN % 64 == 0 && BN > 128 && BN <= 256, "tile");
};

struct PairArgs {
   const float* bias;
   void* out;
   unsigned int* status;
   long long m, n, out_stride;
   int chunks, tiles_m, tiles_n;
};

template<class P> __device__ __forceinline__ void pair_tile(const PairArgs& g, long long t, int* m0, int* n0)
{
   const long long per = (long long)P::GROUP * g.tiles_n;
   const int first = (int)(t / per) * P::GROUP, rows = min(P::GROUP, g.tiles_m - first);
   const int in = (int)(t % per);
   *m0 = (first + in % rows) * 256;
   *n0 = in / rows * P::BN;
}

template<class T, class P, bool SWAP>
__global__ void __launch_bounds__(P::THREADS, 1) matmul_pair_kernel(const __grid_constant__ CUtensorMap ta,
                                                                    const __grid_constant__ CUtensorMap tb,
                                                                    const __grid_constant__ CUtensorMap tsa,
                                                                    const __grid_constant__ CUtensorMap tsb,
                                                                    const __grid_constant__ CUtensorMap tout, PairArgs g)
{
   extern __shared__ uint8_t raw[];
   uint8_t* body = reinterpret_cast<uint8_t*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
   uint8_t* leaving = body + P::STAGES * P::STAGE;
   uint64_t* full = reinterpret_cast<uint64_t*>(leaving + P::EPILOGUE * P::OUT);   // in the even CTA: both halves have landed
   uint64_t* empty = full + P::STAGES;                                         // in each: the products have read the stage
   uint64_t* ready = empty + P::STAGES;                                        // in each: an accumulator is summed
   uint64_t* taken = ready + P::ACC;                                           // in the even CTA: both have read it
   uint32_t* tmem_at = reinterpret_cast<uint32_t*>(taken + P::ACC);

   const int warp = tc::uniform_warp(), lane = threadIdx.x & 31;
   const uint32_t rank = tc::cluster_rank();
   const long long tiles = (long long)g.tiles_m * g.tiles_n, first = blockIdx.x >> 1, step = gridDim.x >> 1;

   if(threadIdx.x == 0) {
      for(int s = 0; s < P::STAGES; ++s) {
         mbar_init(full + s, 1);
         mbar_init(empty + s, 1);
      }
      for(int s = 0; s < P::ACC; ++s) {
         mbar_init(ready + s, 1);
         mbar_init(taken + s, 2 * P::EPILOGUE);
      }
      fence_mbar_init();
      prefetch_tmap(&ta);
      prefetch_tmap(&tb);
      prefetch_tmap(&tsa);
      prefetch_tmap(&tsb);
   }
   if(warp == 1) tc::tmem_alloc_pair<P::TMEM>(tmem_at);
   tc::fence_before_sync();
   tc::cluster_sync();
   tc::fence_after_sync();
   const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_at, 0);

   if(warp == 0) {
      bool ok = true;
      int s = 0;
      uint32_t phase = 1;
      tc::wait_for_previous();
      for(long long t = first; t < tiles && ok; t += step) {
         int m0, n0;
         pair_tile<P>(g, t, &m0, &n0);
         const int a_row = m0 + (int)rank * 128, b_row = n0 + (int)rank * (P::BN / 2);
         const int a_tile = m0 / TILE_ROWS + (int)rank, b_tile = n0 / TILE_ROWS;
         for(int k = 0; k < g.chunks; ++k) {
            if(!mbar_wait(empty + s, phase, g.status)) {
               ok = false;
               break;
            }
            if(tc::elect()) {
               uint8_t* at = body + s * P::STAGE;
               const uint32_t bar = tc::peer_smem(full + s, 0);
               if(rank == 0) mbar_expect_tx(full + s, 2 * P::STAGE);
               tc::tma_load_2d_pair(at, &ta, k * 128, a_row, bar);
               tc::tma_load_2d_pair(at + P::A_BYTES, &tb, k * 128, b_row, bar);
               at += P::A_BYTES + P::B_BYTES;
               tc::tma_load_2d_pair(at, &tsa, k * 256, a_tile, bar);
               tc::tma_load_2d_pair(at + P::SF_BYTES, &tsb, k * 256, b_tile, bar);
               tc::tma_load_2d_pair(at + 2 * P::SF_BYTES, &tsb, k * 256, b_tile + 1, bar);
            }
            __syncwarp();
            if(++s == P::STAGES) {
               s = 0;
               phase ^= 1;
            }
         }
      }
      if(!ok) {   // a wait gave up: time for the copies under way, whose barrier may be the other CTA's, to land
         const uint64_t t0 = globaltimer_ns();
         while(globaltimer_ns() - t0 < 2000000ull) {}
      }
   } else if(warp == 1 && rank == 0) {
      bool ok = true;
      int s = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 1;
      const uint64_t rows0 = tc::rows_desc(smem_u32(body)), scales0 = tc::scales_desc(smem_u32(body) + P::A_BYTES + P::B_BYTES);
      for(long long t = first; t < tiles && ok; t += step) {
         int m0, n0;
         pair_tile<P>(g, t, &m0, &n0);
         if(!mbar_wait<true>(taken + acc, acc_phase, g.status)) break;
         tc::fence_after_sync();
         const uint32_t d = tmem + acc * P::BN, b_col = (uint32_t)(n0 % TILE_ROWS / 32);
         for(int k = 0; k < g.chunks; ++k) {
            if(!mbar_wait<true>(full + s, phase, g.status)) {
               ok = false;
               break;
            }
            tc::fence_after_sync();
            const uint64_t rows = rows0 + (uint32_t)(s * (P::STAGE >> 4)), sf = scales0 + (uint32_t)(s * (P::STAGE >> 4));
            const uint32_t col = tmem + P::SF_AT + s * P::SF_COLS;
            if(tc::elect()) {
#pragma unroll
               for(int h = 0; h < 2; ++h) {
                  tc::copy_scales_pair(col + h * 4, sf + h * (TILE_BYTES >> 4));
                  tc::copy_scales_pair(col + 8 + h * 8, sf + ((P::SF_BYTES + h * TILE_BYTES) >> 4));
                  tc::copy_scales_pair(col + 12 + h * 8, sf + ((2 * P::SF_BYTES + h * TILE_BYTES) >> 4));
               }
#pragma unroll
               for(int q = 0; q < 4; ++q)
                  tc::mma_mxf4_pair(d, rows + q * 2, rows + ((P::A_BYTES + q * 32) >> 4), tc::mxf4_idesc(256, P::BN, (q & 1) * 2),
                                    col + (q >> 1) * 4, col + 8 + (q >> 1) * 8 + b_col, k > 0 || q > 0);
               tc::commit_pair(empty + s);
               if(k + 1 == g.chunks) tc::commit_pair(ready + acc);
            }
            __syncwarp();
            if(++s == P::STAGES) {
               s = 0;
               phase ^= 1;
            }
         }
         if(++acc == P::ACC) {
            acc = 0;
            acc_phase ^= 1;
         }
      }
   } else if(warp >= 2) {
      const int quarter = warp & 3, half = (warp - 2) / 4;   // the lanes that this warp may read; its columns
      const int width = min(P::COLS, P::BN - half * P::COLS);
      long long done = 0;
      T* out = static_cast<T*>(g.out);
      for(long long t = first; t < tiles; t += step, ++done) {
         int m0, n0;
         pair_tile<P>(g, t, &m0, &n0);
         const int acc = (int)(done % P::ACC);
         if(!mbar_wait<true>(ready + acc, (uint32_t)(done / P::ACC & 1), g.status)) break;
         tc::fence_after_sync();
         const uint32_t mine = tmem + ((uint32_t)quarter << 21) + acc * P::BN + half * P::COLS;
         float v[P::COLS];
         __syncwarp();   // rows beyond the last have skipped their stores
#pragma unroll
         for(int j = 0; j < P::COLS; j += 16)
            if(j < width) tc::tmem_load16(mine + j, v + j);
         tc::tmem_load_wait();
         tc::fence_before_sync();
         __syncwarp();
         if(lane == 0) tc::arrive_peer(tc::peer_smem(taken + acc, 0));
         const long long row = m0 + (long long)rank * 128 + quarter * 32 + lane, col = n0 + half * P::COLS;
         const int left = (int)max(0ll, min((long long)width, g.n - col));   // columns that exist
         if(!SWAP && g.bias)
#pragma unroll
            for(int j = 0; j < P::COLS; ++j)
               if(j < left) v[j] += __ldg(g.bias + col + j);
         if constexpr(SWAP) {
            const float bias = g.bias && row < g.m ? g.bias[row] : 0.0f;
#pragma unroll
            for(int j = 0; j < P::COLS; ++j)
               if(j < left && row < g.m) out[(col + j) * g.out_stride + row] = from_f<T>(v[j] + bias);
         } else {
            constexpr int W = 128 / (int)sizeof(T);   // columns of a tile
            uint8_t* mine_out = leaving + (warp - 2) * P::OUT;
            const int row0 = m0 + (int)rank * 128 + quarter * 32;
#pragma unroll
            for(int j = 0; j < P::COLS; j += W) {
               if(j >= left || row0 >= g.m) break;
               if(lane == 0) tc::tma_stores_read();
               __syncwarp();
               // a lane's row of 128 bytes, its 16-byte chunks permuted as the tensor copy will undo
#pragma unroll
               for(int c = 0; c < 8; ++c) {
                  constexpr int PER = W / 8;
                  const float* x = v + j + c * PER;
                  uint4 q;
                  if constexpr(sizeof(T) == 4) q = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                  else q = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
                  *reinterpret_cast<uint4*>(mine_out + lane * 128 + ((c ^ (lane & 7)) << 4)) = q;
               }
               fence_proxy_async_smem();
               __syncwarp();
               if(lane == 0) tc::tma_store_2d(&tout, (int)col + j, row0, mine_out);
            }
         }
      }
   }
   if(!SWAP && warp >= 2 && lane == 0) tc::tma_stores_done();
   __syncwarp();
   tc::fence_before_sync();
   tc::cluster_sync();       // both have read their sums; nothing is under way in either's memory
   if(warp == 1) tc::tmem_free_pair<P::TMEM>(tmem);
}

// 4-bit codes as tiles of box_rows x 128 bytes, 128-byte swizzle; rows beyond the last read as zeros
fufft_status codes_tmap(CUtensorMap* tm, const uint8_t* codes, long long rows, long long pitch, int box_rows)
{
   const cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
   const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
   return encode_tmap(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// the scale tiles of 128 rows x 256 columns, 1024 bytes each as 256 words; tiles beyond the last row read as zeros
fufft_status scales_tmap(CUtensorMap* tm, const uint8_t* scales, long long rows, int chunks)
{
   const cuuint64_t dims[2] = {(cuuint64_t)chunks * 256, (cuuint64_t)ceil_div(rows, TILE_ROWS)}, strides[1] = {(cuuint64_t)chunks * 1024};
   const cuuint32_t box[2] = {256, 1};
   return encode_tmap(tm, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, scales, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

struct Operands {
   const uint8_t *a, *a_scale, *b, *b_scale;
   const float* bias;
   void* out;
   long long m, n, k, out_stride;
   bool follows;             // the kernel before on the stream wrote a (and neither b nor anything else that is read)
};

template<class T, int BN, class A = Packed>
fufft_status launch_split(const Operands& o, int split, const DeviceCtx& ctx, cudaStream_t st, const RawArgs& x = {})
{
   using C = Split<BN>;
   const long long pitch = mx4_pitch(o.k);
   CUtensorMap tp{}, tq{};
   fufft_status s;
   if(o.k) {
      if((s = codes_tmap(&tp, o.b, o.n, pitch, 128)) != FUFFT_OK) return s;
      if(std::is_same_v<A, Packed> && (s = codes_tmap(&tq, o.a, o.m, pitch, BN)) != FUFFT_OK) return s;
   }
   auto kern = matmul_split_kernel<T, BN, A>;
   static std::atomic<uint64_t> configured{0};
   if((s = allow_smem(kern, C::SMEM, configured)) != FUFFT_OK) return s;
   MatmulArgs g{o.b_scale, o.a_scale, o.bias, o.out, ctx.status, o.n, o.m, o.out_stride, (int)(pitch / 128),
                (int)ceil_div(o.n, 128), split};
   cudaLaunchConfig_t cfg = {};
   cfg.gridDim = dim3((unsigned)(g.tiles_p * ceil_div(o.m, BN) * split));
   cfg.blockDim = dim3(128);
   cfg.dynamicSmemBytes = C::SMEM;
   cfg.stream = st;
   cudaLaunchAttribute at[2];
   at[0].id = cudaLaunchAttributeClusterDimension;
   at[0].val.clusterDim.x = (unsigned)split;
   at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
   at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
   at[1].val.programmaticStreamSerializationAllowed = 1;
   cfg.attrs = at;
   cfg.numAttrs = o.follows ? 2 : 1;
   if((s = check(cudaLaunchKernelEx(&cfg, kern, tp, tq, g, x))) != FUFFT_OK) return s;
   count_launch();
   return check(cudaGetLastError());
}

// parts of the summed axis: until two CTAs per SM are there, of two chunks at least
int split_for(long long tiles, int chunks, int sms)
{
   int split = 1;
   while(split < MAX_SPLIT && tiles * split * 2 <= 2ll * sms && chunks >= 4 * split) split *= 2;
   return split;
}

// the result as tiles of 32 rows x 128 bytes
template<class T> fufft_status result_tmap(CUtensorMap* tm, const Operands& o)
{
   const cuuint64_t dims[2] = {(cuuint64_t)o.n, (cuuint64_t)o.m}, strides[1] = {(cuuint64_t)(o.out_stride * sizeof(T))};
   const cuuint32_t box[2] = {(cuuint32_t)(128 / sizeof(T)), 32};
   const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
   return encode_tmap(tm, type, 2, o.out, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template<class T, class P, bool SWAP>
fufft_status launch_pair(const Operands& o, const DeviceCtx& ctx, cudaStream_t st)
{
   const long long pitch = mx4_pitch(o.k);
   CUtensorMap ta, tb, tsa, tsb, tout{};
   fufft_status s;
   PairArgs g{o.bias, o.out, ctx.status, o.m, o.n, o.out_stride, (int)(pitch / 128), (int)ceil_div(o.m, 256),
              (int)ceil_div(o.n, P::BN)};
   if((s = codes_tmap(&ta, o.a, o.m, pitch, 128)) != FUFFT_OK) return s;
   if((s = codes_tmap(&tb, o.b, o.n, pitch, P::BN / 2)) != FUFFT_OK) return s;
   if((s = scales_tmap(&tsa, o.a_scale, o.m, g.chunks)) != FUFFT_OK) return s;
   if((s = scales_tmap(&tsb, o.b_scale, o.n, g.chunks)) != FUFFT_OK) return s;
   if(!SWAP && (s = result_tmap<T>(&tout, o)) != FUFFT_OK) return s;
   auto kern = matmul_pair_kernel<T, P, SWAP>;
   static std::atomic<uint64_t> configured{0};
   if((s = allow_smem(kern, P::SMEM, configured)) != FUFFT_OK) return s;
   cudaLaunchConfig_t cfg = {};
   cfg.gridDim = dim3(2 * (unsigned)std::min<long long>((long long)g.tiles_m * g.tiles_n, sm_count(ctx.device) / 2));
   cfg.blockDim = dim3(P::THREADS);
   cfg.dynamicSmemBytes = P::SMEM;
   cfg.stream = st;
   cudaLaunchAttribute at[2];
   at[0].id = cudaLaunchAttributeClusterDimension;
   at[0].val.clusterDim.x = 2;
   at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
   at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
   at[1].val.programmaticStreamSerializationAllowed = 1;
   cfg.attrs = at;
   cfg.numAttrs = o.follows ? 2 : 1;
   if((s = check(cudaLaunchKernelEx(&cfg, kern, ta, tb, tsa, tsb, tout, g))) != FUFFT_OK) return s;
   count_launch();
   return check(cudaGetLastError());
}
template<class T, class P> fufft_status launch_pair(const Operands& o, const DeviceCtx& ctx, cudaStream_t st)
{
   if(aligned(o.out, 16) && o.out_stride * (long long)sizeof(T) % 16 == 0) return launch_pair<T, P, false>(o, ctx, st);
   const Operands swapped{o.b, o.b_scale, o.a, o.a_scale, o.bias, o.out, o.n, o.m, o.k, o.out_stride, o.follows};
   return launch_pair<T, P, true>(swapped, ctx, st);
}

template<class T> fufft_status matmul(const Operands& o, cudaStream_t st)
{
   DeviceCtx ctx;
   fufft_status s = device_ctx(&ctx);
   if(s != FUFFT_OK) return s;
   const int chunks = (int)(mx4_pitch(o.k) / 128), sms = sm_count(ctx.device);
   const long long tiles_p = ceil_div(o.n, 128);
   if(o.m <= 16) return launch_split<T, 16>(o, split_for(tiles_p, chunks, sms), ctx, st);
   if(o.m <= 32) return launch_split<T, 32>(o, split_for(tiles_p, chunks, sms), ctx, st);
   if(o.m <= 64) return launch_split<T, 64>(o, split_for(tiles_p, chunks, sms), ctx, st);
   // Pairs, unless their tiles leave most of the card idle and a long summed
   // axis pays for joining its parts, or where a small result's rows start
   // anywhere (us, split / pair: 512 x 512 x 8192 9.7 / 13.1, 128 x 1024 x 1024
   // 9.0 / 7.2, 333 x 1537 x 1111 9.4 / 12.0, 333 x 1536 x 1111 9.4 / 6.5).
   const bool aligned_rows = aligned(o.out, 16) && o.out_stride * (long long)sizeof(T) % 16 == 0;
   const long long pairs = sms / 2, narrow = ceil_div(o.m, 256) * ceil_div(o.n, 192), wide = ceil_div(o.m, 256) * ceil_div(o.n, 256);
   if((narrow * MAX_SPLIT <= pairs && chunks >= 8) || (narrow * 2 <= pairs && !aligned_rows))
      return launch_split<T, 128>(o, split_for(tiles_p * ceil_div(o.m, 128), chunks, sms), ctx, st);
   if(chunks == 0) return launch_split<T, 128>(o, 1, ctx, st);
   // 256 columns in one accumulator or 192 in two of them, whichever covers the
   // result in fewer columns' time (us, 256 / 192: 8192^3 189 / 201, 4096^3
   // 28.1 / 26.7, 512 x 4096 x 4096 10.3 / 9.0).  The drain after a tile's
   // last stage, which a single accumulator cannot hide, is not in the rule.
   return ceil_div(wide, pairs) * 256 < ceil_div(narrow, pairs) * 192 ? launch_pair<T, Pair<256, 1>>(o, ctx, st)
                                                                     : launch_pair<T, Pair<192, 2>>(o, ctx, st);
}

// rows of x quantised on the way
template<class T>
fufft_status matmul_raw(const Operands& o, fufft_dtype x_dtype, const RawArgs& x, cudaStream_t st)
{
   DeviceCtx ctx;
   fufft_status s = device_ctx(&ctx);
   if(s != FUFFT_OK) return s;
   const int split = split_for(ceil_div(o.n, 128), (int)(mx4_pitch(o.k) / 128), sm_count(ctx.device));
   switch(x_dtype) {
   case FUFFT_F32: return launch_split<T, 16, Raw<float>>(o, split, ctx, st, x);
   case FUFFT_F16: return launch_split<T, 16, Raw<__half>>(o, split, ctx, st, x);
   default: return launch_split<T, 16, Raw<__nv_bfloat16>>(o, split, ctx, st, x);
   }
}

fufft_status matmul(const Operands& o, fufft_dtype dtype, fufft_stream_t stream)
{
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return matmul<float>(o, st);
   case FUFFT_F16: return matmul<__half>(o, st);
   default: return matmul<__nv_bfloat16>(o, st);
   }
}

}  // namespace mx
}  // namespace fufft

namespace {
fufft_status check_matmul(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales,
                          const float* bias, const void* out, fufft_dtype dtype, int64_t m, int64_t n, int64_t k,
                          int64_t out_stride)
{
   constexpr int64_t MAX = 1ll << 30;
   if(dtype < FUFFT_F32 || dtype > FUFFT_BF16) return FUFFT_ERR_INVALID_ARG;
   if(m < 0 || n < 0 || k < 0 || m > MAX || n > MAX || k > MAX) return FUFFT_ERR_INVALID_SIZE;
   if(m == 0 || n == 0) return FUFFT_OK;
   if(mx::ceil_div(m, 16) > (1ll << 27) / mx::ceil_div(n, 128)) return FUFFT_ERR_INVALID_SIZE;
   if(!out || (k && (!a_codes || !a_scales || !b_codes || !b_scales)) || (m > 1 && out_stride < n)) return FUFFT_ERR_INVALID_ARG;
   if(!aligned(a_codes, 16) || !aligned(a_scales, 16) || !aligned(b_codes, 16) || !aligned(b_scales, 16) ||
      !aligned(bias, 4) || !aligned(out, dtype == FUFFT_F32 ? 4 : 2))
      return FUFFT_ERR_MISALIGNED;
   return FUFFT_OK;
}
}  // namespace

extern "C" {

fufft_status fufft_mx4_matmul(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes,
                              const uint8_t* b_scales, const float* bias, void* out, fufft_dtype dtype, int64_t m,
                              int64_t n, int64_t k, int64_t out_stride, fufft_stream_t stream)
{
   fufft_status s = check_matmul(a_codes, a_scales, b_codes, b_scales, bias, out, dtype, m, n, k, out_stride);
   if(s != FUFFT_OK || m == 0 || n == 0) return s;
   return mx::matmul({a_codes, a_scales, b_codes, b_scales, bias, out, m, n, k, out_stride, false}, dtype, stream);
}

fufft_status fufft_mx4_linear(const void* x, fufft_dtype x_dtype, int64_t m, int64_t k, int64_t x_stride,
                              uint8_t* x_codes, uint8_t* x_scales, const uint8_t* w_codes, const uint8_t* w_scales,
                              int64_t n, const float* bias, void* out, fufft_dtype dtype, int64_t out_stride,
                              fufft_stream_t stream)
{
   // everything is checked before the first launch: a refused call leaves x_codes alone
   const bool direct = m <= FUFFT_MX4_DIRECT_ROWS;
   fufft_status s = check_matmul(direct ? w_codes : x_codes, direct ? w_scales : x_scales, w_codes, w_scales, bias, out, dtype, m, n, k, out_stride);
   if(s != FUFFT_OK || m == 0 || n == 0) return s;
   if(!direct || k == 0) {
      if((s = fufft_mx4_quantize(x, x_dtype, m, k, x_stride, x_codes, x_scales, nullptr, nullptr, stream)) != FUFFT_OK) return s;
      return mx::matmul({x_codes, x_scales, w_codes, w_scales, bias, out, m, n, k, out_stride, k > 0}, dtype, stream);
   }
   if(x_dtype < FUFFT_F32 || x_dtype > FUFFT_BF16 || !x || (m > 1 && x_stride < k)) return FUFFT_ERR_INVALID_ARG;
   const long long size = x_dtype == FUFFT_F32 ? 4 : 2;
   if(!aligned(x, (unsigned)size)) return FUFFT_ERR_MISALIGNED;
   const mx::Operands o{nullptr, nullptr, w_codes, w_scales, bias, out, m, n, k, out_stride, false};
   const mx::RawArgs rows{x, x_stride, k, aligned(x, 32) && (m == 1 || x_stride * size % 32 == 0)};
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return mx::matmul_raw<float>(o, x_dtype, rows, st);
   case FUFFT_F16: return mx::matmul_raw<__half>(o, x_dtype, rows, st);
   default: return mx::matmul_raw<__nv_bfloat16>(o, x_dtype, rows, st);
   }
}

}  // extern "C"
