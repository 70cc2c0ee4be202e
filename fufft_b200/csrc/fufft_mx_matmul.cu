// fufft_mx_matmul.cu -- product of two 4-bit microscaled matrices,
// out[m][n] = sum_k a[m][k] b[n][k] + bias[n], on the tensor cores
// (tcgen05 kind::mxf4: E2M1 products under E8M0 scales, fp32 sums in tensor
// memory).
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

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
// ---------------------------------------------------------------------------
template<int BN> struct Split {
   static constexpr int SF_Q = (BN + 127) / 128;                     // scale tiles of the columns
   static constexpr int P_BYTES = 128 * 128, Q_BYTES = BN * 128, SF_BYTES = 1024;
   static constexpr int STAGE = P_BYTES + Q_BYTES + SF_BYTES * (1 + SF_Q);
   static constexpr int STAGES = BN <= 16 ? 5 : BN <= 64 ? 4 : 3;
   static constexpr int SF_COLS = 8 + 8 * SF_Q;                      // tensor-memory columns of a stage's scales
   static constexpr int NEED = BN + STAGES * SF_COLS;
   static constexpr int TMEM = NEED <= 128 ? 128 : NEED <= 256 ? 256 : 512;
   static constexpr int PITCH = 129;                                 // of a partial column, in floats
   static constexpr int JOIN = BN * PITCH * 4;
   static constexpr int BODY = STAGES * STAGE > JOIN ? STAGES * STAGE : JOIN;
   static constexpr int SMEM = BODY + 1024 + 128;
   static_assert(STAGE % 1024 == 0, "the 128-byte swizzle repeats every 1024 bytes");
};

template<class T, int BN>
__global__ void __launch_bounds__(128) matmul_split_kernel(const __grid_constant__ CUtensorMap tp,
                                                           const __grid_constant__ CUtensorMap tq, MatmulArgs g)
{
   using C = Split<BN>;
   extern __shared__ uint8_t raw[];
   uint8_t* body = reinterpret_cast<uint8_t*>(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
   uint64_t* full = reinterpret_cast<uint64_t*>(body + C::BODY);
   uint64_t* empty = full + C::STAGES;
   uint64_t* done = empty + C::STAGES;
   uint32_t* tmem_at = reinterpret_cast<uint32_t*>(done + 1);

   const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
   const int rank = g.split > 1 ? (int)tc::cluster_rank() : 0;
   const long long tile = blockIdx.x / g.split;
   const int p0 = (int)(tile % g.tiles_p) * 128;
   const long long q0 = tile / g.tiles_p * BN;
   const int per = (g.chunks + g.split - 1) / g.split;
   const int k0 = min(rank * per, g.chunks), k1 = min(k0 + per, g.chunks), n = k1 - k0;

   if(threadIdx.x == 0) {
      for(int s = 0; s < C::STAGES; ++s) {
         mbar_init(full + s, 1);
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
   const uint32_t tmem = *tmem_at;

   if(threadIdx.x == 0) {
      // copies: both operands' 256 columns and their scales, one stage each
      const long long q_tile_last = ceil_div(g.q_rows, TILE_ROWS) - 1;
      int issued = 0;
      bool ok = true;
      for(int i = 0; i < n && ok; ++i) {
         const int s = i % C::STAGES;
         if(!mbar_wait(empty + s, (i / C::STAGES & 1) ^ 1, g.status)) {
            ok = false;
            break;
         }
         uint8_t* at = body + s * C::STAGE;
         mbar_expect_tx(full + s, C::STAGE);
         tma_load_2d(at, &tp, (k0 + i) * 128, p0, full + s);
         tma_load_2d(at + C::P_BYTES, &tq, (k0 + i) * 128, (int)q0, full + s);
         at += C::P_BYTES + C::Q_BYTES;
         bulk_g2s(at, g.p_scale + ((long long)(p0 / TILE_ROWS) * g.chunks + k0 + i) * C::SF_BYTES, C::SF_BYTES, full + s);
         for(int h = 0; h < C::SF_Q; ++h) {
            const long long row_tile = min(q0 / TILE_ROWS + h, q_tile_last);
            bulk_g2s(at + (1 + h) * C::SF_BYTES, g.q_scale + (row_tile * g.chunks + k0 + i) * C::SF_BYTES, C::SF_BYTES, full + s);
         }
         issued = i + 1;
      }
      // after a wait that gave up: no copy may still be landing when the CTA ends
      if(!ok)
         for(int i = max(0, issued - C::STAGES); i < issued; ++i) mbar_wait(full + i % C::STAGES, i / C::STAGES & 1, g.status);
   } else if(threadIdx.x == 32 && n > 0) {
      const uint32_t sf_at = tmem + BN;
      const uint32_t q_col = (uint32_t)(q0 % TILE_ROWS / 32);       // this tile's first scale column of its row tile
      for(int i = 0; i < n; ++i) {
         const int s = i % C::STAGES;
         if(!mbar_wait(full + s, i / C::STAGES & 1, g.status)) break;
         tc::fence_after_sync();
         const uint32_t at = smem_u32(body + s * C::STAGE), sf = at + C::P_BYTES + C::Q_BYTES;
         const uint32_t col = sf_at + s * C::SF_COLS;
#pragma unroll
         for(int t = 0; t < 2; ++t) {
            tc::copy_scales(col + t * 4, tc::scales_desc(sf + t * TILE_BYTES));
#pragma unroll
            for(int h = 0; h < C::SF_Q; ++h)
               tc::copy_scales(col + 8 + (t * C::SF_Q + h) * 4, tc::scales_desc(sf + (1 + h) * C::SF_BYTES + t * TILE_BYTES));
         }
#pragma unroll
         for(int k = 0; k < 4; ++k)
            tc::mma_mxf4(tmem, tc::rows_desc(at + k * 32), tc::rows_desc(at + C::P_BYTES + k * 32),
                         tc::mxf4_idesc(128, BN, (k & 1) * 2), col + (k >> 1) * 4, col + 8 + (k >> 1) * C::SF_Q * 4 + q_col,
                         i > 0 || k > 0);
         tc::commit(empty + s);
      }
      tc::commit(done);
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
      const int rows = (int)min((long long)BN, g.q_rows - q0);
      const long long row = p0 + threadIdx.x;
      if(row < g.p_rows) {
         const float bias = g.bias ? g.bias[row] : 0.0f;
         for(int j = rank; j < rows; j += g.split) {
            float sum = 0.0f;
            for(int r = 0; r < g.split; ++r) sum += tc::load_peer(tc::peer_smem(part + j * C::PITCH + threadIdx.x, r));
            out[(q0 + j) * g.out_stride + row] = from_f<T>(sum + bias);
         }
      }
      tc::cluster_sync();   // nobody leaves while its sums are being read
   }
   tc::fence_before_sync();
   __syncthreads();
   if(warp == 2) tc::tmem_free<C::TMEM>(tmem);
}

// 128-byte rows of 4-bit codes, `rows` of them `pitch` bytes apart
fufft_status codes_tmap(CUtensorMap* tm, const uint8_t* codes, long long rows, long long pitch, int box_rows)
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
   cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows};
   cuuint64_t strides[1] = {(cuuint64_t)pitch};
   cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
   cuuint32_t estr[2] = {1, 1};
   const CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
   return r == CUDA_SUCCESS ? FUFFT_OK : FUFFT_ERR_UNSUPPORTED;
}

struct Operands {
   const uint8_t *a, *a_scale, *b, *b_scale;
   const float* bias;
   void* out;
   long long m, n, k, out_stride;
};

template<class T, int BN>
fufft_status launch_split(const Operands& o, int split, const DeviceCtx& ctx, cudaStream_t st)
{
   using C = Split<BN>;
   const long long pitch = mx4_pitch(o.k);
   CUtensorMap tp{}, tq{};
   fufft_status s;
   if(o.k) {
      if((s = codes_tmap(&tp, o.b, o.n, pitch, 128)) != FUFFT_OK) return s;
      if((s = codes_tmap(&tq, o.a, o.m, pitch, BN)) != FUFFT_OK) return s;
   }
   auto kern = matmul_split_kernel<T, BN>;
   static std::atomic<uint64_t> configured{0};
   if((s = allow_smem(kern, C::SMEM, configured)) != FUFFT_OK) return s;
   MatmulArgs g{o.b_scale, o.a_scale, o.bias, o.out, ctx.status, o.n, o.m, o.out_stride, (int)(pitch / 128),
                (int)ceil_div(o.n, 128), split};
   cudaLaunchConfig_t cfg = {};
   cfg.gridDim = dim3((unsigned)(g.tiles_p * ceil_div(o.m, BN) * split));
   cfg.blockDim = dim3(128);
   cfg.dynamicSmemBytes = C::SMEM;
   cfg.stream = st;
   cudaLaunchAttribute at[1];
   at[0].id = cudaLaunchAttributeClusterDimension;
   at[0].val.clusterDim.x = (unsigned)split;
   at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
   cfg.attrs = at;
   cfg.numAttrs = 1;
   if((s = check(cudaLaunchKernelEx(&cfg, kern, tp, tq, g))) != FUFFT_OK) return s;
   count_launch();
   return check(cudaGetLastError());
}

// parts of the summed axis: until two CTAs per SM are there, of two chunks at least
int split_for(long long tiles, int chunks, int sms)
{
   int split = 1;
   while(split < 8 && tiles * split * 2 <= 2ll * sms && chunks >= 4 * split) split *= 2;
   return split;
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
   return launch_split<T, 128>(o, split_for(tiles_p * ceil_div(o.m, 128), chunks, sms), ctx, st);
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
   const mx::Operands o{a_codes, a_scales, b_codes, b_scales, bias, out, m, n, k, out_stride};
   cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
   switch(dtype) {
   case FUFFT_F32: return mx::matmul<float>(o, st);
   case FUFFT_F16: return mx::matmul<__half>(o, st);
   default: return mx::matmul<__nv_bfloat16>(o, st);
   }
}

fufft_status fufft_mx4_linear(const void* x, fufft_dtype x_dtype, int64_t m, int64_t k, int64_t x_stride,
                              uint8_t* x_codes, uint8_t* x_scales, const uint8_t* w_codes, const uint8_t* w_scales,
                              int64_t n, const float* bias, void* out, fufft_dtype dtype, int64_t out_stride,
                              fufft_stream_t stream)
{
   // everything is checked before the first launch: a refused call leaves x_codes alone
   fufft_status s = check_matmul(x_codes, x_scales, w_codes, w_scales, bias, out, dtype, m, n, k, out_stride);
   if(s != FUFFT_OK || m == 0 || n == 0) return s;
   if((s = fufft_mx4_quantize(x, x_dtype, m, k, x_stride, x_codes, x_scales, nullptr, nullptr, stream)) != FUFFT_OK) return s;
   return fufft_mx4_matmul(x_codes, x_scales, w_codes, w_scales, bias, out, dtype, m, n, k, out_stride, stream);
}

}  // extern "C"
