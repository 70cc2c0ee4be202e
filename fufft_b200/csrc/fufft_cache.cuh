// fufft_cache.cuh -- a paged sequence cache in a microscaled format, as the
// kernels see it.
#pragma once
#include "fufft_internal.cuh"
#include "fufft_mx.cuh"

namespace fufft {
namespace cache {

// tokens x channels / 8 threads of 256 stay below 2^31 blocks with these
constexpr int MAX_CHANNELS = 1 << 16;
constexpr int MAX_BATCH = 1 << 20;
constexpr long long MAX_TOKENS = 1ll << 25;

struct Pages {
   uint8_t* codes;
   uint8_t* scales;
   const int32_t* table;
   long long table_stride;
   int page_size, pages, max_pages, batch;

   explicit Pages(const fufft_cache* c)
      : codes(c->codes), scales(c->scales), table(c->page_table), table_stride(c->table_stride), page_size(c->page_size),
        pages(c->pages), max_pages(c->max_pages), batch(c->batch)
   {
   }

   // row of the flattened pages that holds position pos of sequence b, or -1
   // where the sequence has no page there
   __device__ __forceinline__ long long slot(int b, long long pos) const
   {
      if(pos < 0) return -1;
      const long long k = pos / page_size;
      if(k >= max_pages) return -1;
      const int page = table[b * table_stride + k];
      return page < 0 || page >= pages ? -1 : (long long)page * page_size + (pos - k * page_size);
   }
};

fufft_status check_cache(const fufft_cache* c);

}  // namespace cache
}  // namespace fufft
