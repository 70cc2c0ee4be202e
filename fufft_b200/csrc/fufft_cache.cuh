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
   // where the sequence has no page there.  Lengths are 32 bits, so positions
   // beyond them hold nothing; pages * page_size stays below 2^31.
   __device__ __forceinline__ int slot(int b, long long pos) const
   {
      if(pos < 0 || pos > 0x7fffffffll) return -1;
      const unsigned k = (unsigned)pos / (unsigned)page_size;
      if(k >= (unsigned)max_pages) return -1;
      return row(__ldg(table + b * table_stride + k), (int)((unsigned)pos - k * (unsigned)page_size));
   }
   // position `in` of a page of the table, or -1 where there is no such page
   __device__ __forceinline__ int row(int page, int in) const { return page < 0 || page >= pages ? -1 : page * page_size + in; }
};

fufft_status check_cache(const fufft_cache* c);

}  // namespace cache
}  // namespace fufft
