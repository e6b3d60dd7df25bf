// Copies of whole pages inside one pool, K and V of every kv head: forking a sequence, moving pages together.
//
// The page lists come from host memory, where a pool's bookkeeping is: they are checked there (a list that names a page twice, or
// one as source and destination, has no one result) and travel as kernel arguments, so a call needs no
// device copy of its own and no wait, whatever stream it runs on.  Bound by memory: a page's bytes read and written once.
#include <cstring>
#include <new>

#include "common.h"
#include "runtime.h"

namespace lkv {
namespace {

constexpr int kRuns = 320;         // runs of consecutive pages a launch takes (with the rest below 4 KiB of arguments)
constexpr int kPagesPerItem = 4;   // pages a workgroup copies

struct CopyRuns {
  int32_t n;
  int32_t src[kRuns], dst[kRuns], end[kRuns];  // end: pages of the runs up to and with this one
};

struct CopyParams {
  uint8_t* pool[2];
  uint8_t* scales[2];  // or null: one byte a (page, head)
  int64_t page, head, scale_head;
  int32_t page_bytes, total;
};

// kChunks: 16-byte pieces a thread copies of one page (page_bytes / 4096).  Workgroup x: pages [4 x, 4 x + 4) of the runs, of
// one head's K or V; all of its loads come before its stores.  The run of its first page is searched once.  Sources are read
// with the non-temporal hint (2048 pages of 8 heads in 32 runs: 146 us with a search a page and without the hint, so 97;
// hipMemcpy of the same bytes 90).
template <int kChunks>
__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyParams p, const CopyRuns r) {
  const int h = blockIdx.y, kv = blockIdx.z;
  uint8_t* pool = p.pool[kv] + h * p.head;
  const int i0 = blockIdx.x * kPagesPerItem;
  int run = 0;
  for (int hi = r.n - 1; run < hi;) {  // the first run whose end is past i0
    const int mid = (run + hi) >> 1;
    if (r.end[mid] > i0)
      hi = mid;
    else
      run = mid + 1;
  }
  int end = r.end[run], start = run > 0 ? r.end[run - 1] : 0;
  int src = r.src[run] - start, dst = r.dst[run] - start;
  int from[kPagesPerItem], to[kPagesPerItem];
  uint4 x[kPagesPerItem][kChunks];
#pragma unroll
  for (int q = 0; q < kPagesPerItem; ++q) {
    const int i = min(i0 + q, p.total - 1);
    if (i >= end) {  // (runs are not empty: the next one holds it)
      start = end;
      ++run;
      end = r.end[run];
      src = r.src[run] - start;
      dst = r.dst[run] - start;
    }
    from[q] = src + i;
    to[q] = dst + i;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) x[q][c] = load_nt(pool + from[q] * p.page + (c * 256 + threadIdx.x) * 16);
  }
#pragma unroll
  for (int q = 0; q < kPagesPerItem; ++q) {
    if (i0 + q >= p.total) break;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) *reinterpret_cast<uint4*>(pool + to[q] * p.page + (c * 256 + threadIdx.x) * 16) = x[q][c];
    if (p.scales[kv] != nullptr && threadIdx.x == 0) {
      uint8_t* s = p.scales[kv] + h * p.scale_head;
      s[to[q]] = s[from[q]];
    }
  }
}

// Whether the lists have one result: every page in the pool, no destination twice, none that is a source too.  Few pairs of a
// large pool are compared with each other; else a byte a page says what it is (1 a source, 2 a destination), which for one pair of
// 70000 pages takes 2.1 us and for one of 600000 15, where
// two pairs compared take less than 0.1 and 32 take 1.4.
int32_t check_pairs(const lkv_copy_pages_args* a) {
  const int32_t n = a->count;
  for (int32_t i = 0; i < n; ++i)
    if (a->src[i] < 0 || a->src[i] >= a->num_pages || a->dst[i] < 0 || a->dst[i] >= a->num_pages)
      return fail(LKV_ERR_INVALID_ARGUMENT, "pair %d (%d to %d) is outside the pool's %d pages", i, a->src[i], a->dst[i], a->num_pages);
  const auto twice = [](int32_t page) { return fail(LKV_ERR_INVALID_ARGUMENT, "page %d is a destination twice", page); };
  const auto both = [](int32_t page) { return fail(LKV_ERR_INVALID_ARGUMENT, "page %d is a source and a destination", page); };
  if (static_cast<int64_t>(n) * n <= a->num_pages / 64) {
    for (int32_t i = 0; i < n; ++i)
      for (int32_t j = 0; j < n; ++j) {
        if (a->src[j] == a->dst[i]) return both(a->dst[i]);
        if (j < i && a->dst[j] == a->dst[i]) return twice(a->dst[i]);
      }
    return LKV_OK;
  }
  uint8_t* seen = new (std::nothrow) uint8_t[a->num_pages];
  if (seen == nullptr) return fail(LKV_ERR_INVALID_ARGUMENT, "no memory to check %d pages", a->num_pages);
  std::memset(seen, 0, a->num_pages);
  int32_t status = LKV_OK;
  for (int32_t i = 0; i < n; ++i) seen[a->src[i]] = 1;
  for (int32_t i = 0; i < n && status == LKV_OK; ++i) {
    uint8_t& page = seen[a->dst[i]];
    if (page != 0) status = page & 2 ? twice(a->dst[i]) : both(a->dst[i]);
    page |= 2;
  }
  delete[] seen;
  return status;
}

}  // namespace
}  // namespace lkv

extern "C" int32_t lkv_copy_pages(const lkv_copy_pages_args* a, lkv_stream_t stream) {
  using namespace lkv;
  LKV_REQUIRE(a != nullptr, "null args");
  LKV_REQUIRE(a->struct_size == static_cast<int32_t>(sizeof(lkv_copy_pages_args)),
              "lkv_copy_pages_args size mismatch (caller %d, library %d)", a->struct_size,
              static_cast<int32_t>(sizeof(lkv_copy_pages_args)));
  LKV_REQUIRE(a->count >= 0 && a->heads > 0 && a->num_pages > 0, "bad sizes");
  LKV_REQUIRE(a->page_bytes == 8192 || a->page_bytes == 4096, "page_bytes must be 8192 (bf16) or 4096 (8 bits), got %d", a->page_bytes);
  LKV_REQUIRE(a->k && a->v, "null tensor");
  LKV_REQUIRE((a->k_scales == nullptr) == (a->v_scales == nullptr), "k_scales and v_scales must both be set");
  LKV_REQUIRE(((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15) == 0 &&
                  ((a->page_stride | a->head_stride) & 15) == 0,
              "pages must be 16-byte aligned");
  LKV_REQUIRE(a->page_stride >= a->page_bytes && a->head_stride >= 0 && a->scale_head_stride >= 0, "pages must not overlap");
  LKV_REQUIRE(a->heads <= 65535, "heads must be <= 65535");
  if (a->count == 0) return LKV_OK;
  LKV_REQUIRE(a->src && a->dst, "null page lists");
  if (const int32_t st = check_pairs(a)) return st;
  CopyParams p;
  p.pool[0] = static_cast<uint8_t*>(a->k);
  p.pool[1] = static_cast<uint8_t*>(a->v);
  p.scales[0] = static_cast<uint8_t*>(a->k_scales);
  p.scales[1] = static_cast<uint8_t*>(a->v_scales);
  p.page = a->page_stride;
  p.head = a->head_stride;
  p.scale_head = a->scale_head_stride;
  p.page_bytes = a->page_bytes;
  for (int32_t i = 0; i < a->count;) {
    CopyRuns r;
    r.n = 0;
    p.total = 0;
    while (i < a->count) {
      int32_t m = 1;
      while (i + m < a->count && a->src[i + m] == a->src[i] + m && a->dst[i + m] == a->dst[i] + m) ++m;
      r.src[r.n] = a->src[i];
      r.dst[r.n] = a->dst[i];
      p.total += m;
      r.end[r.n] = p.total;
      i += m;
      if (++r.n == kRuns) break;
    }
    const dim3 grid((p.total + kPagesPerItem - 1) / kPagesPerItem, a->heads, 2);
    if (a->page_bytes == 8192)
      copy_pages_kernel<2><<<grid, 256, 0, as_stream(stream)>>>(p, r);
    else
      copy_pages_kernel<1><<<grid, 256, 0, as_stream(stream)>>>(p, r);
    if (const int32_t st = check_launch("lkv_copy_pages")) return st;
  }
  return LKV_OK;
}
