// llmk_pages.hip — the pages of a cache on the device (gfx950): rows fork,
// grow, shrink and end (pages_fork_kernel, pages_release_kernel,
// pages_grow_kernel), live pages move to the front (pages_rank_kernel,
// pages_list_kernel, pages_move_kernel, pages_remap_kernel), pages are copied
// (pages_copy_kernel).
//
// The state is whole numbers, and every result is the one that the rows
// taken one after another give: counts change by atomics whose order does not
// matter, and what depends on an order (which page a row gets) comes from
// prefix sums over rows and pages.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "llmk_device.h"
#include "llmk_host.h"

namespace llmk {

struct Cache {
  uint32_t rows, max_pages, page_tokens, num_pages;
  uint32_t *table, *lengths, *refs, *used;
  uint32_t words;     // of `used`
  uint32_t* n_moves;  // [2]: pages to copy; pages in use (compaction)
  u2v* moves;         // (from, to)
  uint32_t* holders;  // [num_pages]: growing rows that share a partly filled page ...
  uint32_t* last;     // [num_pages]: ... and 1 + the last of them; 0 between calls
  uint32_t* list;     // [num_pages]: the free pages in ascending order
  uint32_t* mark;     // [rows]: the page a row counted itself at, or EMPTY
  uint32_t* rank;     // [2 * words]: pages that move / holes before each word
};

__device__ __forceinline__ uint32_t pages_of(const Cache& c, uint32_t tokens) {
  return (tokens + c.page_tokens - 1) / c.page_tokens;
}

// ---- update ----------------------------------------------------------------
// Step 1: the child's table begins as its parent's, and every page shared gains
// a holder.  One workgroup per row.
constexpr uint32_t FT = 256;
__global__ __launch_bounds__(FT) void pages_fork_kernel(Cache c, const int32_t* parents,
                                                        const int32_t* new_lengths,
                                                        uint32_t* granted, uint32_t* status) {
  const uint32_t r = blockIdx.x;
  const int32_t p = G(parents)[r];
  if (p < 0) return;
  const uint32_t own = G(c.lengths)[r];
  bool ok = (uint32_t)p < c.rows && (uint32_t)p != r && own == 0;
  const int32_t want = new_lengths ? G(new_lengths)[r] : -1;
  const uint64_t most = (uint64_t)c.max_pages * c.page_tokens;
  if (want > 0 && (uint64_t)(uint32_t)want > most) ok = false;
  uint32_t len = 0;
  if (ok) {
    ok = G(parents)[p] < 0;
    len = G(c.lengths)[p];
    if (len > most) ok = false;
  }
  if (!ok) {  // the whole workgroup agrees
    if (threadIdx.x == 0) {
      G(granted)[r] = 0;
      atomicOr(status, LLMK_STATUS_INVALID_PARAMS);
    }
    return;
  }
  if (want >= 0 && (uint32_t)want < len) len = (uint32_t)want;
  const uint32_t n = pages_of(c, len);
  const uint32_t* from = c.table + (uint64_t)(uint32_t)p * c.max_pages;
  uint32_t* to = c.table + (uint64_t)r * c.max_pages;
  for (uint32_t j = threadIdx.x; j < n; j += FT) {
    const uint32_t e = G(from)[j];
    G(to)[j] = e;
    if (e < c.num_pages)
      atomicAdd(c.refs + e, 1u);
    else
      atomicOr(status, LLMK_STATUS_INVALID_PARAMS);  // not a page: the table was not kept
  }
  __syncthreads();  // every wave has read the row's own length
  if (threadIdx.x == 0) {
    G(c.lengths)[r] = len;
    G(granted)[r] = 1;
  }
}

// Whether row r takes part in steps 2 and 3, and the length it asks for.
__device__ __forceinline__ bool asks(const Cache& c, const int32_t* parents,
                                     const int32_t* new_lengths, const uint32_t* granted,
                                     uint32_t r, uint32_t& want) {
  const int32_t w = G(new_lengths)[r];
  if (w < 0) return false;
  if (parents && G(parents)[r] >= 0 && G(granted)[r] == 0) return false;  // refused
  want = (uint32_t)w;
  return (uint64_t)want <= (uint64_t)c.max_pages * c.page_tokens;
}
__device__ __forceinline__ uint32_t table_entry(const Cache& c, uint32_t r, uint32_t j) {
  return G(c.table)[(uint64_t)r * c.max_pages + j];
}

// Step 2: pages past a row's new end lose a holder; those that lose the last
// one are free.  Rows that will write into a partly filled shared page are
// counted per page for step 3 (counts only fall here, so one that is shared
// after this launch is shared whenever it is looked at).
__global__ __launch_bounds__(FT) void pages_release_kernel(Cache c, const int32_t* parents,
                                                           const int32_t* new_lengths,
                                                           uint32_t* granted, uint32_t* status) {
  const uint32_t r = blockIdx.x;
  if (r == 0 && threadIdx.x == 0) G(c.n_moves)[0] = 0;
  if (!new_lengths) {
    if (threadIdx.x == 0 && !(parents && G(parents)[r] >= 0)) G(granted)[r] = 1;
    return;
  }
  uint32_t want = 0;
  if (!asks(c, parents, new_lengths, granted, r, want)) {
    if (threadIdx.x == 0) {
      G(c.mark)[r] = EMPTY;
      if (!(parents && G(parents)[r] >= 0)) {
        const bool too_long = G(new_lengths)[r] > 0;
        G(granted)[r] = too_long ? 0u : 1u;
        if (too_long) atomicOr(status, LLMK_STATUS_INVALID_PARAMS);
      }
    }
    return;
  }
  const uint32_t cur = G(c.lengths)[r];
  uint32_t marked = EMPTY;
  if (want < cur) {
    uint32_t n = pages_of(c, cur);
    if (n > c.max_pages) n = c.max_pages;
    for (uint32_t j = pages_of(c, want) + threadIdx.x; j < n; j += FT) {
      const uint32_t e = table_entry(c, r, j);
      const uint32_t had = e < c.num_pages ? atomicSub(c.refs + e, 1u) : 0u;
      if (had == 1) atomicAnd(c.used + (e >> 5), ~(1u << (e & 31u)));
      if (had == 0) {  // not a page, or one nobody held: the cache was not kept
        if (e < c.num_pages) atomicAdd(c.refs + e, 1u);
        atomicOr(status, LLMK_STATUS_INVALID_PARAMS);
      }
    }
    __syncthreads();  // every wave has read the old length
    if (threadIdx.x == 0) G(c.lengths)[r] = want;
  } else if (want > cur && threadIdx.x == 0 && cur % c.page_tokens != 0) {
    const uint32_t e = table_entry(c, r, cur / c.page_tokens);
    if (e < c.num_pages &&
        __hip_atomic_load(c.refs + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) > 1u) {
      atomicAdd(c.holders + e, 1u);
      atomicMax(c.last + e, r + 1);
      marked = e;
    }
  }
  if (threadIdx.x == 0) {
    G(granted)[r] = 1;
    G(c.mark)[r] = marked;
  }
}

// Exclusive prefix sum over a workgroup of NT threads, x <= 2^25 + 1 (a wave's
// sum fits 32 bits).
__device__ __forceinline__ uint64_t scan_wide(uint32_t x, LDS uint32_t* red, uint64_t& total) {
  const uint32_t lane = threadIdx.x & 63u, wv = threadIdx.x >> 6;
  const uint32_t incl = wave_incl_scan(x);
  if (lane == 63) red[wv] = incl;
  __syncthreads();
  uint64_t off = 0, sum = 0;
#pragma unroll
  for (uint32_t i = 0; i < NW; ++i) {
    off += i < wv ? red[i] : 0u;
    sum += red[i];
  }
  __syncthreads();
  total = sum;
  return off + incl - x;
}

// The pages in use among a word of `used` (bits past the last page are none).
__device__ __forceinline__ uint32_t used_bits(const Cache& c, uint32_t w) {
  const uint32_t past = c.num_pages - 32 * w;  // pages from the word's first on
  return G(c.used)[w] & (past >= 32 ? 0xffffffffu : (1u << past) - 1u);
}
__device__ __forceinline__ uint32_t page_bits(const Cache& c, uint32_t w) {
  const uint32_t past = c.num_pages - 32 * w;
  return past >= 32 ? 0xffffffffu : (1u << past) - 1u;
}

// Step 3, one workgroup.  The free pages in ascending order (each thread the
// free bits of its run of words, a prefix sum over threads), the rows' needs
// (a prefix sum over rows), then each row's pages.  Counts of shared pages
// stay as step 2 left them until every row has read them; the last of the
// rows that share a page and all grow keeps it.
__global__ __launch_bounds__(NT) void pages_grow_kernel(Cache c, const int32_t* parents,
                                                        const int32_t* new_lengths,
                                                        uint32_t* granted, uint32_t* status) {
  __shared__ uint32_t s_red[NW], s_job[NT][4];
  __shared__ uint32_t s_jobs, s_moves;
  LDS uint32_t* red = (LDS uint32_t*)s_red;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
  const uint32_t per = (c.words + NT - 1) / NT;
  const uint32_t w0 = umin(tid * per, c.words), w1 = umin(w0 + per, c.words);
  uint32_t mine = 0, nfree = 0;
  for (uint32_t w = w0; w < w1; ++w) mine += __popc(page_bits(c, w) & ~used_bits(c, w));
  uint32_t at = block_excl_scan(mine, red, nfree);
  for (uint32_t w = w0; w < w1; ++w)
    for (uint32_t m = page_bits(c, w) & ~used_bits(c, w); m; m &= m - 1)
      G(c.list)[at++] = 32 * w + (uint32_t)__builtin_ctz(m);
  if (tid == 0) s_moves = 0;

  uint64_t total = 0;  // pages asked for by the rows so far
  for (uint32_t r0 = 0; r0 < c.rows; r0 += NT) {
    const uint32_t r = r0 + tid;
    uint32_t want = 0, cur = 0, e = EMPTY, need = 0;
    bool grow = false, tied = false, copy = false;
    if (r < c.rows && asks(c, parents, new_lengths, granted, r, want)) {
      cur = G(c.lengths)[r];
      grow = want > cur;
      e = G(c.mark)[r];
      if (grow && e != EMPTY) {
        const uint32_t refs = G(c.refs)[e];
        tied = refs > 1;
        copy = tied && !(G(c.holders)[e] == refs && G(c.last)[e] == r + 1);
      }
      if (grow) need = pages_of(c, want) - pages_of(c, cur) + (copy ? 1u : 0u);
    }
    if (tid == 0) s_jobs = 0;
    uint64_t sum = 0;
    const uint64_t first = total + scan_wide(umin(need, nfree + 1), red, sum);
    if (grow && first + need > nfree && (need || tied)) {
      G(granted)[r] = 0;
      atomicOr(status, LLMK_STATUS_PAGES_FULL);
      grow = false;
    }
    if (grow) {
      G(c.lengths)[r] = want;
      if (need) {
        const uint32_t k = __hip_atomic_fetch_add((LDS uint32_t*)&s_jobs, 1u, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_WORKGROUP);
        s_job[k][0] = r;
        s_job[k][1] = pages_of(c, cur) - (copy ? 1u : 0u);  // its first new table entry
        s_job[k][2] = (uint32_t)first;
        s_job[k][3] = need;
        if (copy) {
          const uint32_t i = __hip_atomic_fetch_add((LDS uint32_t*)&s_moves, 1u, __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_WORKGROUP);
          G(c.moves)[i] = u2v{e, G(c.list)[first]};
        }
      }
    }
    __syncthreads();
    for (uint32_t k = wv; k < s_jobs; k += NW) {  // a wave per row
      const uint32_t row = s_job[k][0], j0 = s_job[k][1], f = s_job[k][2], n = s_job[k][3];
      for (uint32_t i = lane; i < n; i += WAVE) {
        const uint32_t p = G(c.list)[f + i];
        G(c.table)[(uint64_t)row * c.max_pages + j0 + i] = p;
        G(c.refs)[p] = 1;
        atomicOr(c.used + (p >> 5), 1u << (p & 31u));
      }
    }
    total += sum;
    __syncthreads();  // the jobs are read
  }
  // the copied pages lose the rows that left them; the marks are cleared for
  // the next call
  for (uint32_t i = tid; i < s_moves; i += NT) atomicSub(c.refs + G(c.moves)[i][0], 1u);
  for (uint32_t r = tid; r < c.rows; r += NT) {
    const uint32_t e = G(c.mark)[r];
    if (e != EMPTY) {
      G(c.holders)[e] = 0;
      G(c.last)[e] = 0;
    }
  }
  if (tid == 0) G(c.n_moves)[0] = s_moves;
}

// ---- compaction --------------------------------------------------------------
// One workgroup: the number M of pages in use, and before each word of `used`
// the used pages at or above M (which move) and the free ones below M (the
// holes).  There are as many of one as of the other.
__global__ __launch_bounds__(NT) void pages_rank_kernel(Cache c) {
  __shared__ uint32_t s_red[NW];
  LDS uint32_t* red = (LDS uint32_t*)s_red;
  const uint32_t tid = threadIdx.x, per = (c.words + NT - 1) / NT;
  const uint32_t w0 = umin(tid * per, c.words), w1 = umin(w0 + per, c.words);
  uint32_t n = 0, M = 0, moving = 0, holes = 0;
  for (uint32_t w = w0; w < w1; ++w) n += __popc(used_bits(c, w));
  (void)block_excl_scan(n, red, M);
  auto below = [&](uint32_t w) {  // the word's pages below M
    return 32 * w + 32 <= M ? 0xffffffffu : (32 * w >= M ? 0u : (1u << (M - 32 * w)) - 1u);
  };
  uint32_t a = 0, b = 0;
  for (uint32_t w = w0; w < w1; ++w) {
    const uint32_t u = used_bits(c, w), lo = below(w);
    a += __popc(u & ~lo);
    b += __popc(~u & lo);
  }
  a = block_excl_scan(a, red, moving);
  b = block_excl_scan(b, red, holes);
  for (uint32_t w = w0; w < w1; ++w) {
    const uint32_t u = used_bits(c, w), lo = below(w);
    G(c.rank)[w] = a;
    G(c.rank)[c.words + w] = b;
    a += __popc(u & ~lo);
    b += __popc(~u & lo);
  }
  if (tid == 0) {
    G(c.n_moves)[0] = moving;
    G(c.n_moves)[1] = M;
  }
}
// Every page: its place among those that move, or among the holes.
__global__ __launch_bounds__(FT) void pages_list_kernel(Cache c, uint32_t* map) {
  const uint32_t p = blockIdx.x * FT + threadIdx.x;
  if (p >= c.num_pages) return;
  const uint32_t w = p >> 5, bit = 1u << (p & 31u), M = G(c.n_moves)[1];
  const uint32_t u = used_bits(c, w);
  const uint32_t lo = 32 * w + 32 <= M ? 0xffffffffu : (32 * w >= M ? 0u : (1u << (M - 32 * w)) - 1u);
  GLB uint32_t* pair = (GLB uint32_t*)G(c.moves);
  if (u & ~lo & bit) pair[2 * (G(c.rank)[w] + __popc(u & ~lo & (bit - 1)))] = p;
  if (~u & lo & bit) pair[2 * (G(c.rank)[c.words + w] + __popc(~u & lo & (bit - 1))) + 1] = p;
  G(map)[p] = p;
}
// The pairs' counts, the map, and the words of `used` as they are afterwards.
__global__ __launch_bounds__(FT) void pages_move_kernel(Cache c, uint32_t* map) {
  const uint32_t n = G(c.n_moves)[0], M = G(c.n_moves)[1];
  const uint32_t step = gridDim.x * FT;
  for (uint32_t i = blockIdx.x * FT + threadIdx.x; i < n; i += step) {
    const u2v m = G(c.moves)[i];
    G(map)[m[0]] = m[1];
    G(c.refs)[m[1]] = G(c.refs)[m[0]];
    G(c.refs)[m[0]] = 0;
  }
  for (uint32_t w = blockIdx.x * FT + threadIdx.x; w < c.words; w += step)
    G(c.used)[w] = 32 * w + 32 <= M ? 0xffffffffu : (32 * w >= M ? 0u : (1u << (M - 32 * w)) - 1u);
}
__global__ __launch_bounds__(FT) void pages_remap_kernel(Cache c, const uint32_t* map) {
  const uint32_t r = blockIdx.x;
  uint32_t n = pages_of(c, G(c.lengths)[r]);
  if (n > c.max_pages) n = c.max_pages;
  uint32_t* row = c.table + (uint64_t)r * c.max_pages;
  for (uint32_t j = threadIdx.x; j < n; j += FT) {
    const uint32_t e = G(row)[j];
    if (e < c.num_pages) G(row)[j] = G(map)[e];
  }
}

// ---- copies ------------------------------------------------------------------
struct Copies {
  uint32_t n_pools;
  uint64_t page_bytes;  // the largest
  const uint64_t* pools;  // [n_pools][2]: address, bytes per page
  uint32_t num_pages;
  const uint32_t *src, *dst;  // n pairs, or
  uint32_t n;
  const u2v* moves;           // n_moves[0] pairs of the update or compaction
  const uint32_t* n_moves;
  uint32_t* status;
};

// Work items are (pair, pool, piece of CPIECE bytes), taken in turn by the
// workgroups: the number of pairs may be known on the device alone.
constexpr uint32_t CT = 256, CPIECE = CT * 16 * 4;
__global__ __launch_bounds__(CT) void pages_copy_kernel(Copies a) {
  const uint32_t n = a.moves ? G(a.n_moves)[0] : a.n;
  const uint64_t pieces = (a.page_bytes + CPIECE - 1) / CPIECE;
  const uint64_t items = n * pieces * a.n_pools;
  for (uint64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const uint64_t pair = it / (pieces * a.n_pools), rest = it - pair * (pieces * a.n_pools);
    const uint32_t pool = (uint32_t)(rest / pieces);
    const uint64_t at = (rest - pool * pieces) * CPIECE;
    uint32_t from, to;
    if (a.moves) {
      const u2v m = G(a.moves)[pair];
      from = m[0];
      to = m[1];
    } else {
      from = G(a.src)[pair];
      to = G(a.dst)[pair];
    }
    if (from >= a.num_pages || to >= a.num_pages) {
      if (rest == 0 && threadIdx.x == 0) atomicOr(a.status, LLMK_STATUS_INVALID_PARAMS);
      continue;
    }
    const uint64_t base = G(a.pools)[2 * pool], size = G(a.pools)[2 * pool + 1];
    if (at >= size) continue;
    const uint64_t s = base + from * size + at, d = base + to * size + at;
    const uint32_t len = (uint32_t)(size - at < CPIECE ? size - at : CPIECE);
    const uint32_t t = threadIdx.x;
    if (((s | d) & 15u) == 0) {
      u4v x[4];
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t o = (k * CT + t) * 16;
        if (o + 16 <= len) x[k] = *(const GLB u4v*)(s + o);
      }
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t o = (k * CT + t) * 16;
        if (o + 16 <= len) *(GLB u4v*)(d + o) = x[k];
      }
      for (uint32_t o = (len & ~15u) + t; o < len; o += CT)
        *(GLB uint8_t*)(d + o) = *(const GLB uint8_t*)(s + o);
    } else if (((s | d | len) & 3u) == 0) {
      for (uint32_t o = 4 * t; o < len; o += 4 * CT)
        *(GLB uint32_t*)(d + o) = *(const GLB uint32_t*)(s + o);
    } else {
      for (uint32_t o = t; o < len; o += CT)
        *(GLB uint8_t*)(d + o) = *(const GLB uint8_t*)(s + o);
    }
  }
}

}  // namespace llmk

// ===========================================================================
using namespace llmk;

// The work array: two words, the pairs to copy, then the arrays of Cache.
static uint64_t most_moves(uint32_t rows, uint32_t num_pages) {
  const uint64_t half = (uint64_t)num_pages / 2 + 1;
  return rows > half ? rows : half;
}
static int check_limits(uint32_t rows, uint32_t num_pages) {
  if (rows == 0 || num_pages == 0)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "rows and num_pages must be > 0");
  if (rows > (1u << 20)) return fail(LLMK_ERR_CAPACITY, "rows above 2^20");
  if (num_pages > (1u << 25)) return fail(LLMK_ERR_CAPACITY, "num_pages above 2^25");
  return LLMK_OK;
}

extern "C" int llmk_pages_work_words(uint32_t rows, uint32_t num_pages, uint64_t* words) {
  if (!words) return fail(LLMK_ERR_INVALID_ARGUMENT, "words is NULL");
  const int rc = check_limits(rows, num_pages);
  if (rc != LLMK_OK) return rc;
  *words = 2 + 2 * most_moves(rows, num_pages) + 3ull * num_pages + rows +
           2ull * ((num_pages + 31) / 32);
  return LLMK_OK;
}

static int check_pools(uint32_t n_pools, const uint64_t* pools, uint64_t page_bytes) {
  if (n_pools > 65535) return fail(LLMK_ERR_CAPACITY, "n_pools above 65535");
  if (n_pools && (!pools || page_bytes == 0))
    return fail(LLMK_ERR_INVALID_ARGUMENT, "pools and page_bytes are required");
  if (page_bytes > (1ull << 40)) return fail(LLMK_ERR_CAPACITY, "page_bytes above 2^40");
  return LLMK_OK;
}

static int check_cache(llmk_sampler* s, const llmk_page_cache* k, Cache& c) {
  if (!s) return fail(LLMK_ERR_INVALID_ARGUMENT, "sampler is NULL");
  if (!k) return fail(LLMK_ERR_INVALID_ARGUMENT, "cache is NULL");
  int rc = check_limits(k->rows, k->num_pages);
  if (rc == LLMK_OK) rc = check_pools(k->n_pools, k->pools, k->page_bytes);
  if (rc != LLMK_OK) return rc;
  if (k->max_pages == 0 || k->page_tokens == 0)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "max_pages and page_tokens must be > 0");
  if ((uint64_t)k->max_pages * k->page_tokens > 0x7fffffffu)
    return fail(LLMK_ERR_CAPACITY, "max_pages * page_tokens above 2^31 - 1");
  if (!k->table || !k->lengths || !k->refs || !k->used || !k->work)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "table, lengths, refs, used and work are required");
  if (((uintptr_t)k->work % 8) != 0)
    return fail(LLMK_ERR_ALIGNMENT, "work must be 8-byte aligned");
  c.rows = k->rows;
  c.max_pages = k->max_pages;
  c.page_tokens = k->page_tokens;
  c.num_pages = k->num_pages;
  c.table = k->table;
  c.lengths = k->lengths;
  c.refs = k->refs;
  c.used = k->used;
  c.words = (k->num_pages + 31) / 32;
  c.n_moves = k->work;
  c.moves = (u2v*)(k->work + 2);
  c.holders = k->work + 2 + 2 * most_moves(k->rows, k->num_pages);
  c.last = c.holders + k->num_pages;
  c.list = c.last + k->num_pages;
  c.mark = c.list + k->num_pages;
  c.rank = c.mark + k->rows;
  return LLMK_OK;
}

// Enough workgroups for 8 per CU; fewer if there are fewer pieces.
constexpr uint32_t COPY_GRID = 2048;
static int launch_copies(const Copies& a, uint64_t most_pairs, void* stream) {
  const uint64_t pieces = (a.page_bytes + CPIECE - 1) / CPIECE;
  const uint64_t per = pieces * a.n_pools;
  uint64_t grid = most_pairs > COPY_GRID / per ? COPY_GRID : most_pairs * per;
  if (grid == 0) return LLMK_OK;
  hipLaunchKernelGGL(pages_copy_kernel, dim3((uint32_t)grid), dim3(CT), 0, (hipStream_t)stream, a);
  HIPCHK(hipGetLastError());
  return LLMK_OK;
}
static int launch_moves(llmk_sampler* s, const llmk_page_cache* k, const Cache& c,
                        uint64_t most_pairs, void* stream) {
  if (k->n_pools == 0) return LLMK_OK;
  Copies a{};
  a.n_pools = k->n_pools;
  a.page_bytes = k->page_bytes;
  a.pools = k->pools;
  a.num_pages = k->num_pages;
  a.moves = c.moves;
  a.n_moves = c.n_moves;
  a.status = s->ws.status;
  return launch_copies(a, most_pairs, stream);
}

extern "C" int llmk_pages_update(llmk_sampler* s, const llmk_page_cache* cache,
                                 const int32_t* parents, const int32_t* new_lengths,
                                 uint32_t* out_granted, void* stream) {
  Cache c;
  const int rc = check_cache(s, cache, c);
  if (rc != LLMK_OK) return rc;
  if (!parents && !new_lengths)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "neither parents nor new_lengths: nothing is asked for");
  if (!out_granted) return fail(LLMK_ERR_INVALID_ARGUMENT, "out_granted is required");
  HIPCHK(hipSetDevice(s->device));
  hipStream_t st = (hipStream_t)stream;
  if (parents) {
    hipLaunchKernelGGL(pages_fork_kernel, dim3(c.rows), dim3(FT), 0, st, c, parents, new_lengths,
                       out_granted, s->ws.status);
    HIPCHK(hipGetLastError());
  }
  hipLaunchKernelGGL(pages_release_kernel, dim3(c.rows), dim3(FT), 0, st, c, parents, new_lengths,
                     out_granted, s->ws.status);
  HIPCHK(hipGetLastError());
  if (!new_lengths) return LLMK_OK;
  hipLaunchKernelGGL(pages_grow_kernel, dim3(1), dim3(NT), 0, st, c, parents, new_lengths,
                     out_granted, s->ws.status);
  HIPCHK(hipGetLastError());
  return launch_moves(s, cache, c, c.rows, stream);
}

extern "C" int llmk_pages_compact(llmk_sampler* s, const llmk_page_cache* cache,
                                  uint32_t* out_map, void* stream) {
  Cache c;
  const int rc = check_cache(s, cache, c);
  if (rc != LLMK_OK) return rc;
  if (!out_map) return fail(LLMK_ERR_INVALID_ARGUMENT, "out_map is required");
  HIPCHK(hipSetDevice(s->device));
  hipStream_t st = (hipStream_t)stream;
  const uint32_t blocks = (c.num_pages + FT - 1) / FT;
  hipLaunchKernelGGL(pages_rank_kernel, dim3(1), dim3(NT), 0, st, c);
  HIPCHK(hipGetLastError());
  hipLaunchKernelGGL(pages_list_kernel, dim3(blocks), dim3(FT), 0, st, c, out_map);
  HIPCHK(hipGetLastError());
  hipLaunchKernelGGL(pages_move_kernel, dim3(blocks < 1024 ? blocks : 1024), dim3(FT), 0, st, c,
                     out_map);
  HIPCHK(hipGetLastError());
  hipLaunchKernelGGL(pages_remap_kernel, dim3(c.rows), dim3(FT), 0, st, c,
                     (const uint32_t*)out_map);
  HIPCHK(hipGetLastError());
  return launch_moves(s, cache, c, (uint64_t)c.num_pages / 2 + 1, stream);
}

extern "C" int llmk_pages_copy(llmk_sampler* s, uint32_t n_pools, const uint64_t* pools,
                               uint64_t page_bytes, uint32_t num_pages, uint32_t n,
                               const uint32_t* src, const uint32_t* dst, void* stream) {
  if (!s) return fail(LLMK_ERR_INVALID_ARGUMENT, "sampler is NULL");
  const int rc = check_pools(n_pools, pools, page_bytes);
  if (rc != LLMK_OK) return rc;
  if (n && (!src || !dst)) return fail(LLMK_ERR_INVALID_ARGUMENT, "src and dst are required");
  if (n == 0 || n_pools == 0) return LLMK_OK;
  HIPCHK(hipSetDevice(s->device));
  Copies a{};
  a.n_pools = n_pools;
  a.page_bytes = page_bytes;
  a.pools = pools;
  a.num_pages = num_pages;
  a.src = src;
  a.dst = dst;
  a.n = n;
  a.status = s->ws.status;
  return launch_copies(a, n, stream);
}
