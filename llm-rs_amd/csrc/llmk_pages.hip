// llmk_pages.hip — the pages of a cache on the device (gfx950): rows fork,
// grow, shrink and end (pages_update_kernel), live pages move to the front
// (pages_plan_kernel, pages_compact_kernel), pages are copied
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
#include "llmk_sync.h"

namespace llmk {

struct Cache {
  uint32_t rows, max_pages, page_tokens, num_pages;
  uint32_t *table, *lengths, *refs, *used;
  uint32_t words;     // of `used`
  uint32_t* ctl;      // [CTL_WORDS], below; the counts are 0 between calls
  u2v* moves;         // (from, to)
  uint32_t* holders;  // [num_pages]: growing rows that share a partly filled page ...
  uint32_t* last;     // [num_pages]: ... and 1 + the last of them; 0 between calls
  uint32_t* list;     // [num_pages]: free pages in ascending order; ranks (compaction)
  uint32_t* freed;    // [num_pages]: pages whose last holder left
  uint32_t* row;      // [rows][4]: what each row asks for
};
enum : uint32_t { CTL_MOVES = 0, CTL_LIVE = 1, CTL_ARRIVE = 2, CTL_FREED = 3, CTL_WORDS = 4 };

__device__ __forceinline__ uint32_t pages_of(const Cache& c, uint32_t tokens) {
  return (tokens + c.page_tokens - 1) / c.page_tokens;
}
__device__ __forceinline__ uint32_t table_entry(const Cache& c, uint32_t r, uint32_t j) {
  return G(c.table)[(uint64_t)r * c.max_pages + j];
}
// The pages of a word of `used`, and those in use.
__device__ __forceinline__ uint32_t page_bits(const Cache& c, uint32_t w) {
  const uint32_t past = c.num_pages - 32 * w;  // pages from the word's first on
  return past >= 32 ? 0xffffffffu : (1u << past) - 1u;
}
__device__ __forceinline__ uint32_t used_bits(const Cache& c, uint32_t w) {
  return G(c.used)[w] & page_bits(c, w);
}
constexpr uint32_t UT = 512, UW = UT / WAVE;  // threads and waves of an update's workgroups
constexpr uint32_t FREE_LDS = 4096;           // free pages listed, and words of pages, in LDS

// Exclusive prefix sum over UT threads, x <= 2^25 + 1 (a wave's sum fits 32 bits).
__device__ __forceinline__ uint64_t update_scan(uint32_t x, LDS uint32_t* red, uint64_t& total) {
  const uint32_t lane = threadIdx.x & 63u, wv = threadIdx.x >> 6;
  const uint32_t incl = wave_incl_scan(x);
  if (lane == 63) red[wv] = incl;
  lds_barrier();
  uint64_t off = 0, sum = 0;
#pragma unroll
  for (uint32_t i = 0; i < UW; ++i) {
    off += i < wv ? red[i] : 0u;
    sum += red[i];
  }
  lds_barrier();
  total = sum;
  return off + incl - x;
}

// The same of y, with the sum of x beside it.
__device__ __forceinline__ uint64_t update_scan_and_sum(uint32_t y, uint32_t x, LDS uint32_t* red,
                                                        uint64_t& total, uint64_t& sum_x) {
  const uint32_t lane = threadIdx.x & 63u, wv = threadIdx.x >> 6;
  const uint32_t incl = wave_incl_scan(y), all = wave_incl_scan(x);
  if (lane == 63) {
    red[wv] = incl;
    red[UW + wv] = all;
  }
  lds_barrier();
  uint64_t off = 0, sum = 0, xs = 0;
#pragma unroll
  for (uint32_t i = 0; i < UW; ++i) {
    off += i < wv ? red[i] : 0u;
    sum += red[i];
    xs += red[UW + i];
  }
  lds_barrier();
  total = sum;
  sum_x = xs;
  return off + incl - y;
}

// What a row asks for, as its workgroup leaves it for the last one, and the
// counts at the page it marked.
struct Request {
  uint32_t cur;   // its tokens after steps 1 and 2
  uint32_t want;  // EMPTY: no growth is asked for
  uint32_t mark;  // the shared page it counted itself at, or EMPTY
  uint32_t refs, holders, last;
  uint32_t need, tied, copy;
};
__device__ __forceinline__ Request no_request() { return {0, EMPTY, EMPTY, 0, 0, 0, 0, 0, 0}; }
// (in two steps, so that other loads can go with each)
__device__ __forceinline__ Request read_request(const Cache& c, uint32_t r) {
  Request q = no_request();
  const uint32_t* p = c.row + 4 * (uint64_t)r;
  q.cur = get_agent(p);
  q.want = get_agent(p + 1);
  q.mark = get_agent(p + 2);
  return q;
}
__device__ __forceinline__ void read_mark(const Cache& c, Request& q) {
  const uint32_t e = umin(q.mark, c.num_pages - 1);
  q.refs = get_agent(c.refs + e);
  q.holders = get_agent(c.holders + e);
  q.last = get_agent(c.last + e);
}
__device__ __forceinline__ void settle(const Cache& c, uint32_t r, Request& q) {
  if (q.want == EMPTY) return;
  q.tied = q.mark != EMPTY && q.refs > 1;
  q.copy = q.tied && !(q.holders == q.refs && q.last == r + 1);
  q.need = pages_of(c, q.want) - pages_of(c, q.cur) + q.copy;
}
__device__ __forceinline__ Request request_of(const Cache& c, uint32_t r) {
  Request q = read_request(c, r);
  read_mark(c, q);
  settle(c, r, q);
  return q;
}

// One launch.  A workgroup per row does what rows can do at the same time:
// a child takes its parent's table and raises the pages' counts (step 1), a row
// that shrinks lowers them and notes the pages that reach 0 (step 2), a row
// that grows counts itself at the partly filled page it may share.  Lengths
// stay as they are meanwhile, so a parent may change in the same call; no row
// reads a table that another one writes, since a parent is never a child.
// The counts are sums, whatever their order: a page that reached 0 has been
// given up by every row that held it before, and if forks took it up again its
// count says so at the end.
//
// The last workgroup to finish then takes the rows in order: the pages that
// are free now, the rows' needs (a prefix sum over rows), the lowest free pages
// (a prefix sum over the words of `used`), and each row's share of them.  The
// counts of shared pages change only when every row has read them; of the rows
// that share a page and all grow, the last keeps it.
//
// Bound by latency, 256 rows of 80 K pages 18 us: 5 until every row has arrived,
// 5 for what the last workgroup reads and for the pages given up, 3 for sums and
// the list of free pages, 5 for the rows' shares.  (As four launches 29 us; the
// sums of pages and rows apart, and the words without the taken pages in a pass
// of their own, 20.)  Reading more freed pages at once, spreading them over the
// lanes and smaller code changed nothing.
__global__ __launch_bounds__(UT) void pages_update_kernel(Cache c, const int32_t* parents,
                                                          const int32_t* new_lengths,
                                                          uint32_t* granted, uint32_t* status) {
  __shared__ uint32_t s_red[2 * UW], s_job[UT][4], s_free[FREE_LDS], s_word[FREE_LDS];
  __shared__ uint32_t s_jobs, s_moves, s_taken, s_last;
  LDS uint32_t* red = (LDS uint32_t*)s_red;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
  {
    const uint32_t r = blockIdx.x;
    const int32_t p = parents ? G(parents)[r] : -1, w = new_lengths ? G(new_lengths)[r] : -1;
    const uint32_t own = G(c.lengths)[r];
    const uint64_t most = (uint64_t)c.max_pages * c.page_tokens;
    bool ok = w < 0 || (uint64_t)(uint32_t)w <= most;
    uint32_t cur = own;
    if (p >= 0) {
      ok = ok && (uint32_t)p < c.rows && (uint32_t)p != r && own == 0;
      if (ok) {
        cur = G(c.lengths)[p];
        ok = G(parents)[p] < 0 && cur <= most;
      }
    }
    uint32_t want = EMPTY, mark = EMPTY;
    if (!ok) {
      cur = own;
      if (tid == 0) atomicOr(status, LLMK_STATUS_INVALID_PARAMS);
    } else {
      if (p >= 0) {
        if (w >= 0 && (uint32_t)w < cur) cur = (uint32_t)w;
        const uint32_t n = pages_of(c, cur);
        for (uint32_t j = tid; j < n; j += UT) {
          const uint32_t e = table_entry(c, (uint32_t)p, j);
          put_agent(c.table + (uint64_t)r * c.max_pages + j, e);
          if (e < c.num_pages)
            atomicAdd(c.refs + e, 1u);
          else
            atomicOr(status, LLMK_STATUS_INVALID_PARAMS);  // not a page: the table was not kept
        }
      }
      if (w >= 0 && (uint32_t)w < cur) {
        uint32_t n = pages_of(c, cur);
        if (n > c.max_pages) n = c.max_pages;
        for (uint32_t j = pages_of(c, (uint32_t)w) + tid; j < n; j += UT) {
          const uint32_t e = table_entry(c, r, j);
          const uint32_t had = e < c.num_pages ? atomicSub(c.refs + e, 1u) : 0u;
          if (had == 1) {
            const uint32_t at = atomicAdd(c.ctl + CTL_FREED, 1u);
            if (at < c.num_pages) put_agent(c.freed + at, e);
          }
          if (had == 0) {  // not a page, or one nobody held: the cache was not kept
            if (e < c.num_pages) atomicAdd(c.refs + e, 1u);
            atomicOr(status, LLMK_STATUS_INVALID_PARAMS);
          }
        }
        cur = (uint32_t)w;
      } else if (w >= 0 && (uint32_t)w > cur) {
        want = (uint32_t)w;
        if (tid == 0 && cur % c.page_tokens != 0) {
          const uint32_t e = table_entry(c, p >= 0 ? (uint32_t)p : r, cur / c.page_tokens);
          // without forks counts only fall meanwhile: a page held once is not shared
          if (e < c.num_pages && (parents || get_agent(c.refs + e) > 1u)) {
            atomicAdd(c.holders + e, 1u);
            atomicMax(c.last + e, r + 1);
            mark = e;
          }
        }
      }
    }
    if (tid == 0) {
      uint32_t* q = c.row + 4 * (uint64_t)r;
      put_agent(q, cur);
      put_agent(q + 1, want);
      put_agent(q + 2, mark);
      put_agent(granted + r, ok ? 1u : 0u);
    }
  }
  wait_stores();
  __syncthreads();
  if (tid == 0)
    s_last = __hip_atomic_fetch_add(c.ctl + CTL_ARRIVE, 1u, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;

  // Pages given up that nobody took up again are free; the rows' requests, read
  // once if the rows fit the threads.  Loads of several entries go together.
  const bool one = c.rows <= UT;
  uint32_t nfreed = get_agent(c.ctl + CTL_FREED);
  Request mine = no_request();
  if (one) {
    mine = read_request(c, umin(tid, c.rows - 1));
    if (tid >= c.rows) mine = no_request();
  }
  // The free pages of each word: in LDS up to FREE_LDS words, in memory beyond
  // (where the atomics on a line follow one another, and a row's pages may lie
  // together).
  const bool few = c.words <= FREE_LDS;
  auto memory_word = [&](uint32_t w) {
    return w < c.words ? page_bits(c, w) & ~get_agent(c.used + w) : 0u;
  };
  // (all that one round of loads can bring, then what depends on it; from places
  // inside the arrays, so that no load waits in a branch of its own)
  constexpr uint32_t WB = FREE_LDS / UT, FB = 6;
  uint32_t word[WB], e[FB], refs[FB];
#pragma unroll
  for (uint32_t k = 0; k < WB; ++k) word[k] = get_agent(c.used + umin(k * UT + tid, c.words - 1));
#pragma unroll
  for (uint32_t k = 0; k < FB; ++k) e[k] = get_agent(c.freed + umin(k * UT + tid, c.num_pages - 1));
  read_mark(c, mine);
#pragma unroll
  for (uint32_t k = 0; k < FB; ++k) refs[k] = get_agent(c.refs + umin(e[k], c.num_pages - 1));
  nfreed = umin(nfreed, c.num_pages);
  if (few)
#pragma unroll
    for (uint32_t k = 0; k < WB; ++k)
      if (k * UT + tid < c.words) s_word[k * UT + tid] = page_bits(c, k * UT + tid) & ~word[k];
  if (tid == 0) s_moves = s_taken = s_jobs = 0;
  lds_barrier();
  auto give_up = [&](uint32_t page) {
    const uint32_t w = page >> 5, bit = 1u << (page & 31u);
    if (few)
      __hip_atomic_fetch_or((LDS uint32_t*)s_word + w, bit, __ATOMIC_RELAXED,
                            __HIP_MEMORY_SCOPE_WORKGROUP);
    else
      __hip_atomic_fetch_and(c.used + w, ~bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
#pragma unroll
  for (uint32_t k = 0; k < FB; ++k)
    if (k * UT + tid < nfreed && e[k] < c.num_pages && refs[k] == 0) give_up(e[k]);
  for (uint32_t i = FB * UT + tid; i < nfreed; i += UT) {
    const uint32_t page = get_agent(c.freed + i);
    if (page < c.num_pages && get_agent(c.refs + page) == 0) give_up(page);
  }
  settle(c, tid, mine);
  if (nfreed && !few) wait_stores();
  lds_barrier();
  auto free_word = [&](uint32_t w) {
    return few ? (w < c.words ? s_word[w] : 0u) : memory_word(w);
  };
  uint32_t here = 0;
  for (uint32_t w = tid; w < c.words; w += UT) here += __popc(free_word(w));
  // How many pages all the rows ask for: no more free ones than that are listed.
  // (A row that asks for more than there are gets none, nor does one after it.)
  const uint32_t cap = c.num_pages + 1;
  uint64_t nfree = 0, asked = 0, mine_first = 0;
  if (one) {
    mine_first = update_scan_and_sum(umin(mine.need, cap), here, red, asked, nfree);
  } else {
    (void)update_scan(here, red, nfree);
    for (uint32_t r0 = 0; r0 < c.rows; r0 += UT) {
      uint64_t sum = 0;
      const uint32_t need = r0 + tid < c.rows ? request_of(c, r0 + tid).need : 0u;
      (void)update_scan(umin(need, cap), red, sum);
      asked += sum;
    }
  }
  const uint32_t listed = (uint32_t)(asked < nfree ? asked : nfree);
  const bool in_lds = listed <= FREE_LDS;
  // the listed pages, and the words without them, a round of words at a time
  uint32_t base = 0;
  for (uint32_t w0 = 0; w0 < c.words && base < listed; w0 += UT) {
    const uint32_t w = w0 + tid;
    uint32_t m = free_word(w);
    uint64_t sum = 0;
    uint32_t at = base + (uint32_t)update_scan(__popc(m), red, sum);
    base += (uint32_t)sum;
    if (m == 0 || at >= listed) continue;
    for (; m && at < listed; m &= m - 1, ++at) {
      const uint32_t page = 32 * w + (uint32_t)__builtin_ctz(m);
      if (in_lds)
        s_free[at] = page;
      else
        put_agent(c.list + at, page);
    }
    if (few)
      s_word[w] = m;
    else
      put_agent(c.used + w, page_bits(c, w) & ~m);
  }
  if (!in_lds || !few) wait_stores();
  lds_barrier();
  auto free_page = [&](uint32_t k) { return in_lds ? s_free[k] : get_agent(c.list + k); };

  uint64_t total = 0;  // pages asked for by the rows so far
  for (uint32_t r0 = 0; r0 < c.rows; r0 += UT) {
    const uint32_t r = r0 + tid;
    Request q = mine;
    if (!one) q = r < c.rows ? request_of(c, r) : no_request();
    uint64_t sum = 0, first = mine_first;
    if (!one) {
      if (tid == 0) s_jobs = 0;
      first = total + update_scan(umin(q.need, cap), red, sum);
    }
    bool grow = q.want != EMPTY;
    if (grow && first + q.need > nfree && (q.need || q.tied)) {
      put_agent(granted + r, 0u);
      atomicOr(status, LLMK_STATUS_PAGES_FULL);
      grow = false;
    }
    if (r < c.rows) G(c.lengths)[r] = grow ? q.want : q.cur;
    auto give = [&](uint32_t row, uint32_t j, uint32_t page) {
      put_agent(c.table + (uint64_t)row * c.max_pages + j, page);
      put_agent(c.refs + page, 1u);
    };
    if (grow && q.need) {
      const uint32_t j0 = pages_of(c, q.cur) - q.copy, f = (uint32_t)first;
      __hip_atomic_fetch_max((LDS uint32_t*)&s_taken, f + q.need, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_WORKGROUP);
      if (q.copy) {
        const uint32_t i = __hip_atomic_fetch_add((LDS uint32_t*)&s_moves, 1u, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_WORKGROUP);
        G(c.moves)[i] = u2v{q.mark, free_page(f)};
      }
      if (q.need <= 2) {  // as most rows of a decoding step: by its own thread
        give(r, j0, free_page(f));
        if (q.need == 2) give(r, j0 + 1, free_page(f + 1));
      } else {
        const uint32_t k = __hip_atomic_fetch_add((LDS uint32_t*)&s_jobs, 1u, __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_WORKGROUP);
        s_job[k][0] = r;
        s_job[k][1] = j0;
        s_job[k][2] = f;
        s_job[k][3] = q.need;
      }
    }
    lds_barrier();
    for (uint32_t k = wv; k < s_jobs; k += UW) {  // a wave per row
      const uint32_t row = s_job[k][0], j0 = s_job[k][1], f = s_job[k][2], n = s_job[k][3];
      for (uint32_t i = lane; i < n; i += WAVE) give(row, j0 + i, free_page(f + i));
    }
    total += sum;
    lds_barrier();  // the jobs are read
  }
  // listed pages that no row got are free again
  const uint32_t taken = s_taken;
  if (taken < listed) {
    for (uint32_t i = taken + tid; i < listed; i += UT) give_up(free_page(i));
    lds_barrier();
  }
  if (few && (taken || nfreed))
    for (uint32_t w = tid; w < c.words; w += UT) put_agent(c.used + w, page_bits(c, w) & ~s_word[w]);
  // the copied pages lose the rows that left them; what calls begin with
  __syncthreads();  // (the moves are written)
  for (uint32_t i = tid; i < s_moves; i += UT) atomicSub(c.refs + G(c.moves)[i][0], 1u);
  for (uint32_t r = tid; r < c.rows; r += UT) {
    const uint32_t e = one ? mine.mark : get_agent(c.row + 4 * (uint64_t)r + 2);
    if (e != EMPTY) {
      put_agent(c.holders + e, 0u);
      put_agent(c.last + e, 0u);
    }
  }
  if (tid == 0) {
    put_agent(c.ctl + CTL_MOVES, s_moves);
    put_agent(c.ctl + CTL_ARRIVE, 0u);
    put_agent(c.ctl + CTL_FREED, 0u);
  }
}

// ---- compaction --------------------------------------------------------------
// With M pages in use and U(p) of them below page p: a used page p at or above M
// is the (U(p) - U(M))-th that moves, a free page p below M the (p - U(p))-th
// hole, and there are M - U(M) of each.  Every workgroup counts U for itself
// from the whole bitmap (an eighth of a byte per page), so that one launch
// makes the list of pairs; a workgroup takes `slice` words, a page a thread.
constexpr uint32_t FT = 256;
__device__ __forceinline__ uint32_t count_used(const Cache& c, uint32_t upto, LDS uint32_t* red) {
  uint32_t n = 0;  // used pages below page upto
  for (uint32_t w = threadIdx.x; w < (upto + 31) / 32; w += FT) {
    const uint32_t u = used_bits(c, w), left = upto - 32 * w;
    n += __popc(left >= 32 ? u : u & ((1u << left) - 1u));
  }
  n = bcast63u(wave_incl_scan(n));
  __syncthreads();
  if ((threadIdx.x & 63u) == 0) red[threadIdx.x >> 6] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (uint32_t i = 0; i < FT / WAVE; ++i) n += red[i];
  return n;
}
__global__ __launch_bounds__(FT) void pages_plan_kernel(Cache c, uint32_t* map, uint32_t slice) {
  __shared__ uint32_t s_red[FT / WAVE];
  LDS uint32_t* red = (LDS uint32_t*)s_red;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
  const uint32_t p0 = blockIdx.x * slice * 32, p1 = umin(p0 + slice * 32, c.num_pages);
  const uint32_t M = count_used(c, c.num_pages, red), UM = count_used(c, M, red);
  uint32_t U = count_used(c, p0, red);
  GLB uint32_t* pair = (GLB uint32_t*)G(c.moves);
  for (uint32_t q0 = p0; q0 < p1; q0 += FT) {
    const uint32_t p = q0 + tid;
    const bool in = p < p1;
    const bool used = in && ((used_bits(c, p >> 5) >> (p & 31u)) & 1u);
    const uint64_t who = __ballot(used);
    __syncthreads();
    if (lane == 0) red[wv] = (uint32_t)__popcll(who);
    __syncthreads();
    uint32_t before = U + lanes_below(who), all = 0;
#pragma unroll
    for (uint32_t i = 0; i < FT / WAVE; ++i) {
      before += i < wv ? red[i] : 0u;
      all += red[i];
    }
    U += all;
    if (in && used && p >= M) {
      pair[2 * (before - UM)] = p;
      G(c.list)[p] = before - UM;
    } else if (in) {
      if (!used && p < M) pair[2 * (p - before) + 1] = p;
      G(map)[p] = p;
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    G(c.ctl)[CTL_MOVES] = M - UM;
    G(c.ctl)[CTL_LIVE] = M;
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
// workgroups `first` on: the number of pairs may be known on the device alone.
// Bound by HBM, read and written: 4000 pages of 32 KiB in 4 pools 215 us, 4.9
// TB/s, as a copy of as many bytes in one piece.
constexpr uint32_t CT = 256, CPIECE = CT * 16 * 4;
__device__ __forceinline__ void copy_items(const Copies& a, uint32_t first) {
  const uint32_t n = a.moves ? G(a.n_moves)[0] : a.n;
  const uint32_t pieces = (uint32_t)((a.page_bytes + CPIECE - 1) / CPIECE);  // <= 2^26
  const uint64_t per = (uint64_t)pieces * a.n_pools, items = n * per;
  for (uint64_t it = blockIdx.x - first; it < items; it += gridDim.x - first) {
    const uint64_t pair = it / per, rest = it - pair * per;
    const uint32_t pool = (uint32_t)(rest / pieces);
    const uint64_t at = (rest - (uint64_t)pool * pieces) * CPIECE;
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
__global__ __launch_bounds__(CT) void pages_copy_kernel(Copies a) { copy_items(a, 0); }

// A planned compaction: the first workgroups do the tables, then the counts,
// the map and the words of `used`, the others the contents; none of them reads
// what another one writes.
__global__ __launch_bounds__(CT) void pages_compact_kernel(Cache c, uint32_t* map, Copies a,
                                                           uint32_t row_wgs, uint32_t state_wgs) {
  const uint32_t n = G(c.ctl)[CTL_MOVES], M = G(c.ctl)[CTL_LIVE], t = threadIdx.x;
  if (blockIdx.x < row_wgs) {
    for (uint32_t r = blockIdx.x; r < c.rows; r += row_wgs) {
      uint32_t k = pages_of(c, G(c.lengths)[r]);
      if (k > c.max_pages) k = c.max_pages;
      uint32_t* row = c.table + (uint64_t)r * c.max_pages;
      for (uint32_t j = t; j < k; j += CT) {
        const uint32_t e = G(row)[j];
        if (e < M || e >= c.num_pages) continue;
        const uint32_t i = G(c.list)[e];  // (a page nobody holds has no rank)
        if (i < n) G(row)[j] = G(c.moves)[i][1];
      }
    }
  } else if (blockIdx.x < row_wgs + state_wgs) {
    const uint32_t step = state_wgs * CT, i0 = (blockIdx.x - row_wgs) * CT + t;
    for (uint32_t i = i0; i < n; i += step) {
      const u2v m = G(c.moves)[i];
      G(map)[m[0]] = m[1];
      G(c.refs)[m[1]] = G(c.refs)[m[0]];
      G(c.refs)[m[0]] = 0;
    }
    for (uint32_t w = i0; w < c.words; w += step)
      G(c.used)[w] = 32 * w + 32 <= M ? 0xffffffffu : (32 * w >= M ? 0u : (1u << (M - 32 * w)) - 1u);
  } else {
    copy_items(a, row_wgs + state_wgs);
  }
}

}  // namespace llmk

// ===========================================================================
using namespace llmk;

// The work array: the control words, the pairs to copy, then the arrays of Cache.
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
  *words = CTL_WORDS + 2 * most_moves(rows, num_pages) + 4ull * num_pages + 4ull * rows;
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
  c.ctl = k->work;
  c.moves = (u2v*)(k->work + CTL_WORDS);
  c.holders = k->work + CTL_WORDS + 2 * most_moves(k->rows, k->num_pages);
  c.last = c.holders + k->num_pages;
  c.list = c.last + k->num_pages;
  c.freed = c.list + k->num_pages;
  c.row = c.freed + k->num_pages;
  return LLMK_OK;
}

// Enough workgroups for 8 per CU; fewer if there are fewer pieces.
constexpr uint32_t COPY_GRID = 2048;
static uint64_t copy_grid(const Copies& a, uint64_t most_pairs) {
  const uint64_t per = (a.page_bytes + CPIECE - 1) / CPIECE * a.n_pools;
  return per && most_pairs > COPY_GRID / per ? COPY_GRID : most_pairs * per;
}
static int launch_copies(const Copies& a, uint64_t most_pairs, void* stream) {
  const uint64_t grid = copy_grid(a, most_pairs);
  if (grid == 0) return LLMK_OK;
  hipLaunchKernelGGL(pages_copy_kernel, dim3((uint32_t)grid), dim3(CT), 0, (hipStream_t)stream, a);
  HIPCHK(hipGetLastError());
  return LLMK_OK;
}
static Copies moves_of(llmk_sampler* s, const llmk_page_cache* k, const Cache& c) {
  Copies a{};
  a.n_pools = k->n_pools;
  a.page_bytes = k->page_bytes;
  a.pools = k->pools;
  a.num_pages = k->num_pages;
  a.moves = c.moves;
  a.n_moves = c.ctl + CTL_MOVES;
  a.status = s->ws.status;
  return a;
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
  hipLaunchKernelGGL(pages_update_kernel, dim3(c.rows), dim3(UT), 0, (hipStream_t)stream, c,
                     parents, new_lengths, out_granted, s->ws.status);
  HIPCHK(hipGetLastError());
  // only a row that grows copies a page
  if (!new_lengths || cache->n_pools == 0) return LLMK_OK;
  return launch_copies(moves_of(s, cache, c), c.rows, stream);
}

extern "C" int llmk_pages_compact(llmk_sampler* s, const llmk_page_cache* cache,
                                  uint32_t* out_map, void* stream) {
  Cache c;
  const int rc = check_cache(s, cache, c);
  if (rc != LLMK_OK) return rc;
  if (!out_map) return fail(LLMK_ERR_INVALID_ARGUMENT, "out_map is required");
  HIPCHK(hipSetDevice(s->device));
  // slices of 8 words (a page per thread and round) and more, for 64 workgroups
  // at most beyond a million pages: each of them reads the whole bitmap
  uint32_t slice = (c.words + 1023) / 1024;
  if (c.num_pages > (1u << 20)) slice = (c.words + 63) / 64;
  slice = slice < 8 ? 8 : (slice + 7) / 8 * 8;
  hipLaunchKernelGGL(pages_plan_kernel, dim3((c.words + slice - 1) / slice), dim3(FT), 0,
                     (hipStream_t)stream, c, out_map, slice);
  HIPCHK(hipGetLastError());
  const Copies a = moves_of(s, cache, c);
  const uint32_t row_wgs = c.rows < 1024 ? c.rows : 1024;
  const uint32_t state_wgs = c.words < 16 * CT ? (c.words + CT - 1) / CT : 16;
  const uint64_t copy_wgs = copy_grid(a, (uint64_t)c.num_pages / 2 + 1);
  hipLaunchKernelGGL(pages_compact_kernel, dim3(row_wgs + state_wgs + (uint32_t)copy_wgs), dim3(CT),
                     0, (hipStream_t)stream, c, out_map, a, row_wgs, state_wgs);
  HIPCHK(hipGetLastError());
  return LLMK_OK;
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
