// llmk_logits.hip — operators on a batch of logits rows around the sampling
// call (gfx950):
//
//   process_kernel   softcap, logit bias, penalties, allow-mask and
//                    temperature, from logits to logits
//   logprobs_kernel  log-probability and rank of one token per row, and the
//                    row's likeliest tokens
//
// Both are bound by HBM: every logit is read once, and the first writes each
// once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "llmk_device.h"
#include "llmk_host.h"

namespace llmk {

// 16 bytes of logits at the logits' own alignment: rows start anywhere, and
// gfx950's global memory instructions take unaligned addresses.
typedef uint32_t u4v_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4v_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4v_list __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Elem {
  static constexpr uint32_t SZ = (DT & 3) == LLMK_F32 ? 4 : 2;
  static constexpr uint32_t W = 16 / SZ;  // logits per 16 bytes
};

// The W logits from element e of a row of V, packed; elements past V read as
// zero bits.  e < V.
template <int DT>
__device__ __forceinline__ u4v load_pack(const void* row, uint32_t e, uint32_t V) {
  constexpr uint32_t W = Elem<DT>::W;
  if (e + W <= V) {
    if (Elem<DT>::SZ == 4)
      return (u4v)__builtin_nontemporal_load((const GLB u4v_a4*)G((const uint32_t*)row + e));
    return (u4v)__builtin_nontemporal_load((const GLB u4v_a2*)G((const uint16_t*)row + e));
  }
  u4v r = {0, 0, 0, 0};
#pragma unroll
  for (uint32_t q = 0; q < W; ++q) {
    if (e + q < V) {
      if (Elem<DT>::SZ == 4)
        r[q] = G((const uint32_t*)row)[e + q];
      else
        r[q / 2] |= (uint32_t)G((const uint16_t*)row)[e + q] << (16 * (q & 1));
    }
  }
  return r;
}
template <int DT>
__device__ __forceinline__ float unpack(const u4v& r, uint32_t q) {
  if (Elem<DT>::SZ == 4) return __uint_as_float(r[q]);
  return cvt16<DT>((r[q / 2] >> (16 * (q & 1))) & 0xffffu);
}
template <int OT>
__device__ __forceinline__ uint32_t pack16(float x) {  // rounded to nearest even
  if (OT == LLMK_BF16) return __float_as_uint(round_dt<LLMK_BF16>(x)) >> 16;
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x);
}
template <int OT>
__device__ __forceinline__ void store_one(void* row, uint32_t e, float x) {
  if (OT == LLMK_F32)
    G((float*)row)[e] = x;
  else
    G((uint16_t*)row)[e] = (uint16_t)pack16<OT>(x);
}

// ---------------------------------------------------------------------------
// process
// ---------------------------------------------------------------------------
struct PArgs {
  const void* in;
  void* out;
  uint64_t in_stride, out_stride;
  uint32_t B, V, nseg;
  const uint32_t* row_seq;
  uint32_t sequences;
  const float *T, *rp, *pp, *fp;
  const uint32_t *hoff, *htok, *hlen, *hcnt;
  const uint32_t *xbeg, *xcnt, *xtok;
  const uint32_t *boff, *btok;
  const float* bval;
  const uint32_t* mask;
  uint32_t mask_words, mask_rows;
  const int32_t* mask_index;
  float sc_m1, sc_cap;  // softcap: 1 / cap and cap
  uint32_t* status;
};

constexpr uint32_t PT = 256;  // threads of a workgroup

// Adds the list's tokens that fall in [lo, lo + n) to their counts.
__device__ __forceinline__ void count_tokens(LDS uint32_t* cnt, const uint32_t* tok,
                                             const uint32_t* times, uint32_t len, uint32_t lo,
                                             uint32_t n) {
  auto add = [&](uint32_t t, uint32_t k) {
    if (t - lo < n)
      __hip_atomic_fetch_add(cnt + (t - lo), k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  const uint32_t whole = len & ~3u;
  for (uint32_t j = 4 * threadIdx.x; j < whole; j += 4 * PT) {
    const u4v_list t = *(const GLB u4v_list*)G(tok + j);
    u4v_list k = {1, 1, 1, 1};
    if (times) k = *(const GLB u4v_list*)G(times + j);
#pragma unroll
    for (int q = 0; q < 4; ++q) add(t[q], times && k[q] == 0 ? 1u : k[q]);
  }
  const uint32_t j = whole + threadIdx.x;
  if (j < len) {
    const uint32_t k = times ? G(times)[j] : 1u;
    add(G(tok)[j], k ? k : 1u);
  }
}

// One workgroup per (row, segment of PT * W * CH logits).  A thread requests
// its logits first; while they travel, the workgroup counts the history's
// tokens of the segment in LDS, one word per logit (a segment is small enough
// for that, and it needs no table, no hash and no limit on a history), and
// then reads the counts back beside its logits: 4 bytes of LDS a logit, far
// below what LDS delivers in the time of the logit's HBM traffic.  The
// segments of a row re-read its history from L2, so they share an XCD.
//
// Biases are added in the same way through a word of LDS per logit.  A token
// listed more than once gets its biases summed in listing order: the first
// entry (an LDS minimum over the list's positions) sums all of them, so the
// result does not depend on the order in which threads run.
template <int DT, int OT, int CH>
__global__ __launch_bounds__(PT) void process_kernel(PArgs a) {
  extern __shared__ uint32_t psm[];
  constexpr uint32_t W = Elem<DT>::W, SEG = PT * W * CH;
  const uint32_t tid = threadIdx.x;
  uint32_t b, g;
  if ((a.B & 7u) == 0) {  // blocks go round the 8 XCDs: a row's segments on one
    const uint32_t k = blockIdx.x >> 3;
    b = (k / a.nseg) * 8 + (blockIdx.x & 7u);
    g = k % a.nseg;
  } else {
    b = blockIdx.x / a.nseg;
    g = blockIdx.x % a.nseg;
  }
  const uint32_t lo = g * SEG, n = umin(SEG, a.V - lo);
  const char* row = (const char*)a.in + (uint64_t)b * a.in_stride * Elem<DT>::SZ;
  char* orow = (char*)a.out + (uint64_t)b * a.out_stride * Elem<OT>::SZ;

  u4v r[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t e = lo + (c * PT + tid) * W;
    r[c] = u4v{0, 0, 0, 0};
    if (e < a.V) r[c] = load_pack<DT>(row, e, a.V);
  }

  const uint32_t q = a.row_seq ? G(a.row_seq)[b] : b;
  bool bad = a.row_seq && q >= a.sequences;
  const uint32_t qs = bad ? 0u : q;
  int32_t mi = -1;
  if (a.mask) {
    mi = a.mask_index ? G(a.mask_index)[b] : (int32_t)b;
    if (mi >= 0 && (uint32_t)mi >= a.mask_rows) bad = true;
  }
  RowP P;
  P.T = *G(row_or(a.T, qs, &kOneF));
  P.rp = *G(row_or(a.rp, qs, &kOneF));
  P.pp = *G((const float*)row_or(a.pp, qs, &kZeroU));
  P.fp = *G((const float*)row_or(a.fp, qs, &kZeroU));
  if (!finitef(P.T) || !finitef(P.rp) || !finitef(P.pp) || !finitef(P.fp)) bad = true;
  if (bad) {  // the whole workgroup agrees
    for (uint32_t e = lo + tid; e < lo + n; e += PT) store_one<OT>(orow, e, __builtin_nanf(""));
    if (g == 0 && tid == 0) atomicOr(a.status, LLMK_STATUS_INVALID_PARAMS);
    return;
  }
  const uint32_t* mrow =
      a.mask && mi >= 0 ? a.mask + (uint64_t)(uint32_t)mi * a.mask_words : nullptr;
  uint32_t mw[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t e = lo + (c * PT + tid) * W;
    mw[c] = 0xffffffffu;
    if (mrow && e < a.V) mw[c] = G(mrow)[e >> 5] >> (e & 31u);  // W divides 32
  }

  LDS uint32_t* cnt = (LDS uint32_t*)psm;
  LDS float* bsum = (LDS float*)psm + SEG;  // present if a.boff
  bool bias = false;
  if (a.boff) {
    const uint32_t j0 = G(a.boff)[qs], j1 = G(a.boff)[qs + 1];
    const uint32_t nb = j1 > j0 ? j1 - j0 : 0u;
    bias = nb > 0;
    if (bias) {
      const uint32_t* bt = a.btok + j0;
      for (uint32_t i = tid; i < SEG; i += PT) {
        cnt[i] = EMPTY;
        bsum[i] = 0.0f;
      }
      __syncthreads();
      for (uint32_t j = tid; j < nb; j += PT) {
        const uint32_t t = G(bt)[j] - lo;
        if (t < n)
          __hip_atomic_fetch_min(cnt + t, j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      __syncthreads();
      for (uint32_t j = tid; j < nb; j += PT) {  // later entries mark the first one's word
        const uint32_t t = G(bt)[j] - lo;
        if (t < n && (cnt[t] & 0x7fffffffu) != j)
          __hip_atomic_fetch_or(cnt + t, 0x80000000u, __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      __syncthreads();
      for (uint32_t j = tid; j < nb; j += PT) {
        const uint32_t tok = G(bt)[j], t = tok - lo;
        if (t < n) {
          const uint32_t w = cnt[t];
          if ((w & 0x7fffffffu) == j) {
            float v = G(a.bval)[j0 + j];
            if (w >> 31)
              for (uint32_t k = j + 1; k < nb; ++k)
                if (G(bt)[k] == tok) v += G(a.bval)[j0 + k];
            bsum[t] = v;
          }
        }
      }
      __syncthreads();
    }
  }
  const bool pen = P.rp != 1.0f || P.pp != 0.0f || P.fp != 0.0f;
  bool have = false;
  if (pen && (a.hoff || a.xbeg)) {
    const uint32_t h0 = a.hoff ? G(a.hoff)[qs] : 0u;
    const uint32_t h1 = a.hoff ? (a.hlen ? h0 + G(a.hlen)[qs] : G(a.hoff)[qs + 1]) : 0u;
    const uint32_t hn = h1 > h0 ? h1 - h0 : 0u, xn = a.xbeg ? G(a.xcnt)[b] : 0u;
    have = hn > 0 || xn > 0;
    if (have) {
      for (uint32_t i = tid; i < SEG / 4; i += PT) *(LDS u4v*)(cnt + 4 * i) = u4v{0, 0, 0, 0};
      __syncthreads();
      if (hn) count_tokens(cnt, a.htok + h0, a.hcnt ? a.hcnt + h0 : nullptr, hn, lo, n);
      if (xn) count_tokens(cnt, a.xtok + G(a.xbeg)[b], nullptr, xn, lo, n);
      __syncthreads();
    }
  }
  const bool divide = P.T != 1.0f && P.T > 1e-5f;

#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t at = (c * PT + tid) * W, e = lo + at;
    if (e >= a.V) break;
    float x[W];
#pragma unroll
    for (uint32_t k = 0; k < W; ++k) {
      x[k] = unpack<DT>(r[c], k);
      if (DT & SOFTCAP) x[k] = tanh_ref(x[k] * a.sc_m1) * a.sc_cap;
    }
    if (bias) {
#pragma unroll
      for (uint32_t k = 0; k < W; ++k) {
        const float v = bsum[at + k];
        if (v != 0.0f) x[k] += v;  // (a logit of -0 without a bias stays -0)
      }
    }
    if (have) {
#pragma unroll
      for (uint32_t h = 0; h < W; h += 4) {
        const u4v m = *(LDS u4v*)(cnt + at + h);
        if (m[0] | m[1] | m[2] | m[3]) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (m[k]) x[h + k] = penalize(x[h + k], P, m[k]);
        }
      }
    }
#pragma unroll
    for (uint32_t k = 0; k < W; ++k) {
      if (!((mw[c] >> k) & 1u)) x[k] = NEG_INF;
      if (divide) x[k] = x[k] / P.T;
    }
    if (e + W <= a.V) {
      if (OT == LLMK_F32) {
#pragma unroll
        for (uint32_t h = 0; h < W; h += 4) {
          const u4v o = {__float_as_uint(x[h]), __float_as_uint(x[h + 1]),
                         __float_as_uint(x[h + 2]), __float_as_uint(x[h + 3])};
          *(GLB u4v_a4*)G((uint32_t*)orow + e + h) = (u4v_a4)o;
        }
      } else {
        u4v o;
#pragma unroll
        for (uint32_t k = 0; k < W / 2; ++k)
          o[k] = pack16<OT>(x[2 * k]) | (pack16<OT>(x[2 * k + 1]) << 16);
        *(GLB u4v_a2*)G((uint16_t*)orow + e) = (u4v_a2)o;
      }
    } else {
#pragma unroll
      for (uint32_t k = 0; k < W; ++k)
        if (e + k < a.V) store_one<OT>(orow, e + k, x[k]);
    }
  }
}

// ---------------------------------------------------------------------------
// logprobs
// ---------------------------------------------------------------------------
struct LArgs {
  const void* logits;
  uint64_t stride;
  uint32_t B, V, G, tps, ntiles;  // G segments of tps tiles per row
  float sc_m1, sc_cap;
  const uint32_t* tokens;
  float* out_lp;
  uint32_t* out_rank;
  uint32_t top_n;
  uint32_t* out_ids;
  float* out_top;
  uint32_t* arrive;  // [B]
  f2v* part;         // [B][G]: max, sum
  u2v* cand;         // [B * G][CAND_CAP]: (rank count, -), then the segment's top list
};

constexpr uint32_t LT = 256, LWAVES = LT / WAVE;
constexpr uint32_t TOP_MAX = 32;   // largest top_n
constexpr uint32_t TLIST = 256;    // candidates of a wave
constexpr uint32_t TMERGE = 512;   // candidates of a row's segments: G * top_n

// A token's place in the order (logit descending, index ascending) as a
// number that falls along it; no token has 0.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t e) {
  return ((uint64_t)fkey(x + 0.0f) << 32) | (uint32_t)~e;  // -0 is 0
}
__device__ __forceinline__ float key_value(uint64_t k) { return funkey((uint32_t)(k >> 32)); }

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// list[0 .. m) to its n first in order, sorted, by one wave; returns how many
// there are.  Each lane counts the entries before its own ones.  m <= 64 * Q.
template <int Q>
__device__ __forceinline__ uint32_t keep_first(LDS uint64_t* list, uint32_t m, uint32_t n) {
  const uint32_t lane = threadIdx.x & 63u;
  uint64_t k[Q];
  uint32_t before[Q];
  wave_sync();
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const uint32_t at = i * 64 + lane;
    k[i] = at < m ? list[at] : 0u;
    before[i] = 0;
  }
  for (uint32_t j = 0; j < m; ++j) {
    const uint64_t x = list[j];
#pragma unroll
    for (int i = 0; i < Q; ++i) before[i] += x > k[i] ? 1u : 0u;
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < Q; ++i)
    if (k[i] && before[i] < n) list[before[i]] = k[i];
  wave_sync();
  return umin(m, n);
}

// The n-th largest of the lanes' order-preserving keys (n <= 64), by bits.
template <int Q>
__device__ __forceinline__ uint32_t nth_key(const uint32_t (&key)[Q], uint32_t n) {
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < Q; ++i) m += (uint32_t)__popcll(__ballot(key[i] >= c));
    if (m >= n) t = c;
  }
  return t;
}

constexpr float kLog2e = 0x1.715476p+0f;
__device__ __forceinline__ float exp_diff(float x, float m) {  // e^(x - m), x <= m
  return __builtin_amdgcn_exp2f((x - m) * kLog2e);
}

// One workgroup per (row, segment): four waves, each with every fourth
// 1024-logit tile of the segment.  A lane keeps the running maximum m and sum
// s = sum e^(x - m) of its logits; the wave keeps its first top_n tokens in
// order in LDS: a tile whose maximum does not pass the last of them is done
// with, and only tiles that hold a new one look at single logits.  The first
// tile starts from the top_n-th largest of the lanes' maxima, below which no
// logit of the tile can belong to the list.
template <int DT, bool TOP>
__global__ __launch_bounds__(LT) void logprobs_kernel(LArgs a) {
  __shared__ uint64_t s_list[LWAVES * TLIST];
  __shared__ float s_m[LWAVES], s_s[LWAVES];
  __shared__ uint32_t s_c[LWAVES], s_n[LWAVES], s_last;
  constexpr uint32_t W = Elem<DT>::W, NP = 16 / W;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
  const uint32_t b = blockIdx.x / a.G, g = blockIdx.x % a.G;
  const void* row = (const char*)a.logits + (uint64_t)b * a.stride * Elem<DT>::SZ;
  const uint32_t t0 = g * a.tps, t1 = umin(t0 + a.tps, a.ntiles);
  LDS uint64_t* list = (LDS uint64_t*)s_list + wv * TLIST;

  u4v raw[NP];
  auto request = [&](uint32_t t) {
#pragma unroll
    for (uint32_t j = 0; j < NP; ++j) {
      const uint32_t e = t * TILE + (j * 64 + lane) * W;
      raw[j] = u4v{0, 0, 0, 0};
      if (e < a.V) raw[j] = load_pack<DT>(row, e, a.V);
    }
  };
  uint32_t t = t0 + wv;
  if (t < t1) request(t);
  const uint32_t tok = a.tokens ? G(a.tokens)[b] : EMPTY;
  const bool chosen = tok < a.V;
  auto raw_logit = [&](uint32_t e) {
    const float x = Elem<DT>::SZ == 4 ? G((const float*)row)[e]
                                      : cvt16<DT>(G((const uint16_t*)row)[e]);
    return x == x ? x : NEG_INF;
  };
  const float lt = chosen ? raw_logit(tok) : __builtin_huge_valf();

  float m = NEG_INF, s = 0.0f;
  uint32_t before = 0, held = 0;
  float bar = NEG_INF;  // the value the list's last token has, once it is full
  bool full = false;
  for (; t < t1; t += LWAVES) {
    float x[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      x[i] = unpack<DT>(raw[i / W], i % W);
      if (!(x[i] == x[i])) x[i] = NEG_INF;
    }
    const uint32_t base = t * TILE;
    auto index = [&](uint32_t i) { return base + ((i / W) * 64 + lane) * W + i % W; };
    if (base + TILE > a.V) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (index(i) >= a.V) x[i] = NEG_INF;
    }
    if (t + LWAVES < t1) request(t + LWAVES);
    float mx = x[0];
#pragma unroll
    for (uint32_t i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    // tokens before the chosen one
    if (chosen) {
      if (base + TILE <= tok) {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) before += x[i] >= lt ? 1u : 0u;
      } else if (base > tok) {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) before += x[i] > lt ? 1u : 0u;
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i)
          before += x[i] > lt || (x[i] == lt && index(i) < tok) ? 1u : 0u;
      }
    }
    if (TOP) {
      if (!full || __any(mx > bar)) {
        float least = bar;
        if (!full) {
          const uint32_t k[1] = {fkey(mx + 0.0f)};
          least = funkey(nth_key<1>(k, a.top_n));
        }
        // Entries equal to the bar are taken along: within the tile an equal
        // one may come earlier in the order.
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
          const bool take = x[i] >= least && index(i) < a.V;
          const uint64_t who = __ballot(take);
          if (who) {
            if (take) list[held + lanes_below(who)] = order_key(x[i], index(i));
            held += (uint32_t)__popcll(who);
            if (held > TLIST - 64) {
              held = keep_first<TLIST / 64>(list, held, a.top_n);
              if (held == a.top_n) least = key_value(list[a.top_n - 1]);
            }
          }
        }
        if (!full || held > a.top_n + 16) {
          held = keep_first<TLIST / 64>(list, held, a.top_n);
          full = held == a.top_n;
          if (full) bar = key_value(list[a.top_n - 1]);
        }
      }
    }
    if (DT & SOFTCAP) {
      // tanh z = 1 - 2 / (1 + e^2z)
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const float z2 = __builtin_amdgcn_exp2f(x[i] * (2.0f * kLog2e) * a.sc_m1);
        const float y = a.sc_cap - 2.0f * a.sc_cap * __builtin_amdgcn_rcpf(1.0f + z2);
        x[i] = x[i] == NEG_INF ? NEG_INF : y;  // (a masked token stays one)
      }
      mx = x[0];
#pragma unroll
      for (uint32_t i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    }
    if (mx > m) {
      s *= exp_diff(m, mx);  // (0 the first time)
      m = mx;
    }
    const float mm = m == NEG_INF ? 0.0f : m;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) s += exp_diff(x[i], mm);
  }
  // the wave's, then the workgroup's share
  const float wm = wave_max(m);
  s = wave_tree_sum(m == NEG_INF ? 0.0f : s * exp_diff(m, wm));
  before = bcast63u(wave_incl_scan(before));
  if (TOP) held = keep_first<TLIST / 64>(list, held, a.top_n);
  if (lane == 0) {
    s_m[wv] = wm;
    s_s[wv] = s;
    s_c[wv] = before;
    s_n[wv] = held;
  }
  __syncthreads();
  if (wv != 0 && a.G == 1) return;
  float M = NEG_INF, S = 0.0f;
  uint32_t C = 0, N = 0;
  LDS uint64_t* all = (LDS uint64_t*)s_list;
  if (wv == 0) {
#pragma unroll
    for (uint32_t i = 0; i < LWAVES; ++i) {
      M = fmaxf(M, s_m[i]);
      C += s_c[i];
    }
#pragma unroll
    for (uint32_t i = 0; i < LWAVES; ++i)
      if (s_m[i] != NEG_INF) S += s_s[i] * exp_diff(s_m[i], M);
    if (TOP) {
      // the waves' lists end to end (each moves down, none past its own start)
      N = s_n[0];
      for (uint32_t i = 1; i < LWAVES; ++i) {
        const uint32_t ni = s_n[i];
        const uint64_t k = lane < ni ? all[i * TLIST + lane] : 0u;
        wave_sync();
        if (lane < ni) all[N + lane] = k;
        N += ni;
      }
      N = keep_first<LWAVES * TOP_MAX / 64>(all, N, a.top_n);
    }
  }
  if (a.G > 1) {
    // publish; the row's last workgroup joins the segments
    u2v* mine = a.cand + (uint64_t)blockIdx.x * CAND_CAP;
    if (wv == 0) {
      if (lane == 0) {
        G(a.part)[(uint64_t)b * a.G + g] = f2v{M, S};
        G(mine)[0] = u2v{C, N};
      }
      if (TOP && lane < N) {
        const uint64_t k = all[lane];
        G(mine)[1 + lane] = u2v{(uint32_t)k, (uint32_t)(k >> 32)};
      }
      wait_stores();
    }
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      const uint32_t seen = atomicAdd(a.arrive + b, 1u);
      s_last = seen == a.G - 1;
      if (s_last) {
        __threadfence();
        G(a.arrive)[b] = 0;  // for the next call
      }
    }
    __syncthreads();
    if (!s_last || wv != 0) return;
    const u2v* first = a.cand + (uint64_t)b * a.G * CAND_CAP;
    float m1 = NEG_INF, s1 = 0.0f;
    uint32_t c1 = 0, n1 = 0;
    if (lane < a.G) {
      const f2v ms = G(a.part)[(uint64_t)b * a.G + lane];
      const u2v cn = G(first)[(uint64_t)lane * CAND_CAP];
      m1 = ms[0];
      s1 = ms[1];
      c1 = cn[0];
      n1 = cn[1];
    }
    M = wave_max(m1);
    S = wave_tree_sum(m1 == NEG_INF ? 0.0f : s1 * exp_diff(m1, M));
    C = bcast63u(wave_incl_scan(c1));
    if (TOP) {
      // of the segments' lists, the entries not below the top_n-th largest
      // value; entry i of the G * top_n belongs to segment i / top_n
      constexpr int Q = TMERGE / 64;
      uint32_t hi[Q], lo[Q];
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        const uint32_t at = i * 64 + lane, sg = at / a.top_n;
        hi[i] = lo[i] = 0;
        if (sg < a.G) {
          const u2v k = G(first)[(uint64_t)sg * CAND_CAP + 1 + at % a.top_n];
          const uint32_t ns = G(first)[(uint64_t)sg * CAND_CAP][1];
          if (at % a.top_n < ns) {
            lo[i] = k[0];
            hi[i] = k[1];
          }
        }
      }
      const uint32_t least = nth_key<Q>(hi, a.top_n);
      N = 0;
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        const bool take = hi[i] >= least && hi[i] != 0;
        const uint64_t who = __ballot(take);
        if (take) all[N + lanes_below(who)] = ((uint64_t)hi[i] << 32) | lo[i];
        N += (uint32_t)__popcll(who);
      }
      N = keep_first<Q>(all, N, a.top_n);
    }
  }
  // log p(x) = (x - M) - log S; a raw logit of -inf has none
  const float logS = __logf(S);
  auto logp = [&](float raw_x) {
    if (raw_x == NEG_INF) return NEG_INF;
    const float y = DT & SOFTCAP ? tanh_ref(raw_x * a.sc_m1) * a.sc_cap : raw_x;
    return (y - M) - logS;
  };
  if (lane == 0 && a.tokens) {
    G(a.out_lp)[b] = chosen ? logp(lt) : __builtin_nanf("");
    if (a.out_rank) G(a.out_rank)[b] = chosen ? C : EMPTY;
  }
  if (TOP && lane < a.top_n) {
    const uint64_t k = lane < N ? all[lane] : 0u;
    G(a.out_ids)[(uint64_t)b * a.top_n + lane] = k ? ~(uint32_t)k : EMPTY;
    G(a.out_top)[(uint64_t)b * a.top_n + lane] = k ? logp(key_value(k)) : NEG_INF;
  }
}

}  // namespace llmk

// ===========================================================================
using namespace llmk;

static bool known_dtype(int32_t dt) {
  return dt == LLMK_F32 || dt == LLMK_BF16 || dt == LLMK_F16;
}

// Checks what both operators ask of their rows of logits.
static int check_rows(const void* p, int32_t dtype, uint32_t vocab, uint64_t stride,
                      const char* what) {
  if (!known_dtype(dtype))
    return fail(LLMK_ERR_INVALID_ARGUMENT,
                std::string(what) + ": dtype must be LLMK_F32, LLMK_BF16 or LLMK_F16");
  if (stride < vocab) return fail(LLMK_ERR_INVALID_ARGUMENT, std::string(what) + ": stride < vocab");
  if (((uintptr_t)p % (dtype == LLMK_F32 ? 4 : 2)) != 0)
    return fail(LLMK_ERR_ALIGNMENT, std::string(what) + " must be aligned to their elements");
  return LLMK_OK;
}
static int check_softcap(float c) {
  if (!(c >= 0.0f) || !(c < __builtin_huge_valf()))
    return fail(LLMK_ERR_INVALID_ARGUMENT, "softcap must be finite and >= 0 (0 = off)");
  return LLMK_OK;
}

// Whether the rows written may be written while the rows read are read: apart
// from each other, or row for row the same ones.
static bool rows_apart(const llmk_process_logits_args* a) {
  const uint64_t si = a->dtype == LLMK_F32 ? 4 : 2, so = a->out_dtype == LLMK_F32 ? 4 : 2;
  const uint64_t pi = a->row_stride * si, po = a->out_stride * so;  // bytes from row to row
  const uint64_t wi = a->vocab * si, wo = a->vocab * so;
  const uintptr_t i0 = (uintptr_t)a->logits, o0 = (uintptr_t)a->out;
  const uintptr_t i1 = i0 + (a->batch - 1) * pi + wi, o1 = o0 + (a->batch - 1) * po + wo;
  if (i1 <= o0 || o1 <= i0) return true;
  if (i0 == o0 && a->dtype == a->out_dtype && (pi == po || a->batch == 1)) return true;
  if (pi != po) return false;
  // interleaved rows of one pitch: each row of one lies between two of the other
  const uint64_t d = o0 >= i0 ? (o0 - i0) % pi : (pi - (i0 - o0) % pi) % pi;
  return d >= wi && d + wo <= pi;
}

extern "C" int llmk_process_logits(llmk_sampler* s, const llmk_process_logits_args* in,
                                   void* stream) {
  if (!s) return fail(LLMK_ERR_INVALID_ARGUMENT, "sampler is NULL");
  if (!in) return fail(LLMK_ERR_INVALID_ARGUMENT, "args is NULL");
  if (in->vocab == 0) return fail(LLMK_ERR_EMPTY_LOGITS, "Empty logits passed to process_logits");
  if (!in->logits || !in->out)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "logits and out are required");
  int rc = check_rows(in->logits, in->dtype, in->vocab, in->row_stride, "logits");
  if (rc == LLMK_OK) rc = check_rows(in->out, in->out_dtype, in->vocab, in->out_stride, "out");
  if (rc == LLMK_OK) rc = check_softcap(in->softcap);
  if (rc != LLMK_OK) return rc;
  if (in->out_dtype != LLMK_F32 && in->out_dtype != in->dtype)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "out_dtype must be LLMK_F32 or the logits' dtype");
  if (in->vocab > 0x7fffffffu) return fail(LLMK_ERR_CAPACITY, "vocab above 2^31 - 1");
  if ((in->hist_offsets == nullptr) != (in->hist_tokens == nullptr))
    return fail(LLMK_ERR_INVALID_ARGUMENT, "hist_offsets and hist_tokens go together");
  if ((in->hist_lengths || in->hist_counts) && !in->hist_offsets)
    return fail(LLMK_ERR_INVALID_ARGUMENT,
                "hist_lengths and hist_counts need hist_offsets and hist_tokens");
  if (!in->extra_begin != !in->extra_count || !in->extra_begin != !in->extra_tokens)
    return fail(LLMK_ERR_INVALID_ARGUMENT,
                "extra_begin, extra_count and extra_tokens go together");
  if (!in->bias_offsets != !in->bias_tokens || !in->bias_offsets != !in->bias_values)
    return fail(LLMK_ERR_INVALID_ARGUMENT,
                "bias_offsets, bias_tokens and bias_values go together");
  if (in->allow_mask && in->mask_words_per_row < (in->vocab + 31) / 32)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "mask_words_per_row < ceil(vocab/32)");
  if (in->mask_index && !in->allow_mask)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "mask_index needs allow_mask");
  if (in->allow_mask && !in->mask_index && in->mask_rows < in->batch)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "without mask_index allow_mask needs a row per row");
  if (in->row_seq && in->sequences == 0)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "row_seq needs sequences > 0");
  if (in->batch == 0) return LLMK_OK;
  if (!rows_apart(in))
    return fail(LLMK_ERR_INVALID_ARGUMENT,
                "out overlaps logits: in place needs the same address, dtype and stride");
  // Segments of 8192 logits where that makes two workgroups per CU or more,
  // of 2048 where it does not.
  const uint32_t big = 8192, small = 2048;
  const bool large = (uint64_t)in->batch * ((in->vocab + big - 1) / big) >= 512;
  const uint32_t seg = large ? big : small;
  const uint32_t nseg = (in->vocab + seg - 1) / seg;
  const uint64_t blocks = (uint64_t)in->batch * nseg;
  if (blocks > 0x7fffffffu) return fail(LLMK_ERR_CAPACITY, "batch * vocab too large for one call");
  HIPCHK(hipSetDevice(s->device));
  PArgs a;
  a.in = in->logits;
  a.out = in->out;
  a.in_stride = in->row_stride;
  a.out_stride = in->out_stride;
  a.B = in->batch;
  a.V = in->vocab;
  a.nseg = nseg;
  a.row_seq = in->row_seq;
  a.sequences = in->sequences;
  a.T = in->temperature;
  a.rp = in->repetition_penalty;
  a.pp = in->presence_penalty;
  a.fp = in->frequency_penalty;
  a.hoff = in->hist_offsets;
  a.htok = in->hist_tokens;
  a.hlen = in->hist_lengths;
  a.hcnt = in->hist_counts;
  a.xbeg = in->extra_begin;
  a.xcnt = in->extra_count;
  a.xtok = in->extra_tokens;
  a.boff = in->bias_offsets;
  a.btok = in->bias_tokens;
  a.bval = in->bias_values;
  a.mask = in->allow_mask;
  a.mask_words = in->mask_words_per_row;
  a.mask_rows = in->mask_rows;
  a.mask_index = in->mask_index;
  a.sc_m1 = in->softcap > 0.0f ? (float)(1.0 / (double)in->softcap) : 0.0f;
  a.sc_cap = in->softcap;
  a.status = s->ws.status;
  const bool sc = in->softcap > 0.0f;
  const bool counts = in->hist_offsets || in->extra_begin;
  const size_t lds = in->bias_offsets ? 8 * (size_t)seg : (counts ? 4 * (size_t)seg : 0);
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((uint32_t)blocks), dim3(PT), lds, (hipStream_t)stream, a);
  };
#define LLMK_PROCESS(DT, OT)                                                   \
  do {                                                                         \
    constexpr int C = (DT) == LLMK_F32 ? 8 : 4;                                \
    if (sc && large) launch(process_kernel<(DT) | SOFTCAP, OT, C>);            \
    else if (sc) launch(process_kernel<(DT) | SOFTCAP, OT, C / 4>);            \
    else if (large) launch(process_kernel<DT, OT, C>);                         \
    else launch(process_kernel<DT, OT, C / 4>);                                \
  } while (0)
  if (in->dtype == LLMK_F32) LLMK_PROCESS(LLMK_F32, LLMK_F32);
  else if (in->dtype == LLMK_BF16 && in->out_dtype == LLMK_F32) LLMK_PROCESS(LLMK_BF16, LLMK_F32);
  else if (in->dtype == LLMK_BF16) LLMK_PROCESS(LLMK_BF16, LLMK_BF16);
  else if (in->out_dtype == LLMK_F32) LLMK_PROCESS(LLMK_F16, LLMK_F32);
  else LLMK_PROCESS(LLMK_F16, LLMK_F16);
#undef LLMK_PROCESS
  HIPCHK(hipGetLastError());
  return LLMK_OK;
}

extern "C" int llmk_logprobs(llmk_sampler* s, const llmk_logprobs_args* in, void* stream) {
  if (!s) return fail(LLMK_ERR_INVALID_ARGUMENT, "sampler is NULL");
  if (!in) return fail(LLMK_ERR_INVALID_ARGUMENT, "args is NULL");
  if (in->vocab == 0) return fail(LLMK_ERR_EMPTY_LOGITS, "Empty logits passed to logprobs");
  if (!in->logits) return fail(LLMK_ERR_INVALID_ARGUMENT, "logits are required");
  int rc = check_rows(in->logits, in->dtype, in->vocab, in->row_stride, "logits");
  if (rc == LLMK_OK) rc = check_softcap(in->softcap);
  if (rc != LLMK_OK) return rc;
  if (!in->tokens && in->top_n == 0)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "neither tokens nor top_n: nothing is asked for");
  if (in->tokens && !in->out_logprobs)
    return fail(LLMK_ERR_INVALID_ARGUMENT, "tokens need out_logprobs");
  if (in->top_n > TOP_MAX) return fail(LLMK_ERR_CAPACITY, "top_n above 32");
  if (in->top_n && (!in->out_top_ids || !in->out_top_logprobs))
    return fail(LLMK_ERR_INVALID_ARGUMENT, "top_n needs out_top_ids and out_top_logprobs");
  if (in->vocab > MAX_TILES * TILE) return fail(LLMK_ERR_CAPACITY, "vocab above 2^20");
  if (in->batch == 0) return LLMK_OK;
  HIPCHK(hipSetDevice(s->device));
  LArgs a;
  a.logits = in->logits;
  a.stride = in->row_stride;
  a.B = in->batch;
  a.V = in->vocab;
  a.sc_m1 = in->softcap > 0.0f ? (float)(1.0 / (double)in->softcap) : 0.0f;
  a.sc_cap = in->softcap;
  a.tokens = in->tokens;
  a.out_lp = in->out_logprobs;
  a.out_rank = in->out_ranks;
  a.top_n = in->top_n;
  a.out_ids = in->out_top_ids;
  a.out_top = in->out_top_logprobs;
  a.arrive = s->ws.row_arrive;
  a.part = s->ws.tile_part;
  a.cand = s->ws.cand;
  a.ntiles = (a.V + TILE - 1) / TILE;
  // Segments per row: 1024 workgroups, four a CU, while each wave has a tile;
  // the segments' lists fit the last workgroup's (TMERGE) and the workspace.
  const uint32_t pool = s->max_batch > MAX_WGS ? s->max_batch : MAX_WGS;
  uint32_t g = (1024 + a.B - 1) / a.B;
  const uint32_t most = (a.ntiles + LWAVES - 1) / LWAVES;
  if (g > most) g = most;
  if (g > MAX_SEG) g = MAX_SEG;
  if (a.top_n && g > TMERGE / a.top_n) g = TMERGE / a.top_n;
  if (a.B > s->max_batch || (uint64_t)a.B * g > pool) g = 1;
  a.tps = (a.ntiles + g - 1) / g;
  a.G = (a.ntiles + a.tps - 1) / a.tps;
  const uint64_t blocks = (uint64_t)a.B * a.G;
  if (blocks > 0x7fffffffu) return fail(LLMK_ERR_CAPACITY, "batch above 2^31 - 1");
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((uint32_t)blocks), dim3(LT), 0, (hipStream_t)stream, a);
  };
#define LLMK_LOGPROBS(DT)                                     \
  do {                                                        \
    if (in->top_n) launch(logprobs_kernel<DT, true>);         \
    else launch(logprobs_kernel<DT, false>);                  \
  } while (0)
  const bool sc = in->softcap > 0.0f;
  if (in->dtype == LLMK_F32) {
    if (sc) LLMK_LOGPROBS(LLMK_F32 | SOFTCAP);
    else LLMK_LOGPROBS(LLMK_F32);
  } else if (in->dtype == LLMK_BF16) {
    if (sc) LLMK_LOGPROBS(LLMK_BF16 | SOFTCAP);
    else LLMK_LOGPROBS(LLMK_BF16);
  } else {
    if (sc) LLMK_LOGPROBS(LLMK_F16 | SOFTCAP);
    else LLMK_LOGPROBS(LLMK_F16);
  }
#undef LLMK_LOGPROBS
  HIPCHK(hipGetLastError());
  return LLMK_OK;
}
