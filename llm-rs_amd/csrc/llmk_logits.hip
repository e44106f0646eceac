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
#include <type_traits>

#include "llmk_device.h"
#include "llmk_host.h"
#include "llmk_sync.h"

namespace llmk {

// 16 bytes of logits at the logits' own alignment: rows start anywhere, and
// gfx950's global memory instructions take unaligned addresses.
typedef uint32_t u4v_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4v_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2v_a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u4v_list __attribute__((ext_vector_type(4), aligned(4)));

template <int DT>
struct Elem {
  static constexpr uint32_t SZ = (DT & 3) == LLMK_F32 ? 4 : 2;
  static constexpr uint32_t W = 16 / SZ;  // logits per 16 bytes
};

// The W logits from element e of a row of V, packed (W = 4 of 16 bits: the
// first two words); elements past V read as zero bits.  e < V.
template <int DT, uint32_t W = Elem<DT>::W>
__device__ __forceinline__ u4v load_pack(const void* row, uint32_t e, uint32_t V) {
  if (e + W <= V) {
    if (Elem<DT>::SZ == 4)
      return (u4v)__builtin_nontemporal_load((const GLB u4v_a4*)G((const uint32_t*)row + e));
    if (W == 4) {
      const u2v p = (u2v)__builtin_nontemporal_load((const GLB u2v_a2*)G((const uint16_t*)row + e));
      return u4v{p[0], p[1], 0, 0};
    }
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

// tanh within 4 units of 2^-24 of the result.  Below 1: z + z^3 q(z^2), q the
// interpolation of (tanh z / z - 1) / z^2 at the Chebyshev nodes of z^2 in
// [0, 1] (off by 1.4 units with the rounding of its steps).  From 1 on:
// 1 - 2 / (1 + e^2z), whose error of 6.5 units falls on a difference from 1 of
// at most 0.24.  (glibc's steps, which llmk_sample_batch repeats bit for bit,
// take about four times the operations: 256 x 128256 bf16 to f32 with a softcap
// takes 40 us with these, and took 51 longer with those.)
__device__ __forceinline__ float tanh_f32(float z) {
  const float a = __builtin_fabsf(z), s = z * z;
  float q = -0x1.bc54ap-12f;
  q = __builtin_fmaf(q, s, 0x1.4a425ap-9f);
  q = __builtin_fmaf(q, s, -0x1.0da91p-7f);
  q = __builtin_fmaf(q, s, 0x1.62f81cp-6f);
  q = __builtin_fmaf(q, s, -0x1.b9d83p-5f);
  q = __builtin_fmaf(q, s, 0x1.11100ep-3f);
  q = __builtin_fmaf(q, s, -0x1.555554p-2f);
  const float near = __builtin_fmaf(z * s, q, z);
  const float e = __builtin_amdgcn_exp2f(a * 0x1.715476p+1f);  // 2 log2(e)
  const float far = __builtin_copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + e), z);
  return a < 1.0f ? near : far;
}

// The softcap (DT & SOFTCAP) of a logit; a logit from memory.
template <int DT>
__device__ __forceinline__ float cap_f32(float x, float m1, float cap) {
  return DT & SOFTCAP ? tanh_f32(x * m1) * cap : x;
}
template <int DT>
__device__ __forceinline__ float raw_f32(const void* row, uint32_t e) {
  return Elem<DT>::SZ == 4 ? G((const float*)row)[e] : cvt16<DT>(G((const uint16_t*)row)[e]);
}


// x / T as IEEE division rounds it, for 2^-17 < T < 2^20: with r = 1 / T
// rounded, two steps q += (x - q T) r (each residual one fused operation, so
// exact) leave the correctly rounded quotient (Markstein: the last step does
// if r is the rounded reciprocal of a T whose significand is not all ones and
// q is within a unit of the quotient).  Five operations instead of a dozen.
// Numbers that could leave the normal range on the way, zeros, infinities and
// NaN take the division itself.
struct Divisor {
  float T, r;
  bool fast;
};
__device__ __forceinline__ Divisor divisor(float T) {
  const uint32_t m = __float_as_uint(T) & 0x7fffffu;
  return {T, 1.0f / T, T > 0x1p-17f && T < 0x1p+20f && m != 0x7fffffu};
}
__device__ __forceinline__ void divide4(float* x, const Divisor& d) {
  const float hi = fmaxf(fmaxf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1])),
                         fmaxf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3])));
  const float lo = fminf(fminf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1])),
                         fminf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3])));
  const float all = x[0] + x[1] + x[2] + x[3];  // NaN if one is (hi and lo leave it out)
  if (d.fast && hi < 0x1p+100f && lo > 0x1p-90f && all == all) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float q = x[k] * d.r;
      q = __builtin_fmaf(__builtin_fmaf(-q, d.T, x[k]), d.r, q);
      x[k] = __builtin_fmaf(__builtin_fmaf(-q, d.T, x[k]), d.r, q);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = x[k] / d.T;
  }
}

constexpr uint32_t PT = 256;        // threads of process_kernel
constexpr uint32_t TOUCHED = 2048;  // tokens listed per segment (below)

// One workgroup per (row, segment of PT * N logits).  LDS holds a word per
// logit of the segment: how often its token occurs, less one (all ones:
// never).  A segment is small enough for a word per logit, so this needs no
// table, no hash and no limit on a history.  A row with biases first uses the
// words for those: each token's bias, or, where the segment has a token that is
// listed more than once, its biases' sum, which the thread that holds its logit
// adds up from the list in its order: work in proportion to the list (64 x
// 151936 f32 with 20000 biases 76 us, 150 with one of them repeated in a row,
// 234 with half of them; a walk down the list per token took 34 ms and 76 ms).
//
// Bound by HBM without lists (512 x 128256 bf16 to bf16 47 us, 5.5 TB/s).  With
// them by the steps before the last logit can be written: extents, tokens,
// words, each a wait that only the CU's other seven workgroups fill (with
// histories of 1000 tokens 66 us; 256 x 151936 f32 with 2048 tokens 60 us,
// 5.2 TB/s).  So workgroups are small (512 threads for segments twice as long
// took up to 8 % longer, 1024 threads 5 to 29 %, 128 threads up to 7 %), the
// tokens are requested before the logits (loads come back in order), barriers
// wait for LDS alone, and the penalties are computed where the logits are,
// though that costs a wave an operation for each of its logits as soon as one
// of the 64 neighbours has a count: a list of the touched tokens, penalised by
// a thread each from memory, took 9 % longer.
// TOUCHED_ONLY, for calls in place that change no other logit (no softcap, bias,
// mask or temperature), has such a list, and reads and writes nothing else.
// Fewer, longer workgroups that run over several segments with the next one's
// logits on their way took 90 us: fewer of them fit a CU.  The segments of a
// row re-read its lists from L2, so they share an XCD.
template <int DT, int OT, uint32_t N, bool TOUCHED_ONLY>
__global__ __launch_bounds__(PT, 8) void process_kernel(PArgs a) {
  extern __shared__ uint32_t psm[];
  __shared__ uint16_t s_list[TOUCHED_ONLY ? TOUCHED : 1];
  __shared__ uint32_t s_listed, s_twice, s_here[PT / WAVE];
  __shared__ u2v s_pair[TOUCHED_ONLY ? 1 : PT];
  // 16 bytes a lane from memory or, where the results are wider, to it: then a
  // wave's stores fill lines (512 x 128257 bf16 to f32 75 us; 83 with 16 bytes
  // read a lane, whose 32 bytes go out in two halves).
  constexpr uint32_t W = OT == LLMK_F32 ? 4 : Elem<DT>::W, CH = N / W, SEG = PT * N;
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

  const uint32_t q = a.row_seq ? G(a.row_seq)[b] : b;
  int32_t mi = -1;
  if (a.mask) mi = a.mask_index ? G(a.mask_index)[b] : (int32_t)b;
  const uint32_t x0 = *G(row_or(a.xbeg, b, &kZeroU)), xc = *G(row_or(a.xcnt, b, &kZeroU));
  bool bad = (a.row_seq && q >= a.sequences) || (mi >= 0 && (uint32_t)mi >= a.mask_rows);
  const uint32_t qs = a.row_seq && q >= a.sequences ? 0u : q;
  RowP P;
  P.T = *G(row_or(a.T, qs, &kOneF));
  P.rp = *G(row_or(a.rp, qs, &kOneF));
  P.pp = *G((const float*)row_or(a.pp, qs, &kZeroU));
  P.fp = *G((const float*)row_or(a.fp, qs, &kZeroU));
  const uint32_t h0 = *G(row_or(a.hoff, qs, &kZeroU));
  const uint32_t hl = *G(row_or(a.hlen, qs, &kZeroU));
  const uint32_t he = *G(row_or(a.hlen ? nullptr : a.hoff, qs + 1, &kZeroU));
  const uint32_t j0 = *G(row_or(a.boff, qs, &kZeroU)), j1 = *G(row_or(a.boff, qs + 1, &kZeroU));
  if (!finitef(P.T) || !finitef(P.rp) || !finitef(P.pp) || !finitef(P.fp)) bad = true;
  if (bad) {  // the whole workgroup agrees
    for (uint32_t e = lo + tid; e < lo + n; e += PT) store_one<OT>(orow, e, __builtin_nanf(""));
    if (g == 0 && tid == 0) atomicOr(a.status, LLMK_STATUS_INVALID_PARAMS);
    return;
  }

  // the lists: the first tokens of each thread
  const bool pen = P.rp != 1.0f || P.pp != 0.0f || P.fp != 0.0f;
  const uint32_t h1 = a.hlen ? h0 + hl : he;
  const uint32_t hn = pen && h1 > h0 ? h1 - h0 : 0u, xn = pen ? xc : 0u;
  const uint32_t nb = j1 > j0 ? j1 - j0 : 0u, whole = hn & ~3u;
  const uint32_t *ht = a.htok + h0, *hc = a.hcnt ? a.hcnt + h0 : nullptr;
  const uint32_t *xt = a.xtok + x0, *bt = a.btok + j0;
  const float* bv = a.bval + j0;
  u4v_list ht0 = {EMPTY, EMPTY, EMPTY, EMPTY}, hc0 = {1, 1, 1, 1};
  uint32_t ht1 = EMPTY, hc1 = 1, xt0 = EMPTY, bt0 = EMPTY, bv0 = 0;
  if (4 * tid < whole) {
    ht0 = *(const GLB u4v_list*)G(ht + 4 * tid);
    if (hc) hc0 = *(const GLB u4v_list*)G(hc + 4 * tid);
  }
  if (whole + tid < hn) {
    ht1 = G(ht)[whole + tid];
    if (hc) hc1 = G(hc)[whole + tid];
  }
  if (tid < xn) xt0 = G(xt)[tid];
  if (tid < nb) {
    bt0 = G(bt)[tid];
    bv0 = G((const uint32_t*)bv)[tid];
  }
  // the mask's words and the logits
  const uint32_t* mrow =
      a.mask && mi >= 0 ? a.mask + (uint64_t)(uint32_t)mi * a.mask_words : nullptr;
  uint32_t mw[CH];
  if (mrow) {
#pragma unroll
    for (uint32_t c = 0; c < CH; ++c)  // (no lane skips a load: it would be waited for here)
      mw[c] = G(mrow)[umin(lo + (c * PT + tid) * W, a.V - 1) >> 5];
  }
  u4v r[CH];
  auto request = [&]() {
#pragma unroll
    for (uint32_t c = 0; c < CH; ++c) {
      const uint32_t e = lo + (c * PT + tid) * W;
      r[c] = u4v{0, 0, 0, 0};
      if (e < a.V) r[c] = load_pack<DT, W>(row, e, a.V);
    }
  };
  if (!TOUCHED_ONLY) request();

  LDS uint32_t* cnt = (LDS uint32_t*)psm;
  LDS uint16_t* list = (LDS uint16_t*)s_list;
  auto clear = [&]() {
    for (uint32_t i = tid; i < SEG / 4; i += PT)
      *(LDS u4v*)(cnt + 4 * i) = u4v{EMPTY, EMPTY, EMPTY, EMPTY};
  };
  float add[N];  // biases of the thread's logits
  if (hn | xn | nb) {
    clear();
    if (tid == 0) s_listed = s_twice = 0;
    lds_barrier();
  }
  if (nb && !TOUCHED_ONLY) {
    auto place = [&](uint32_t t, uint32_t v) {
      if (t < n && __hip_atomic_exchange(cnt + t, v == EMPTY ? 0x7fc00000u : v, __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_WORKGROUP) != EMPTY)
        s_twice = 1;
    };
    if (tid < nb) place(bt0 - lo, bv0);  // (waves without a pair wait for no load)
    for (uint32_t j = PT + tid; j < nb; j += PT)
      place(G(bt)[j] - lo, G((const uint32_t*)bv)[j]);
    lds_barrier();
    if (s_twice != 0) {
      // Each token's sum instead: PT pairs at a time, those of the segment in
      // listing order, by the threads that hold their logits.
      LDS uint32_t* here = (LDS uint32_t*)s_here;
      LDS u2v* pair = (LDS u2v*)s_pair;
      const uint32_t wv = tid >> 6;
      clear();
      for (uint32_t j0 = 0; j0 < nb; j0 += PT) {
        const uint32_t j = j0 + tid, t = j < nb ? G(bt)[j] - lo : EMPTY;
        const uint32_t v = t < n ? G((const uint32_t*)bv)[j] : 0u;
        const uint64_t who = __ballot(t < n);
        if ((tid & 63u) == 0) here[wv] = (uint32_t)__popcll(who);
        lds_barrier();
        uint32_t at = lanes_below(who), all = 0;
#pragma unroll
        for (uint32_t i = 0; i < PT / WAVE; ++i) {
          at += i < wv ? here[i] : 0u;
          all += here[i];
        }
        if (t < n) pair[at] = u2v{t, v};
        lds_barrier();
        all = (uint32_t)__builtin_amdgcn_readfirstlane((int)all);
        for (uint32_t i = 0; i < all; ++i) {
          const u2v p = pair[i];
          if (p[0] / W % PT != tid) continue;
          const uint32_t m = cnt[p[0]];
          const float sum = m == EMPTY ? __uint_as_float(p[1])
                                       : __uint_as_float(m) + __uint_as_float(p[1]);
          cnt[p[0]] = sum == sum ? __float_as_uint(sum) : 0x7fc00000u;
        }
        lds_barrier();  // the pairs are read
      }
    }
#pragma unroll
    for (uint32_t h = 0; h < N; h += 4) {
      const uint32_t at = ((h / W) * PT + tid) * W + h % W;
      const u4v m = *(LDS u4v*)(cnt + at);
      if ((m[0] & m[1] & m[2] & m[3]) != EMPTY)  // for the counts
        *(LDS u4v*)(cnt + at) = u4v{EMPTY, EMPTY, EMPTY, EMPTY};
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k) add[h + k] = m[k] == EMPTY ? 0.0f : __uint_as_float(m[k]);
    }
    lds_barrier();
  }
  if (hn | xn) {
    // the atomics of several tokens together, then what they found
    auto count = [&](auto tok, auto times, auto how_many) {
      constexpr int K = decltype(how_many)::value;
      uint32_t was[K];
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const uint32_t t = tok(i) - lo, k = times(i);
        was[i] = 0;
        if (t < n)
          was[i] = __hip_atomic_fetch_add(cnt + t, k ? k : 1u, __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_WORKGROUP);
      }
#pragma unroll
      for (int i = 0; i < K; ++i) {
        if (!TOUCHED_ONLY || was[i] != EMPTY) continue;
        const uint32_t at = __hip_atomic_fetch_add((LDS uint32_t*)&s_listed, 1u, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_WORKGROUP);
        if (at < TOUCHED) list[at] = (uint16_t)(tok(i) - lo);
      }
    };
    count([&](int i) { return i < 4 ? ht0[i & 3] : i == 4 ? ht1 : xt0; },
          [&](int i) { return i < 4 ? hc0[i & 3] : i == 4 ? hc1 : 1u; },
          std::integral_constant<int, 6>());
    for (uint32_t j = 4 * (PT + tid); j < whole; j += 4 * PT) {
      const u4v_list t = *(const GLB u4v_list*)G(ht + j);
      u4v_list k = {1, 1, 1, 1};
      if (hc) k = *(const GLB u4v_list*)G(hc + j);
      count([&](int i) { return t[i]; }, [&](int i) { return k[i]; },
            std::integral_constant<int, 4>());
    }
    for (uint32_t j = PT + tid; j < xn; j += PT) {
      const uint32_t t = G(xt)[j];
      count([&](int) { return t; }, [](int) { return 1u; }, std::integral_constant<int, 1>());
    }
    lds_barrier();
  }
  if (TOUCHED_ONLY) {  // the touched logits alone, by the list or, if it is full, by the words
    const uint32_t listed = hn | xn ? s_listed : 0u, m = listed > TOUCHED ? n : listed;
    for (uint32_t i = tid; i < m; i += PT) {
      const uint32_t t = listed > TOUCHED ? i : list[i], c = cnt[t] + 1u;
      if (c) store_one<OT>(orow, lo + t, penalize(raw_f32<DT>(row, lo + t), P, c));
    }
    return;
  }
  const bool divide = P.T != 1.0f && P.T > 1e-5f;
  const Divisor D = divisor(P.T);

#pragma unroll
  for (uint32_t c = 0; c < CH; ++c) {
    const uint32_t at = (c * PT + tid) * W, e = lo + at;
    if (e >= a.V) break;
    float x[W];
#pragma unroll
    for (uint32_t k = 0; k < W; ++k) x[k] = cap_f32<DT>(unpack<DT>(r[c], k), a.sc_m1, a.sc_cap);
    if (nb) {
#pragma unroll
      for (uint32_t k = 0; k < W; ++k) {
        const float v = add[c * W + k];
        if (v != 0.0f) x[k] += v;  // (a logit of -0 without a bias stays -0)
      }
    }
    if (hn | xn) {
#pragma unroll
      for (uint32_t h = 0; h < W; h += 4) {
        const u4v m = *(LDS u4v*)(cnt + at + h);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
          if (m[k] != EMPTY) x[h + k] = penalize(x[h + k], P, m[k] + 1u);
      }
    }
    if (divide) {
#pragma unroll
      for (uint32_t h = 0; h < W; h += 4) divide4(x + h, D);
    }
    if (mrow) {
#pragma unroll
      for (uint32_t k = 0; k < W; ++k)
        if (!((mw[c] >> ((e & 31u) + k)) & 1u)) x[k] = NEG_INF;  // W divides 32
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
  float* tmax;       // [B][2 * MAX_SLOTS]: the tiles' maxima
  uint32_t* part;    // [B * G][4]: m, s, tokens before the chosen one
};

constexpr uint32_t TOP_MAX = 32;  // largest top_n
constexpr uint32_t TLIST = 256;   // candidates of a wave

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

template <int DT>
__device__ __forceinline__ float raw_logit(const void* row, uint32_t e) {
  const float x = Elem<DT>::SZ == 4 ? G((const float*)row)[e]
                                    : cvt16<DT>(G((const uint16_t*)row)[e]);
  return x == x ? x : NEG_INF;
}

constexpr float kLog2e = 0x1.715476p+0f;
__device__ __forceinline__ float exp_diff(float x, float m) {  // e^(x - m), x <= m
  return __builtin_amdgcn_exp2f((x - m) * kLog2e);
}

// The 1024 logits of a tile, 16 a lane: raw bits, and element i's index.
template <int DT>
struct Tile16 {
  static constexpr uint32_t W = Elem<DT>::W, NP = 16 / W;
  u4v raw[NP];
  __device__ __forceinline__ void request(const void* row, uint32_t t, uint32_t V) {
#pragma unroll
    for (uint32_t j = 0; j < NP; ++j) {
      const uint32_t e = t * TILE + (j * 64 + (threadIdx.x & 63u)) * W;
      raw[j] = u4v{0, 0, 0, 0};
      if (e < V) raw[j] = load_pack<DT>(row, e, V);
    }
  }
  static __device__ __forceinline__ uint32_t index(uint32_t t, uint32_t i) {
    return t * TILE + ((i / W) * 64 + (threadIdx.x & 63u)) * W + i % W;
  }
  // as floats, what lies past V as -inf
  __device__ __forceinline__ void values(uint32_t t, uint32_t V, float (&x)[16]) const {
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) x[i] = unpack<DT>(raw[i / W], i % W);
    if (t * TILE + TILE > V) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (index(t, i) >= V) x[i] = NEG_INF;
    }
  }
};

// One workgroup per (row, segment), its waves taking the segment's 1024-logit
// tiles in turn.  A lane keeps the running maximum m and sum s = sum e^(x - m)
// of its logits and how many come before the chosen token; the wave leaves
// each tile's maximum.  The row's last workgroup joins the segments.
//
// The likeliest tokens lie in the top_n tiles that are first by (maximum
// descending, index ascending): a token of any other tile has the top_n
// maxima of those before it.  So the stream carries no list; the last
// workgroup reads top_n tiles again and picks from them.  (A list of
// candidates kept by every wave took 90 us instead of 30 for 256 x 151936 f32
// with a list of 8.)  A row of fewer tiles than that has no bound on the list's
// last token, and one of about as many has a low one: all or many of its logits
// are gathered, do not fit, and are read again by the lists that the last lines
// keep.  That takes several times as long (f32, 64 x 16000 with a list of 8 11 us,
// of 20 65; 1000 x 5000 with a list of 1 12 us, of 20 96; 64 x 32000 with a list
// of 20 14 us, of 32 93).
//
// Bound by HBM: that call reads its 156 MB at 5.2 TB/s, without a list at 5.5
// TB/s.  64 registers, so that 8 waves fit a SIMD (2047 x 32000 f16 with a
// list of 1: 35 us with 80 registers, 31.6 with 64); the last steps are kept in
// short loops, since their code comes from L2 when a workgroup first gets there.
template <int DT, bool TOP, uint32_t LT>
__global__ __launch_bounds__(LT, 8) void logprobs_kernel(LArgs a) {
  constexpr uint32_t LWAVES = LT / WAVE;
  __shared__ uint64_t s_list[TOP ? LWAVES * TLIST : 1];
  __shared__ float s_tmax[TOP ? MAX_TILES : 1];
  __shared__ float s_m[LWAVES], s_s[LWAVES];
  __shared__ uint32_t s_c[LWAVES], s_n[LWAVES], s_sel[TOP_MAX], s_last, s_count, s_bound;
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wv = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t b = blockIdx.x / a.G, g = blockIdx.x % a.G;
  const void* row = (const char*)a.logits + (uint64_t)b * a.stride * Elem<DT>::SZ;
  const uint32_t t0 = g * a.tps, t1 = umin(t0 + a.tps, a.ntiles);

  Tile16<DT> in;
  uint32_t t = t0 + wv;
  if (t < t1) in.request(row, t, a.V);
  const uint32_t tok = a.tokens ? G(a.tokens)[b] : EMPTY;
  const bool chosen = tok < a.V;
  const float lt = chosen ? raw_logit<DT>(row, tok) : __builtin_huge_valf();

  // NaN counts as -inf.  The maximum and the comparisons leave it out by
  // themselves, and the sum shows it; only then, or where -inf is what is
  // compared with, are a tile's logits replaced.  (16-bit logits are bound by
  // these operations as much as by memory: with each NaN replaced and the counts
  // kept by lanes, 512 x 128256 bf16 took 33.7 us instead of 29.7.)
  const bool lowest = lt == NEG_INF;
  float m = NEG_INF, s = 0.0f;
  uint32_t before = 0;  // the wave's
  for (; t < t1; t += LWAVES) {
    float x[16], mx, m2, sum;
    in.values(t, a.V, x);
    if (t + LWAVES < t1) in.request(row, t + LWAVES, a.V);
    auto tile = [&]() {
      mx = x[0];
#pragma unroll
      for (uint32_t i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
      float y[16], my = mx;
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) y[i] = x[i];
      if (DT & SOFTCAP) {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i)  // (a masked token stays one)
          y[i] = x[i] == NEG_INF ? NEG_INF : cap_f32<DT>(x[i], a.sc_m1, a.sc_cap);
        my = y[0];
#pragma unroll
        for (uint32_t i = 1; i < 16; ++i) my = fmaxf(my, y[i]);
      }
      m2 = fmaxf(m, my);
      const float mm = m2 == NEG_INF ? 0.0f : m2;
      sum = m2 > m ? s * exp_diff(m, mm) : s;  // (0 the first time)
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) sum += exp_diff(y[i], mm);
    };
    tile();
    if (lowest || __any(!(sum == sum))) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (!(x[i] == x[i])) x[i] = NEG_INF;
      tile();
    }
    m = m2;
    s = sum;
    if (TOP) {
      const float w = wave_max(mx);
      if (lane == 0) s_tmax[t - t0] = w;
    }
    if (chosen) {
      auto count = [&](auto comes_before) {
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) before += (uint32_t)__popcll(__ballot(comes_before(i)));
      };
      if (t * TILE + TILE <= tok)
        count([&](uint32_t i) { return x[i] >= lt; });
      else if (t * TILE > tok)
        count([&](uint32_t i) { return x[i] > lt; });
      else
        count([&](uint32_t i) {
          return x[i] > lt || (x[i] == lt && Tile16<DT>::index(t, i) < tok);
        });
    }
  }
  // the wave's, then the workgroup's share
  const float wm = wave_max(m);
  s = wave_tree_sum(m == NEG_INF ? 0.0f : s * exp_diff(m, wm));
  if (lane == 0) {
    s_m[wv] = wm;
    s_s[wv] = s;
    s_c[wv] = before;
  }
  if (TOP) {
    if (tid == 0) s_count = 0;
    s_list[tid] = 0;
    if (tid < 4) s_list[LT + tid] = 0;
  }
  __syncthreads();
  float M = s_m[0], S = 0.0f;
  uint32_t C = 0;
#pragma unroll
  for (uint32_t i = 1; i < LWAVES; ++i) M = fmaxf(M, s_m[i]);
#pragma unroll
  for (uint32_t i = 0; i < LWAVES; ++i) {
    if (s_m[i] != NEG_INF) S += s_s[i] * exp_diff(s_m[i], M);
    C += s_c[i];
  }
  if (a.G > 1) {
    // what the row's last workgroup reads
    uint32_t* part = a.part + (uint64_t)blockIdx.x * 4;
    float* tmax = a.tmax + (uint64_t)b * (2 * MAX_SLOTS);
    if (TOP)
      for (uint32_t i = tid; i < t1 - t0; i += LT) put_agent((uint32_t*)tmax + t0 + i, __float_as_uint(s_tmax[i]));
    if (tid == 0) {
      put_agent(part, __float_as_uint(M));
      put_agent(part + 1, __float_as_uint(S));
      put_agent(part + 2, C);
    }
    wait_stores();
    __syncthreads();
    if (tid == 0) {
      const uint32_t last = __hip_atomic_fetch_add(a.arrive + b, 1u, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT) == a.G - 1;
      if (last) put_agent(a.arrive + b, 0u);  // for the next call
      s_last = last;
    }
    __syncthreads();
    if (!s_last) return;
    const uint32_t* first = a.part + (uint64_t)b * a.G * 4;
    float m1 = NEG_INF, s1 = 0.0f;
    uint32_t c1 = 0;
    if (lane < a.G) {
      m1 = __uint_as_float(get_agent(first + 4 * lane));
      s1 = __uint_as_float(get_agent(first + 4 * lane + 1));
      c1 = get_agent(first + 4 * lane + 2);
    }
    if (TOP)
      for (uint32_t i = tid; i < a.ntiles; i += LT)
        s_tmax[i] = __uint_as_float(get_agent((const uint32_t*)tmax + i));
    M = wave_max(m1);
    S = wave_tree_sum(m1 == NEG_INF ? 0.0f : s1 * exp_diff(m1, M));
    C = bcast63u(wave_incl_scan(c1));
    __syncthreads();
  }
  // log p(x) = (x - M) - log S; a raw logit of -inf has none
  const float logS = __logf(S);
  auto logp = [&](float raw_x) {
    if (raw_x == NEG_INF) return NEG_INF;
    const float y = cap_f32<DT>(raw_x, a.sc_m1, a.sc_cap);
    return (y - M) - logS;
  };
  if (tid == 0 && a.tokens) {
    G(a.out_lp)[b] = chosen ? logp(lt) : __builtin_nanf("");
    if (a.out_rank) G(a.out_rank)[b] = chosen ? C : EMPTY;
  }
  if (!TOP) return;
  // The first top_n groups of tiles (a group is one tile up to 256 of them), by
  // one wave: a lower bound of the top_n-th largest maximum, bit by bit until
  // few more than top_n groups reach it, and those groups; where many are
  // equal to it, the first of them.
  const uint32_t per = (a.ntiles + 255) / 256, groups = (a.ntiles + per - 1) / per;
  if (wv == 0) {
    const uint32_t n = umin(a.top_n, groups), most = umin(TOP_MAX, n + 4);
    uint32_t key[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = i * 64 + lane;
      key[i] = 0;
      for (uint32_t j = at * per; j < umin(at * per + per, a.ntiles); ++j)
        key[i] = umax(key[i], fkey(s_tmax[j] + 0.0f));
    }
    auto reach = [&](uint32_t c) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) m += (uint32_t)__popcll(__ballot(key[i] >= c));
      return m;
    };
    uint32_t bound = wave_max_u32(umax(umax(key[0], key[1]), umax(key[2], key[3])));
    uint32_t many = reach(bound);
    if (many < n) {
      bound = 0;
      many = groups;
#pragma unroll 1
      for (uint32_t bit = 0x80000000u; bit && many > most; bit >>= 1) {
        const uint32_t m = reach(bound | bit);
        if (m >= n) {
          bound |= bit;
          many = m;
        }
      }
    }
    uint32_t equal = many > most ? n - reach(bound + 1) : EMPTY, at = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t eq = __ballot(key[i] == bound);
      const bool take = key[i] && (key[i] > bound || (key[i] == bound && lanes_below(eq) < equal));
      const uint64_t who = __ballot(take);
      if (take) s_sel[at + lanes_below(who)] = i * 64 + lane;
      at += (uint32_t)__popcll(who);
      equal -= umin(equal, (uint32_t)__popcll(eq));
    }
    if (lane == 0) {
      s_n[0] = at;
      s_bound = n == a.top_n ? bound : 0u;
    }
  }
  __syncthreads();
  const uint32_t ns = s_n[0];
  // Nothing below the bound belongs to the list: what does not fall below is
  // gathered by all waves.  With fewer than top_n groups that is the whole row.
  const float least = s_bound > fkey(NEG_INF) ? funkey(s_bound) : NEG_INF;
  // the selected tiles in turn, a wave each
  auto selected = [&](uint32_t k) {
    const uint32_t t2 = k < ns * per ? s_sel[k / per] * per + k % per : EMPTY;
    return t2 < a.ntiles ? t2 : EMPTY;
  };
  auto gather = [&](const float (&x)[16], uint32_t tt) {
    uint32_t mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)  // (a NaN is none below -inf)
      mine |= least == NEG_INF || x[i] >= least ? 1u << i : 0u;
    while (mine) {  // (few: the logit is read again, which keeps this code short)
      const uint32_t e = Tile16<DT>::index(tt, (uint32_t)__builtin_ctz(mine));
      mine &= mine - 1;
      if (e < a.V) {
        const uint32_t at = __hip_atomic_fetch_add((LDS uint32_t*)&s_count, 1u, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_WORKGROUP);
        if (at < LT) s_list[at] = order_key(raw_logit<DT>(row, e), e);
      }
    }
  };
  uint32_t k = wv, tt = selected(k);
  if (tt != EMPTY) in.request(row, tt, a.V);
  while (k < ns * per) {
    float x[16];
    in.values(tt == EMPTY ? a.ntiles : tt, a.V, x);
    const uint32_t done = tt;
    k += LWAVES;
    tt = k < ns * per ? selected(k) : EMPTY;
    if (tt != EMPTY) in.request(row, tt, a.V);
    if (done != EMPTY) gather(x, done);
  }
  __syncthreads();
  const uint32_t found = s_count;
  if (found <= LT) {
    // each thread counts the tokens before its own one
    const uint64_t mine = tid < found ? s_list[tid] : 0u;
    uint32_t p = 0;
    for (uint32_t j = 0; j < found; j += 4) {  // (zeros follow the last one)
      uint64_t o[4];
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) o[q] = s_list[j + q];
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) p += o[q] > mine ? 1u : 0u;
    }
    if (tid < found && p < a.top_n) {
      G(a.out_ids)[(uint64_t)b * a.top_n + p] = ~(uint32_t)mine;
      G(a.out_top)[(uint64_t)b * a.top_n + p] = logp(key_value(mine));
    }
    if (tid >= found && tid < a.top_n) {
      G(a.out_ids)[(uint64_t)b * a.top_n + tid] = EMPTY;
      G(a.out_top)[(uint64_t)b * a.top_n + tid] = NEG_INF;
    }
    return;
  }
  // More than that (rows of few tiles for the list's length, rows of equal
  // logits, masked rows with fewer tokens left than the list holds): by lists that
  // keep the first top_n.
  __syncthreads();
  LDS uint64_t* list = (LDS uint64_t*)s_list + wv * TLIST;
  uint32_t held = 0;
  uint64_t bar = ((uint64_t)fkey(least) << 32) - 1;
  for (k = wv; k < ns * per; k += LWAVES) {
    tt = selected(k);
    if (tt == EMPTY) continue;
#pragma unroll 4
    for (uint32_t i = 0; i < 16; ++i) {
      const uint32_t e = tt * TILE + i * 64 + lane;
      const uint64_t key = e < a.V ? order_key(raw_logit<DT>(row, e), e) : 0u;
      const bool take = key > bar;
      const uint64_t who = __ballot(take);
      if (who) {
        if (take) list[held + lanes_below(who)] = key;
        held += (uint32_t)__popcll(who);
        if (held > TLIST - 64) {
          held = keep_first<TLIST / 64>(list, held, a.top_n);
          if (held == a.top_n) bar = list[a.top_n - 1];
        }
      }
    }
  }
  held = keep_first<TLIST / 64>(list, held, a.top_n);
  if (lane == 0) s_n[wv] = held;
  __syncthreads();
  if (wv != 0) return;
  // the waves' lists end to end (each moves down, none past its own start)
  LDS uint64_t* all = (LDS uint64_t*)s_list;
  uint32_t N = s_n[0];
  for (uint32_t i = 1; i < LWAVES; ++i) {
    const uint32_t ni = s_n[i];
    const uint64_t x = lane < ni ? all[i * TLIST + lane] : 0u;
    wave_sync();
    if (lane < ni) all[N + lane] = x;
    N += ni;
  }
  N = keep_first<LWAVES * TOP_MAX / 64>(all, N, a.top_n);
  if (lane < a.top_n) {
    const uint64_t x = lane < N ? all[lane] : 0u;
    G(a.out_ids)[(uint64_t)b * a.top_n + lane] = x ? ~(uint32_t)x : EMPTY;
    G(a.out_top)[(uint64_t)b * a.top_n + lane] = x ? logp(key_value(x)) : NEG_INF;
  }
}

}  // namespace llmk

// ===========================================================================
using namespace llmk;

// The most threads that a launch's grid has along x: HIP takes a grid by its
// threads, in 32 bits.
constexpr uint32_t GRID_THREADS = 0xffffffffu;

static bool known_dtype(int32_t dt) {
  return dt == LLMK_F32 || dt == LLMK_BF16 || dt == LLMK_F16;
}

// Checks what both operators ask of their rows of logits.
static int check_rows(const void* p, int32_t dtype, uint32_t batch, uint32_t vocab,
                      uint64_t stride, const char* what) {
  if (!known_dtype(dtype))
    return fail(LLMK_ERR_INVALID_ARGUMENT,
                std::string(what) + ": dtype must be LLMK_F32, LLMK_BF16 or LLMK_F16");
  if (stride < vocab) return fail(LLMK_ERR_INVALID_ARGUMENT, std::string(what) + ": stride < vocab");
  if (batch && stride > (1ull << 55) / batch)  // (so that no offset in bytes overflows)
    return fail(LLMK_ERR_CAPACITY, std::string(what) + ": batch * stride above 2^55");
  if (((uintptr_t)p % (dtype == LLMK_F32 ? 4 : 2)) != 0)
    return fail(LLMK_ERR_ALIGNMENT, std::string(what) + " must be aligned to their elements");
  return LLMK_OK;
}
static int check_softcap(float c) {
  if (!(c >= 0.0f) || !(c < __builtin_huge_valf()))
    return fail(LLMK_ERR_INVALID_ARGUMENT, "softcap must be finite and >= 0 (0 = off)");
  if (c > 0.0f && c < 0x1p-126f)  // 1 / softcap overflows, and a logit of 0 would be NaN
    return fail(LLMK_ERR_INVALID_ARGUMENT, "softcap below 2^-126");
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
  int rc = check_rows(in->logits, in->dtype, in->batch, in->vocab, in->row_stride, "logits");
  if (rc == LLMK_OK) rc = check_rows(in->out, in->out_dtype, in->batch, in->vocab, in->out_stride, "out");
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
  // Segments of 4096 logits where that makes four workgroups per CU or more,
  // of 2048 where it does not.
  constexpr uint32_t big = 16, small = 8;  // logits per thread
  const bool large = (uint64_t)in->batch * ((in->vocab + big * PT - 1) / (big * PT)) >= 1024;
  const uint32_t seg = (large ? big : small) * PT;
  const uint32_t nseg = (in->vocab + seg - 1) / seg;
  const uint64_t blocks = (uint64_t)in->batch * nseg;
  if (blocks > GRID_THREADS / PT)
    return fail(LLMK_ERR_CAPACITY, "batch * vocab too large for one call");
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
  const size_t lds = counts || in->bias_offsets ? 4 * (size_t)seg : 0;
  const bool touched_only = in->out == in->logits && !sc && !in->temperature && !in->allow_mask &&
                            !in->bias_offsets;
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((uint32_t)blocks), dim3(PT), lds,
                       (hipStream_t)stream, a);
  };
#define LLMK_PROCESS(DT, OT)                                                      \
  do {                                                                            \
    if (touched_only && large) launch(process_kernel<DT, DT, big, true>);         \
    else if (touched_only) launch(process_kernel<DT, DT, small, true>);           \
    else if (sc && large) launch(process_kernel<(DT) | SOFTCAP, OT, big, false>); \
    else if (sc) launch(process_kernel<(DT) | SOFTCAP, OT, small, false>);        \
    else if (large) launch(process_kernel<DT, OT, big, false>);                   \
    else launch(process_kernel<DT, OT, small, false>);                            \
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
  int rc = check_rows(in->logits, in->dtype, in->batch, in->vocab, in->row_stride, "logits");
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
  a.tmax = (float*)s->ws.tile_part;
  a.part = (uint32_t*)s->ws.cand;
  a.ntiles = (a.V + TILE - 1) / TILE;
  // The workgroup's size only matters to the last steps of a row with a top
  // list, where one workgroup reads tiles again: the more waves the shorter
  // they take, but the fewer rows a CU holds meanwhile.  Up to 256 rows each has a
  // CU to itself, and 1024 threads are as fast as fewer or faster (256 x 152552
  // bf16 top 5: 256, 512 and 1024 threads 24.3, 22.5, 20.5 us; 64 x 50257 f32 14.9,
  // 11.9, 11.5), one row more and rows wait for each other (257 x 152552: 25.0,
  // 25.3, 28.7).  Rows of fewer than 40 tiles have less than three for each of 16
  // waves, and take one size less: 200 x 39912 f32 16.8, 16.3, 17.2; but 256 x
  // 20456 15.6, 13.9, 11.3.  Past 256 rows 512 threads for long ones (512 x 102376
  // f32 43.9, 40.1, 42.8), 256 for short ones, which is right for many (2047 x
  // 32000 f16 top 1 31.6, 33.4, 43.8) and not for some hundreds (512 x 20456 f32
  // 18.2, 15.0, 16.2).
  const uint32_t lt = !in->top_n ? 256 : (a.ntiles < 40 ? (a.B <= 256 ? 512 : 256)
                                                        : (a.B <= 256 ? 1024 : 512));
  if (a.B > GRID_THREADS / lt) return fail(LLMK_ERR_CAPACITY, "batch too large for one call");
  // Segments per row: 4096 waves, four on each SIMD, while each has a tile.
  const uint32_t pool = s->max_batch > MAX_WGS ? s->max_batch : MAX_WGS, waves = lt / WAVE;
  uint32_t g = (4096 / waves + a.B - 1) / a.B;
  const uint32_t most = (a.ntiles + waves - 1) / waves;
  if (g > most) g = most;
  if (g > MAX_SEG) g = MAX_SEG;
  if (a.B > s->max_batch || (uint64_t)a.B * g > pool) g = 1;
  a.tps = (a.ntiles + g - 1) / g;
  a.G = (a.ntiles + a.tps - 1) / a.tps;
  HIPCHK(hipSetDevice(s->device));
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(a.B * a.G), dim3(lt), 0, (hipStream_t)stream, a);
  };
#define LLMK_LOGPROBS(DT)                                              \
  do {                                                                 \
    if (!in->top_n) launch(logprobs_kernel<DT, false, 256>);           \
    else if (lt == 256) launch(logprobs_kernel<DT, true, 256>);        \
    else if (lt == 512) launch(logprobs_kernel<DT, true, 512>);        \
    else launch(logprobs_kernel<DT, true, 1024>);                      \
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
