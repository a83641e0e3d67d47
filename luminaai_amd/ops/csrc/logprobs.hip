// Log probabilities of given tokens, entropy and the most likely
// alternatives of each row of logits, and the gradient, for CDNA4 (gfx950).
//
//   lp = x_t - lse      H = lse - sum_j p_j x_j      p_j = exp(x_j - lse)
//   dx_j = g_lp (1[j = t] - p_j) - g_H p_j (log p_j + H)
//
// A workgroup takes a row and reads it once: each thread keeps a running
// maximum m, the sum of 2^y and the sum of y 2^y with y = (x - m) log2(e). The
// difference is taken first: it is exact near the maximum and cannot overflow
// at a mask of the type's lowest value. The kernel is bound by the bytes of the
// logits, with the exponentials close behind: 8192 rows of 50304 in bf16, 0.8 GB:
// 190 us, 4.3 TB/s. The gradient reads them once more and writes as much: 270 us,
// 6.1 TB/s, a part of it from the last-level cache.
//
// Alternatives: the k-th largest of 64 group maxima is a lower bound of the k-th
// largest logit (a little less will do), so only the elements of threads whose own
// maximum reaches it are looked at again (from L2); the candidates go to LDS, where
// each is ranked by counting. Ties go to the lowest index: value and index make one
// 64-bit key. More candidates than fit mean many equal logits, a mask's usually:
// then the bound is made exact, and what lies above it is taken with the first of
// those equal to it (eight rows of five tokens beside a mask, 20 alternatives: 19
// us). If that does not fit either, k rounds of a maximum over the row are taken
// (368 us there). Eight rows of 50304 in fp32 with 20 alternatives take
// 10.8 us: few rows wait for one row's chain of reductions, not for bytes.
#include "common.h"

#define LOG2E 1.4426950408889634f
#define LN2 0.6931471805599453f
#define LP_MAX_K 64
#define LP_CAP 1024            // candidates that fit into LDS

template <typename S> struct Vec8;
template <> struct Vec8<uint16_t> { uint16_t v[8]; };
template <> struct Vec8<float> { float v[8]; };

struct BF16In {
  using S = uint16_t;
  static DEV_INLINE float get(uint16_t u) { return bf16_to_f32(u); }
  static DEV_INLINE uint16_t put(float f) { return f32_to_bf16(f); }
};
struct F16In {
  using S = uint16_t;
  static DEV_INLINE float get(uint16_t u) {
    return (float)__builtin_bit_cast(_Float16, u);
  }
  static DEV_INLINE uint16_t put(float f) {
    return __builtin_bit_cast(uint16_t, (_Float16)f);
  }
};
struct F32In {
  using S = float;
  static DEV_INLINE float get(float f) { return f; }
  static DEV_INLINE float put(float f) { return f; }
};

// rows start at any element: memcpy leaves the choice of the load to the
// compiler, which takes 16-byte loads (global memory takes any alignment)
template <typename S>
DEV_INLINE Vec8<S> load8(const S* p) {
  Vec8<S> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

// The maximum, NaN if one of them is: an instruction for two of them
// (v_maximum3_f32). fmaxf of loaded numbers takes three, since it has to quiet
// NaNs, and made the forward kernel bound by arithmetic.
DEV_INLINE float max_nan(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

// orders floats as unsigned numbers; NaN above all, the two zeros equal. No key is
// all ones, so that of a NaN at index 0 stays below 2^64 - 1 (pair_key).
DEV_INLINE uint32_t order_key(float f) {
  if (f != f) return 0xfffffffeu;
  const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
DEV_INLINE float from_order_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
DEV_INLINE uint64_t pair_key(float f, int idx) {
  return ((uint64_t)order_key(f) << 32) | (uint32_t)~idx;
}

struct RowState { float m, s, t; };   // maximum, sum 2^y, sum y 2^y

DEV_INLINE RowState join(RowState a, RowState b) {
  if (b.s == 0.f) return a;
  if (a.s == 0.f) return b;
  RowState r;
  r.m = fmaxf(a.m, b.m);
  const float da = (a.m - r.m) * LOG2E, db = (b.m - r.m) * LOG2E;
  const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
  r.s = a.s * fa + b.s * fb;
  // a difference past the type's range has factor 0: -1e30 keeps 0 * inf out
  r.t = fa * (a.t + a.s * fmaxf(da, -1e30f))
        + fb * (b.t + b.s * fmaxf(db, -1e30f));
  return r;
}

struct LogprobArgs {
  const void* x;
  const void* tok;
  float* lp;
  float* ent;
  float* stat;                 // [N, 2]: row maximum, log2 of sum exp(x - max)
  float* top_lp;
  int64_t* top_id;
  int64_t N, row_stride;
  int64_t ignore;
  int V, k, tok64;
};

DEV_INLINE int64_t token_of(const void* tok, int is64, int64_t row) {
  return is64 ? reinterpret_cast<const int64_t*>(tok)[row]
              : (int64_t)reinterpret_cast<const int32_t*>(tok)[row];
}

template <typename E, int BLOCK, bool TOP>
__global__ __launch_bounds__(BLOCK)
void logprob_fwd_kernel(const LogprobArgs a) {
  using S = typename E::S;
  constexpr int NW = BLOCK / 64;
  __shared__ float red[NW][3];
  __shared__ float gmax[TOP ? NW : 1][64];
  __shared__ uint64_t cand[TOP ? LP_CAP : 1];
  __shared__ uint64_t best[NW];
  __shared__ int n_cand, equals[NW];
  __shared__ float thr;

  const int64_t row = blockIdx.x;
  const S* x = reinterpret_cast<const S*>(a.x) + row * a.row_stride;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int nvec = a.V >> 3;
  // asked for now, so that nothing waits for it at the end
  const int64_t tk = token_of(a.tok, a.tok64, row);
  const bool inside = tk >= 0 && tk < a.V;
  const float xt = E::get(x[inside ? tk : 0]);

  float mx = -INFINITY, ref = 0.f, s = 0.f, t = 0.f;
  auto take = [&](const float* f, int n) {
    float cm = f[0];
    #pragma unroll
    for (int j = 1; j < n; ++j) cm = max_nan(cm, f[j]);
    if (!(cm <= mx)) {
      // the reference is 0 while all is -inf (inf - inf otherwise): s is 0
      if (mx > -INFINITY) {
        const float d = (mx - cm) * LOG2E, sc = __builtin_amdgcn_exp2f(d);
        t = sc * (t + s * fmaxf(d, -1e30f));
        s *= sc;
      }
      ref = mx = cm;
    }
    #pragma unroll
    for (int j = 0; j < n; ++j) {
      const float y = (f[j] - ref) * LOG2E;
      const float e = __builtin_amdgcn_exp2f(y);
      s += e;
      t = __builtin_fmaf(e, fmaxf(y, -200.f), t);   // 0 * -inf is 0 here
    }
  };
  constexpr int U = sizeof(S) == 2 ? 4 : 2;
  int i = threadIdx.x;
  for (; i + (U - 1) * BLOCK < nvec; i += U * BLOCK) {
    Vec8<S> v[U];
    #pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load8(x + 8 * (int64_t)(i + u * BLOCK));
    float f[8 * U];
    #pragma unroll
    for (int u = 0; u < U; ++u)
      #pragma unroll
      for (int j = 0; j < 8; ++j) f[8 * u + j] = E::get(v[u].v[j]);
    take(f, 8 * U);
  }
  for (; i < nvec; i += BLOCK) {
    const Vec8<S> v = load8(x + 8 * (int64_t)i);
    float f[8];
    #pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = E::get(v.v[j]);
    take(f, 8);
  }
  const int tail = 8 * nvec + threadIdx.x;
  if (tail < a.V) {
    const float f = E::get(x[tail]);
    take(&f, 1);
  }

  // ---- the row's state, joined in a fixed order
  RowState st = {mx, s, t};
  #pragma unroll
  for (int o = 32; o; o >>= 1) {
    RowState b = {__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64),
                  __shfl_xor(st.t, o, 64)};
    st = lane & o ? join(b, st) : join(st, b);
  }
  if (lane == 0) {
    red[wave][0] = st.m; red[wave][1] = st.s; red[wave][2] = st.t;
  }
  if (TOP) gmax[wave][lane] = mx == mx ? mx : -INFINITY;   // NaN: not known
  if (threadIdx.x == 0) n_cand = 0;
  __syncthreads();
  RowState r = {red[0][0], red[0][1], red[0][2]};
  #pragma unroll
  for (int w = 1; w < NW; ++w)
    r = join(r, RowState{red[w][0], red[w][1], red[w][2]});
  // a row of nothing but -inf has no distribution: NaN, as -inf - -inf
  if (r.s == 0.f) r.s = __builtin_nanf("");
  const float ls = __builtin_log2f(r.s);
  if (threadIdx.x == 0) {
    float lp = __builtin_nanf("");         // a token outside the vocabulary
    if (tk == a.ignore) lp = 0.f;
    else if (inside) lp = xt - r.m - LN2 * ls;
    a.lp[row] = lp;
    a.ent[row] = LN2 * (ls - r.t / r.s);
    if (a.stat) {
      a.stat[2 * row] = r.m;
      a.stat[2 * row + 1] = ls;
    }
  }
  if (!TOP) return;

  // the order key's upper bits, from bit `last` on, of the k-th largest group
  // maximum, by bisection; at least k of them are that or more. Many alternatives
  // take the threads' maxima themselves, whose k-th is larger and leaves fewer
  // candidates: 8 rows of 50304, groups / threads: 20 alternatives 11.3 / 11.8 us,
  // 48 16.4 / 14.2, 64 53.6 / 16.6.
  auto bound = [&](int last) {
    uint32_t key[NW];
    uint32_t all = 0;
    #pragma unroll
    for (int w = 0; w < NW; ++w) {
      key[w] = order_key(gmax[w][lane]);
      all = all > key[w] ? all : key[w];
    }
    const bool fine = a.k > 32;
    uint32_t lo = 0;
    #pragma unroll
    for (int bit = 31; bit >= last; --bit) {
      const uint32_t mid = lo | (1u << bit);
      int n = 0;
      if (fine) {
        #pragma unroll
        for (int w = 0; w < NW; ++w)
          n += __builtin_popcountll(__ballot(key[w] >= mid));
      } else {
        n = __builtin_popcountll(__ballot(all >= mid));
      }
      if (n >= a.k) lo = mid;
    }
    if (lane == 0)                         // keys below -inf's are no numbers
      thr = lo < 0x007fffffu ? -INFINITY : from_order_key(lo);
  };
  if (wave == 0) bound(16);
  __syncthreads();
  const float T = thr;
  // Threads whose maximum reaches T (or that met a NaN) have their vectors looked
  // through: by their wave, 16 lanes for each of up to four of them, or, where that
  // would take more trips to L2, by themselves (12 rows of 1024, 32 alternatives:
  // 11.4 -> 7.8 us).
  auto look = [&](int q) {
    const Vec8<S> v = load8(x + 8 * (int64_t)q);
    int n = 0;
    #pragma unroll
    for (int j = 0; j < 8; ++j) n += E::get(v.v[j]) < T ? 0 : 1;
    if (n == 0) return 0;
    int at = atomicAdd(&n_cand, n);
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = E::get(v.v[j]);
      if (!(f < T)) {
        if (at < LP_CAP) cand[at] = pair_key(f, 8 * q + j);
        ++at;
      }
    }
    return at;
  };
  const bool hit = mx >= T || s != s;
  unsigned long long hits = __ballot(hit);
  if (__builtin_popcountll(hits) * BLOCK > 4 * nvec) {
    hits = 0;
    for (int q = threadIdx.x; q - lane < nvec; q += BLOCK) {
      const int at = hit && q < nvec ? look(q) : 0;
      if (__any(at > LP_CAP)) break;         // they do not fit, see below
    }
  }
  while (hits) {
    int owner = -1;
    #pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (hits && lane >> 4 == u) owner = wave * 64 + __builtin_ctzll(hits);
      hits &= hits - 1;                      // 0 & -1 stays 0
    }
    int at = 0;
    for (int q = owner < 0 ? nvec : owner + (lane & 15) * BLOCK; q < nvec;
         q += 16 * BLOCK)
      at = look(q);
    if (__any(at > LP_CAP)) hits = 0;
  }
  if (tail < a.V && threadIdx.x < 8) {
    const float f = E::get(x[tail]);
    if (!(f < T)) {
      const int at = atomicAdd(&n_cand, 1);
      if (at < LP_CAP) cand[at] = pair_key(f, tail);
    }
  }
  __syncthreads();
  auto put = [&](int rank, uint64_t key) {
    a.top_id[row * a.k + rank] = (int)~(uint32_t)key;
    a.top_lp[row * a.k + rank] =
        from_order_key((uint32_t)(key >> 32)) - r.m - LN2 * ls;
  };
  int n = n_cand;
  if (n > LP_CAP) {
    __syncthreads();                       // all have read it
    if (threadIdx.x == 0) n_cand = 0;
    if (wave == 0) bound(0);
    __syncthreads();
    const float B = thr;
    auto keep = [&](float f, int idx) {
      const int at = atomicAdd(&n_cand, 1);
      if (at < LP_CAP) cand[at] = pair_key(f, idx);
    };
    // a thread that met a NaN (s != s) may hold any of them: its maximum started
    // anew behind it
    if (!(mx <= B) || s != s)
      for (int q = threadIdx.x; q < nvec; q += BLOCK) {
        const Vec8<S> v = load8(x + 8 * (int64_t)q);
        #pragma unroll
        for (int j = 0; j < 8; ++j)
          if (!(E::get(v.v[j]) <= B)) keep(E::get(v.v[j]), 8 * q + j);
      }
    if (tail < a.V && threadIdx.x < 8 && !(E::get(x[tail]) <= B))
      keep(E::get(x[tail]), tail);
    __syncthreads();
    const int strict = n_cand;
    n = strict;
    // fewer than k above it: then the k-th is equal to it, and the first of its
    // equals fill up, in order
    for (int q0 = 0; n < a.k && q0 < a.V; q0 += BLOCK) {
      const int q = q0 + threadIdx.x;
      const bool eq = q < a.V && E::get(x[q]) == B;
      const unsigned long long who = __ballot(eq);
      __syncthreads();                     // the last round's counts are read
      if (lane == 0) equals[wave] = __builtin_popcountll(who);
      __syncthreads();
      int at = n + __builtin_popcountll(who & ((1ull << lane) - 1));
      #pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w < wave) at += equals[w];
        n += equals[w];
      }
      if (eq && at < a.k) cand[at] = pair_key(B, q);
    }
    if (strict < a.k && n > a.k) n = a.k;
    __syncthreads();
  }
  if (n <= LP_CAP) {
    // a wave ranks a candidate: 64 comparisons at once
    for (int c = wave; c < n; c += NW) {
      const uint64_t key = cand[c];
      int rank = 0;
      for (int j = lane; j - lane < n; j += 64)
        rank += __builtin_popcountll(__ballot(j < n && cand[j < n ? j : 0]
                                              > key));
      if (lane == 0 && rank < a.k) put(rank, key);
    }
    return;
  }
  uint64_t prev = ~0ull;                 // above every key
  for (int rank = 0; rank < a.k; ++rank) {
    uint64_t b = 0;
    for (int q = threadIdx.x; q < a.V; q += BLOCK) {
      const uint64_t key = pair_key(E::get(x[q]), q);
      if (key < prev && key > b) b = key;
    }
    #pragma unroll
    for (int o = 32; o; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)b, o, 64);
      b = other > b ? other : b;
    }
    __syncthreads();                     // the last round's reads are done
    if (lane == 0) best[wave] = b;
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < NW; ++w) b = best[w] > b ? best[w] : b;
    prev = b;
    if (threadIdx.x == 0) put(rank, b);
  }
}

struct LogprobBwdArgs {
  const void* x;
  const void* tok;
  const float* stat;
  const float* ent;
  const float* g_lp;           // null: zero
  const float* g_ent;          // null: zero
  void* dx;                    // [N, V]
  int64_t N, row_stride, ignore;
  int V, pieces, tok64;
};

#define LP_BWD_VECS 1024       // vectors of 8 that a workgroup takes

// Elementwise over a row's saved maximum and sum: reads x once, writes dx once.
template <typename E>
__global__ __launch_bounds__(256)
void logprob_bwd_kernel(const LogprobBwdArgs a) {
  using S = typename E::S;
  const int64_t row = blockIdx.x / a.pieces;
  const int piece = (int)(blockIdx.x - row * a.pieces);
  const S* x = reinterpret_cast<const S*>(a.x) + row * a.row_stride;
  S* dx = reinterpret_cast<S*>(a.dx) + row * (int64_t)a.V;
  const float mx = a.stat[2 * row], ls = a.stat[2 * row + 1];
  const float H = a.ent[row];
  const int64_t tk = token_of(a.tok, a.tok64, row);
  float gl = a.g_lp ? a.g_lp[row] : 0.f;
  const float ge = a.g_ent ? a.g_ent[row] : 0.f;
  int hot = -1;
  if (tk == a.ignore) gl = 0.f;
  else if (tk >= 0 && tk < a.V) hot = (int)tk;
  else gl = __builtin_nanf("");
  // -p (gl + ge (ln2 y + H)) with y = log2 p
  const float c0 = -(gl + ge * H), c1 = -ge * LN2;
  auto grad = [&](float f, int idx) {
    const float y = __builtin_fmaf(f - mx, LOG2E, -ls);
    const float p = __builtin_amdgcn_exp2f(y);
    const float d = p * __builtin_fmaf(c1, fmaxf(y, -200.f), c0);
    return idx == hot ? d + gl : d;
  };
  const int nvec = a.V >> 3;
  const int v0 = piece * LP_BWD_VECS;
  const int v1 = v0 + LP_BWD_VECS < nvec ? v0 + LP_BWD_VECS : nvec;
  for (int i = v0 + threadIdx.x; i < v1; i += 256) {
    const Vec8<S> v = load8(x + 8 * (int64_t)i);
    Vec8<S> o;
    #pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = E::put(grad(E::get(v.v[j]), 8 * i + j));
    __builtin_memcpy(dx + 8 * (int64_t)i, &o, sizeof(o));
  }
  const int tail = 8 * nvec + threadIdx.x;
  if (piece == a.pieces - 1 && tail < a.V)
    dx[tail] = E::put(grad(E::get(x[tail]), tail));
}

template <typename E, int BLOCK>
static void fwd_launch(const LogprobArgs& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.N), block(BLOCK);
  if (a.k > 0)
    logprob_fwd_kernel<E, BLOCK, true><<<grid, block, 0, stream>>>(a);
  else
    logprob_fwd_kernel<E, BLOCK, false><<<grid, block, 0, stream>>>(a);
}

// dtype: 0 bf16, 1 fp16, 2 fp32
extern "C" hipError_t lumina_logprob_fwd(
    const void* x, int dtype, const void* tok, int tok64, float* lp,
    float* ent, float* stat, float* top_lp, int64_t* top_id, int64_t N, int V,
    int64_t row_stride, int k, int64_t ignore, hipStream_t stream) {
  if (N > 0x7fffffff || k > LP_MAX_K) return hipErrorInvalidValue;
  LogprobArgs a;
  a.x = x; a.tok = tok; a.lp = lp; a.ent = ent; a.stat = stat;
  a.top_lp = top_lp; a.top_id = top_id; a.N = N; a.row_stride = row_stride;
  a.ignore = ignore; a.V = V; a.k = k; a.tok64 = tok64;
  if (dtype == 0) fwd_launch<BF16In, 512>(a, stream);
  else if (dtype == 1) fwd_launch<F16In, 512>(a, stream);
  else if (dtype == 2) fwd_launch<F32In, 512>(a, stream);
  else return hipErrorInvalidValue;
  HIP_CHECK_LAST();
  return hipSuccess;
}

extern "C" hipError_t lumina_logprob_bwd(
    const void* x, int dtype, const void* tok, int tok64, const float* stat,
    const float* ent, const float* g_lp, const float* g_ent, void* dx,
    int64_t N, int V, int64_t row_stride, int64_t ignore, hipStream_t stream) {
  LogprobBwdArgs a;
  a.x = x; a.tok = tok; a.stat = stat; a.ent = ent; a.g_lp = g_lp;
  a.g_ent = g_ent; a.dx = dx; a.N = N; a.row_stride = row_stride;
  a.ignore = ignore; a.V = V; a.tok64 = tok64;
  const int nvec = V / 8;
  a.pieces = nvec > LP_BWD_VECS ? (nvec + LP_BWD_VECS - 1) / LP_BWD_VECS : 1;
  if (N * a.pieces > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)(N * a.pieces)), block(256);
  if (dtype == 0) logprob_bwd_kernel<BF16In><<<grid, block, 0, stream>>>(a);
  else if (dtype == 1) logprob_bwd_kernel<F16In><<<grid, block, 0, stream>>>(a);
  else if (dtype == 2) logprob_bwd_kernel<F32In><<<grid, block, 0, stream>>>(a);
  else return hipErrorInvalidValue;
  HIP_CHECK_LAST();
  return hipSuccess;
}
