// Paged key/value cache for CDNA4 (gfx950): single-token attention over pages,
// appending new keys and values, and copying pages.
//
// A pool holds pages [P, HKV, page, W] (bf16 for attention): W is head_dim
// padded to a multiple of 8, `page` a power of two >= 16. A sequence is a
// row of page numbers and a length. Strides are arguments, so a layer's slice
// of a pool over all layers works as it is.
#include "common.h"

#include <cfloat>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) float  floatx2;

#define LOG2E 1.4426950408889634f

DEV_INLINE uint32_t pack_bf16(float lo, float hi) {
  floatx2 f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

// ===========================================================================
// Attention of one new token per sequence.
//
//   o[h] = sum_t softmax_t(scale * q[h] . k[t]) v[t],  t < seq_len
//
// Bound by the bytes of K and V, so nothing is staged: a wave takes 32 tokens
// a step straight from global memory into matrix operands.
//   S^T = K Q^T   mfma 16x16x32, A = 16 tokens x 32 channels (a lane's 16-byte
//                 load is its fragment), B = the group's heads (G <= 16).
//                 The result has head = lane & 15 and tokens in registers,
//                 4 g + r of each 16-token tile (g = lane >> 4).
//   O^T = V^T P^T contracts over tokens, whose order is free as long as P and
//                 V agree: lane group g takes tokens {4g..4g+3} of both tiles,
//                 which is what it already holds of P. V rows are loaded
//                 whole (16 lanes x NDW dwords) and the eight tokens of one
//                 channel are put together with one byte permute per two.
// Softmax state and the O accumulator are lane-local in the head. The running
// maximum moves only when it grew by more than 2^8, so most steps need no
// cross-lane traffic. P enters the product as a bf16 pair hi + lo (16 bits of
// mantissa): the matrix pipe is idle anyway, and the result's error is
// that of its own rounding.
//
// Work is split over the contexts in chunks of a length that follows from the sum
// of the lengths, so that the wanted number comes out however wide the table is:
// chunk c of all sequences goes to workgroups c HKV HG .., without gaps. The
// hardware deals workgroups out to the units in turn, and gaps in a regular
// pattern leave units idle: with a fixed number of chunks a sequence, 64 rows of
// 1000 tokens took 83 us in a table of 4096 columns and 124 in one of 131072, and
// take 45 in any; 8 rows 16 and 35, now 12. A sequence that fits one chunk is
// finished here, the others are joined by paged_attn_join_kernel in the order of
// their chunks.
//
// Measured, join included: 64 rows of 32:8 heads x 128 with 1001 .. 32690 tokens,
// 4.4 GB: 757 us, 5.8 TB/s (a plain read of as much 6.1 to 6.2). Small calls wait
// for a chain of loads (lengths, page number, K and V) and for the second launch:
// eight rows of up to 4096 tokens, 52 MB: 16.3 us (a plain read 11.3); one of 2041
// with 12:4 x 159, 5 MB: 10.3, of which the join takes 3.
// ===========================================================================
struct PagedAttnArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  const int* table;
  const int* lens;
  float* part;                 // [chunks, H, D] unnormalised partial outputs
  float* ml;                   // [chunks, H, 2] their maximum and sum
  int64_t q_sb, q_sh;          // strides in elements
  int64_t k_sp, k_sh, k_st;
  int64_t v_sp, v_sh, v_st;
  int64_t table_sb;
  int64_t P;
  int B, H, HKV, D, W, page_shift, M, HG;
  int2* where;                 // [B] a sequence's first chunk and how many
  int* plan;                   // paged_plan_kernel's result, or null
  float inv_few, inv_many;     // 1 / the chunks wanted, see steps_of_chunk
  float scale2;                // scale * log2(e)
};

DEV_INLINE int clampi(int x, int lo, int hi) {
  return x < lo ? lo : (x > hi ? hi : x);
}

// a length longer than the table's row is cut to it
DEV_INLINE int length_of(const PagedAttnArgs& a, int b) {
  return b < a.B ? clampi(a.lens[b], 0, a.M << a.page_shift) : 0;
}

// Steps (128 tokens, 32 for each of the four waves) of a chunk, for the sum of the
// sequences' steps: more than all / few, but where that passes 8 only as much
// more than 8 as exceeds all / many. Hence there are no more than many + B chunks,
// an empty sequence's one among them.
DEV_INLINE int steps_of_chunk(const PagedAttnArgs& a, int all) {
  const int few = (int)((float)all * a.inv_few) + 1;
  const int many = (int)((float)all * a.inv_many) + 1;
  return few <= 8 ? few : clampi(many, 8, 1 << 22);     // 2^29 tokens: a row
}

// steps / n upwards and at least 1, inv = 1 / n. Rounding may make it one more
// than that, and the last chunk empty.
DEV_INLINE int chunks_of(int steps, int n, float inv) {
  const int q = (int)((float)steps * inv);
  return q * n < steps || q == 0 ? q + 1 : q;
}

// For many rows: the steps of a chunk plan[1], the chunks plan[0], and for each
// of them its sequence and number in it, plan[4 + 2 i ..]. Up to 128 rows every
// workgroup finds its chunk by itself, which costs less than the launch. 300 tokens
// each, without / with the plan: 128 rows 34 / 36 us, 256 68 / 63, 1024 320 / 236,
// 4096 1816 / 903 (5.6 TB/s).
#define PLAN_THREADS 1024

__global__ __launch_bounds__(PLAN_THREADS)
void paged_plan_kernel(const PagedAttnArgs a) {
  __shared__ int ws[PLAN_THREADS / 64], all;
  const int tid = threadIdx.x;
  if (tid == 0) all = 0;
  __syncthreads();
  int steps = 0;
  for (int b = tid; b < a.B; b += PLAN_THREADS)
    steps += (length_of(a, b) + 127) >> 7;
  steps = wave_sum(steps);
  if ((tid & 63) == 0) atomicAdd(&all, steps);
  __syncthreads();
  const int per = steps_of_chunk(a, all);
  const float inv = 1.f / (float)per;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += PLAN_THREADS) {
    const int b = b0 + tid;
    const int c = b < a.B
        ? chunks_of((length_of(a, b) + 127) >> 7, per, inv) : 0;
    const int upto = before + block_scan(c, ws);
    for (int i = 0; i < c; ++i)
      reinterpret_cast<int2*>(a.plan + 4)[upto - c + i] = int2{b, i};
    if (b < a.B && a.where) a.where[b] = int2{upto - c, c};
    __syncthreads();
    if (tid == PLAN_THREADS - 1) all = upto;
    __syncthreads();
    before = all;
  }
  if (tid == 0) {
    a.plan[0] = before;
    a.plan[1] = per;
  }
}

template <int NDW, bool PLAN>  // W <= 32 * NDW
__global__ __launch_bounds__(256, 2)
void paged_attn_kernel(const PagedAttnArgs a) {
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.H / a.HKV;

  // workgroup -> (chunk of all sequences, kv head, group of 16 heads);
  // neighbours share a chunk's pages
  const uint32_t hg = blockIdx.x % (uint32_t)a.HG;
  const uint32_t rest = blockIdx.x / (uint32_t)a.HG;
  const int hkv = (int)(rest % (uint32_t)a.HKV);
  const int item = (int)(rest / (uint32_t)a.HKV);

  int b = -1, len = 0, split = 0, count = 0, per;
  if (PLAN) {
    per = a.plan[1];
    if (item < a.plan[0]) {
      const int2 it = reinterpret_cast<const int2*>(a.plan + 4)[item];
      b = it.x;
      split = it.y;
      len = length_of(a, b);
      const int steps = (len + 127) >> 7;
      count = chunks_of(steps, per, 1.f / (float)per);
    }
  } else {
    int steps = 0, before = 0;
    for (int i = lane; i < a.B; i += 64) steps += (length_of(a, i) + 127) >> 7;
    per = steps_of_chunk(a, wave_sum(steps));
    const float inv = 1.f / (float)per;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int n = length_of(a, b0 + lane);
      const int c = b0 + lane < a.B ? chunks_of((n + 127) >> 7, per, inv) : 0;
      const int upto = before + wave_scan(c);
      const unsigned long long more = __ballot(upto > item);
      if (more) {
        const int j = __builtin_ctzll(more);
        b = b0 + j;
        len = __builtin_amdgcn_readlane(n, j);
        count = __builtin_amdgcn_readlane(c, j);
        split = item - (__builtin_amdgcn_readlane(upto, j) - count);
        break;
      }
      before = __builtin_amdgcn_readlane(upto, 63);
    }
  }
  if (b < 0) return;                         // fewer chunks than there could be
  const int chunk = 128 * per;
  if (!PLAN && a.where && split == 0 && hkv == 0 && hg == 0 && threadIdx.x == 0)
    a.where[b] = int2{item, count};
  const int t_begin = split * chunk;
  const int t_end = len - t_begin < chunk ? len : t_begin + chunk;

  const int g = lane >> 4, c16 = lane & 15;
  const int gh = (int)hg * 16 + c16;       // this lane's head in the group
  const bool head_ok = gh < G;
  const int h = hkv * G + (head_ok ? gh : 0);

  bf16x8 qf[NDW];
  {
    const uint16_t* qp = a.q + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh;
    #pragma unroll
    for (int ks = 0; ks < NDW; ++ks) {
      const uintx4 x = load8_ragged(qp, 4 * ks + g, a.D);
      qf[ks] = __builtin_bit_cast(bf16x8,
                                  head_ok ? x : uintx4{0u, 0u, 0u, 0u});
    }
  }
  // channels past head_dim in K's last 8 may hold anything: cut them
  uintx4 kmask;
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int left = a.D - (a.D & ~7) - 2 * j;
    kmask[j] = left >= 2 ? 0xffffffffu : (left == 1 ? 0xffffu : 0u);
  }

  // channels of O: this lane loads dwords [off, off + NDW) of a V row; lanes
  // past the row's end repeat its last ones
  const int off = clampi(NDW * c16, 0, a.W / 2 - NDW);

  floatx4 oacc[2 * NDW];
  #pragma unroll
  for (int i = 0; i < 2 * NDW; ++i) oacc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -FLT_MAX, l = 0.f;             // below every score
  bool seen = false;                       // a token, whatever its score
  const int* tb = a.table + (int64_t)b * a.table_sb;
  const int pmask = (1 << a.page_shift) - 1;
  const uint16_t* kh = a.k + hkv * a.k_sh;
  const uint16_t* vh = a.v + hkv * a.v_sh;

  for (int t0 = t_begin + 32 * wave; t0 < t_end; t0 += 128) {
    // tokens at and after the end repeat the last live one: nothing behind
    // a sequence is read, and its score is set to -inf below
    uintx4 kr[2][NDW];
    uint32_t vr[8][NDW];
    bool ok[2];
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int last = t_end - 1;
      const int tt = t0 + 16 * i <= last ? t0 + 16 * i : (last & ~15);
      const int pg = tb[tt >> a.page_shift];
      ok[i] = pg >= 0 && pg < a.P;
      seen |= ok[i] && t0 + 16 * i < t_end;
      const int64_t pgc = ok[i] ? pg : 0;
      const uint16_t* kp = kh + pgc * a.k_sp;
      const uint16_t* vp = vh + pgc * a.v_sp;
      const int tk = tt + c16 <= last ? tt + c16 : last;
      const uint16_t* krow = kp + (int64_t)(tk & pmask) * a.k_st;
      #pragma unroll
      for (int ks = 0; ks < NDW; ++ks) {
        const int d0 = 32 * ks + 8 * g;
        kr[i][ks] = *reinterpret_cast<const uintx4*>(
            krow + (d0 < a.W ? d0 : 0));
      }
      #pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int tv = tt + 4 * g + r <= last ? tt + 4 * g + r : last;
        const uint16_t* vrow = vp + (int64_t)(tv & pmask) * a.v_st + 2 * off;
        __builtin_memcpy(vr[4 * i + r], __builtin_assume_aligned(vrow, 4),
                         4 * NDW);
      }
    }
    floatx4 st[2];
    #pragma unroll
    for (int i = 0; i < 2; ++i) {
      st[i] = floatx4{0.f, 0.f, 0.f, 0.f};
      #pragma unroll
      for (int ks = 0; ks < NDW; ++ks) {
        const int d0 = 32 * ks + 8 * g;
        uintx4 kf = kr[i][ks];
        if (d0 >= a.D) kf = uintx4{0u, 0u, 0u, 0u};
        else if (d0 + 8 > a.D) kf &= kmask;
        st[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, kf), qf[ks], st[i], 0, 0, 0);
      }
    }
    float s[8];
    #pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int t = t0 + 16 * (j >> 2) + 4 * g + (j & 3);
      const float x = st[j >> 2][j & 3] * a.scale2;
      s[j] = t < t_end && ok[j >> 2] ? x : -INFINITY;
    }
    if (!(ok[0] && ok[1])) {
      // a page number outside the pool: its tokens are left out
      #pragma unroll
      for (int j = 0; j < 8; ++j)
        #pragma unroll
        for (int w = 0; w < NDW; ++w)
          vr[j][w] = ok[j >> 2] ? vr[j][w] : 0u;
    }
    float pm = s[0];
    #pragma unroll
    for (int j = 1; j < 8; ++j) pm = fmaxf(pm, s[j]);
    if (__any(pm > m + 8.f)) {
      pm = fmaxf(pm, __shfl_xor(pm, 16, 64));
      pm = fmaxf(pm, __shfl_xor(pm, 32, 64));
      const float mn = fmaxf(m, pm);
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
      #pragma unroll
      for (int i = 0; i < 2 * NDW; ++i) oacc[i] *= alpha;
    }
    uint32_t ph[4], pl[4];
    #pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float p0 = __builtin_amdgcn_exp2f(s[j] - m);
      const float p1 = __builtin_amdgcn_exp2f(s[j + 1] - m);
      l += p0 + p1;
      const uint32_t u = pack_bf16(p0, p1);
      ph[j / 2] = u;
      pl[j / 2] = pack_bf16(p0 - __builtin_bit_cast(float, u << 16),
                            p1 - __builtin_bit_cast(float, u & 0xffff0000u));
    }
    const bf16x8 pfh = __builtin_bit_cast(bf16x8, uintx4{ph[0], ph[1], ph[2], ph[3]});
    const bf16x8 pfl = __builtin_bit_cast(bf16x8, uintx4{pl[0], pl[1], pl[2], pl[3]});
    #pragma unroll
    for (int w = 0; w < NDW; ++w) {
      #pragma unroll
      for (int e = 0; e < 2; ++e) {
        uintx4 u;
        #pragma unroll
        for (int j = 0; j < 4; ++j)
          u[j] = __builtin_amdgcn_perm(vr[2 * j + 1][w], vr[2 * j][w],
                                       e ? 0x07060302u : 0x05040100u);
        const bf16x8 vf = __builtin_bit_cast(bf16x8, u);
        oacc[2 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            vf, pfl, oacc[2 * w + e], 0, 0, 0);
        oacc[2 * w + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            vf, pfh, oacc[2 * w + e], 0, 0, 0);
      }
    }
  }

  // ---- join the four waves: LDS holds [wave][head of 16][2 + D]. A part without
  // tokens has -inf as its maximum. No tokens at all give zeros; tokens whose scores
  // are all -inf have no softmax: 0 / 0.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  const int nh = G - (int)hg * 16 < 16 ? G - (int)hg * 16 : 16;
  const int rowf = a.D + 2;
  if (c16 < nh) {
    float* row = lds + ((int64_t)wave * nh + c16) * rowf;
    if (g == 0) { row[0] = seen ? m : -INFINITY; row[1] = l; }
    #pragma unroll
    for (int i = 0; i < 2 * NDW; ++i)
      #pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 2 * clampi(NDW * (4 * g + r), 0, a.W / 2 - NDW) + i;
        if (d < a.D) row[2 + d] = oacc[i][r];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * a.D; i += 256) {
    const int hh = i / a.D, d = i - hh * a.D;
    float mw[4], top = -INFINITY;
    #pragma unroll
    for (int w = 0; w < 4; ++w) {
      mw[w] = lds[(w * nh + hh) * rowf];
      top = fmaxf(top, mw[w]);
    }
    const float mm = fmaxf(top, -FLT_MAX);
    float ls = 0.f, os = 0.f;
    #pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(mw[w] - mm);
      ls += f * lds[(w * nh + hh) * rowf + 1];
      os += f * lds[(w * nh + hh) * rowf + 2 + d];
    }
    const int head = hkv * G + (int)hg * 16 + hh;
    if (count == 1) {
      a.o[((int64_t)b * a.H + head) * a.D + d] =
          f32_to_bf16(top == -INFINITY ? 0.f : os / ls);
    } else {
      const int64_t at = (int64_t)item * a.H + head;
      a.part[at * a.D + d] = os;
      if (d == 0) {
        a.ml[at * 2] = top;
        a.ml[at * 2 + 1] = ls;
      }
    }
  }
}

// Joins the chunks of one (sequence, head), always in the same order: wave w
// takes chunks w, w + 4, .., four at a time, so that their loads are under way
// together; what a small call waits for here is one trip to memory, not one for
// the maxima and one for the rest.
__global__ __launch_bounds__(256)
void paged_attn_join_kernel(const PagedAttnArgs a) {
  __shared__ float so[4][192], sm[4], sl[4];
  constexpr int U = 4;
  const int64_t bh = blockIdx.x;
  const int b = (int)(bh / a.H);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int2 at = a.where[b];
  const int n = at.y;
  if (n == 1) return;                          // finished by its only chunk
  const int64_t first = (int64_t)at.x * a.H + (bh - (int64_t)b * a.H);
  const float* ml = a.ml + first * 2;
  const float* part = a.part + first * a.D;
  const int64_t step = a.H;                    // from chunk to chunk
  float m = -FLT_MAX, l = 0.f, acc[3] = {0.f, 0.f, 0.f};
  float top = -INFINITY;
  for (int s0 = wave; s0 < n; s0 += 4 * U) {
    float cm[U], cl[U], x[U][3];
    #pragma unroll
    for (int u = 0; u < U; ++u) {
      // past the end the last one again, with weight 0
      const bool ok = s0 + 4 * u < n;
      const int64_t s = step * (ok ? s0 + 4 * u : n - 1);
      cm[u] = ml[2 * s];
      cl[u] = ml[2 * s + 1];
      #pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int d = lane + 64 * i;
        x[u][i] = d < a.D ? part[s * a.D + d] : 0.f;
      }
      if (!ok) cm[u] = -INFINITY;
    }
    #pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, cm[u]);
    const float mn = fmaxf(m, top);
    const float f = __builtin_amdgcn_exp2f(m - mn);
    l *= f;
    #pragma unroll
    for (int i = 0; i < 3; ++i) acc[i] *= f;
    m = mn;
    #pragma unroll
    for (int u = 0; u < U; ++u) {
      const float g = __builtin_amdgcn_exp2f(cm[u] - mn);
      l += g * cl[u];
      #pragma unroll
      for (int i = 0; i < 3; ++i) acc[i] += g * x[u][i];
    }
  }
  #pragma unroll
  for (int i = 0; i < 3; ++i)
    if (lane + 64 * i < a.D) so[wave][lane + 64 * i] = acc[i];
  if (lane == 0) {
    sm[wave] = top;
    sl[wave] = l;
  }
  __syncthreads();
  top = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float mm = fmaxf(top, -FLT_MAX);
  float g[4], ls = 0.f;
  #pragma unroll
  for (int w = 0; w < 4; ++w) {
    g[w] = __builtin_amdgcn_exp2f(sm[w] - mm);
    ls += g[w] * sl[w];
  }
  const int d = threadIdx.x;
  if (d < a.D) {
    float os = 0.f;
    #pragma unroll
    for (int w = 0; w < 4; ++w) os += g[w] * so[w][d];
    a.o[bh * a.D + d] = f32_to_bf16(top == -INFINITY ? 0.f : os / ls);
  }
}

extern "C" hipError_t lumina_paged_attn(
    const void* q, const void* k, const void* v, void* o, const int* table,
    const int* lens, float* part, float* ml, int* where, int* plan,
    const int64_t* strides, int64_t P, int B, int H, int HKV, int D, int W,
    int page_shift, int M, int few, int many, int chunks, float scale,
    hipStream_t stream) {
  PagedAttnArgs a;
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.o = (uint16_t*)o; a.table = table; a.lens = lens; a.part = part; a.ml = ml;
  a.q_sb = strides[0]; a.q_sh = strides[1];
  a.k_sp = strides[2]; a.k_sh = strides[3]; a.k_st = strides[4];
  a.v_sp = strides[5]; a.v_sh = strides[6]; a.v_st = strides[7];
  a.table_sb = strides[8];
  a.P = P; a.B = B; a.H = H; a.HKV = HKV; a.D = D; a.W = W;
  a.page_shift = page_shift; a.M = M;
  a.where = (int2*)where; a.plan = plan;
  a.inv_few = 1.f / few; a.inv_many = 1.f / many;
  const int G = H / HKV;
  a.HG = (G + 15) / 16;
  a.scale2 = scale * LOG2E;
  const int64_t blocks = (int64_t)chunks * HKV * a.HG;
  if (blocks > 0x7fffffff || (int64_t)B * H > 0x7fffffff)
    return hipErrorInvalidValue;
  const int nh = G < 16 ? G : 16;
  const size_t lds = 4 * (size_t)nh * (D + 2) * sizeof(float);
  if (plan) {
    paged_plan_kernel<<<dim3(1), dim3(PLAN_THREADS), 0, stream>>>(a);
    HIP_CHECK_LAST();
  }
  const dim3 grid((uint32_t)blocks), block(256);
  switch ((W + 31) / 32) {
#define PAGED_ATTN(NDW)                                                      \
    if (plan)                                                                \
      paged_attn_kernel<NDW, true><<<grid, block, lds, stream>>>(a);         \
    else                                                                     \
      paged_attn_kernel<NDW, false><<<grid, block, lds, stream>>>(a);        \
    break;
    case 1:
    case 2: PAGED_ATTN(2)
    case 3: PAGED_ATTN(3)
    case 4: PAGED_ATTN(4)
    case 5: PAGED_ATTN(5)
    case 6: PAGED_ATTN(6)
#undef PAGED_ATTN
    default: return hipErrorInvalidValue;
  }
  HIP_CHECK_LAST();
  if (part) {
    paged_attn_join_kernel<<<dim3((uint32_t)((int64_t)B * H)), block, 0,
                             stream>>>(a);
    HIP_CHECK_LAST();
  }
  return hipSuccess;
}

// ===========================================================================
// Appending: k_pages[page(t), h, row(t), :] = k[t, h, :], zero past head_dim,
// and the same for v. A thread writes 8 elements of a row. Bound by bytes: 8179
// tokens of 4 heads x 159, 42 MB: 10.3 us, 4.1 TB/s. Small calls by the launch: 64
// tokens of 8 x 128: 4.4 us.
// ===========================================================================
struct PagedAppendArgs {
  const char* src[2];
  char* dst[2];
  const int* table;
  const int* pos;
  const int* ids;              // null: token t belongs to sequence t
  int64_t s_t[2], s_h[2];      // source strides in elements
  int64_t d_p[2], d_h[2], d_t[2];
  int64_t table_sb;
  int64_t P, T;
  int B, HKV, D, chunks, page_shift, M, per;   // per: tokens of a workgroup
};

template <typename E>
__global__ __launch_bounds__(256)
void paged_append_kernel(const PagedAppendArgs a) {
  const int which = blockIdx.y;
  const int64_t t0 = (int64_t)blockIdx.x * a.per;
  const int64_t left = a.T - t0;
  // 32 bits count a workgroup's pieces: 64-bit divisions cost more than the bytes
  const uint32_t heads = a.HKV, chunks = a.chunks;
  const uint32_t n = (uint32_t)(left < a.per ? left : a.per) * heads * chunks;
  #pragma unroll 2
  for (uint32_t i = threadIdx.x; i < n; i += 256) {
    const uint32_t row = i / chunks, c = i - row * chunks;
    const uint32_t tr = row / heads, h = row - tr * heads;
    const int64_t t = t0 + tr;
    const int seq = a.ids ? a.ids[t] : (int)t;
    const int pos = a.pos[t];
    // tokens without a place (negative position, past the table, a page number
    // outside the pool) are not written
    if (seq < 0 || seq >= a.B || pos < 0) continue;
    const int pi = pos >> a.page_shift;
    if (pi >= a.M) continue;
    const int pg = a.table[seq * a.table_sb + pi];
    if (pg < 0 || pg >= a.P) continue;
    const E* src = reinterpret_cast<const E*>(a.src[which]) + t * a.s_t[which]
                   + h * a.s_h[which];
    E* dst = reinterpret_cast<E*>(a.dst[which]) + pg * a.d_p[which]
             + h * a.d_h[which]
             + (pos & ((1 << a.page_shift) - 1)) * a.d_t[which] + 8 * c;
    if constexpr (sizeof(E) == 2) {
      *reinterpret_cast<uintx4*>(dst) = load8_ragged(src, c, a.D);
    } else {
      #pragma unroll
      for (int j = 0; j < 8; ++j)
        dst[j] = 8 * (int)c + j < a.D ? src[8 * c + j] : (E)0;
    }
  }
}

extern "C" hipError_t lumina_paged_append(
    const void* k, const void* v, void* kp, void* vp, const int* table,
    const int* pos, const int* ids, const int64_t* strides, int64_t P,
    int64_t T, int B, int HKV, int D, int W, int page_shift, int M,
    int elem_size, hipStream_t stream) {
  PagedAppendArgs a;
  a.src[0] = (const char*)k; a.src[1] = (const char*)v;
  a.dst[0] = (char*)kp; a.dst[1] = (char*)vp;
  a.table = table; a.pos = pos; a.ids = ids;
  for (int i = 0; i < 2; ++i) {
    a.s_t[i] = strides[2 * i]; a.s_h[i] = strides[2 * i + 1];
    a.d_p[i] = strides[4 + 3 * i]; a.d_h[i] = strides[5 + 3 * i];
    a.d_t[i] = strides[6 + 3 * i];
  }
  a.table_sb = strides[10];
  a.P = P; a.B = B; a.HKV = HKV; a.D = D; a.chunks = W / 8;
  a.page_shift = page_shift; a.M = M;
  a.T = T;
  // Tokens of a workgroup: one, so that small calls have enough workgroups, or eight,
  // which keep its threads busy. One / eight, bf16, us: 8 x 128 64 tokens 2.7 / 4.7,
  // 2048 5.4 / 6.2, 4096 8.4 / 8.8, 6000 12.0 / 11.5, 16384 27 / 23; 4 x 159 1024
  // 3.7 / 4.5, 2048 5.2 / 5.2, 4096 8.0 / 6.7, 8192 14.3 / 10.2; 8 x 64 1536 3.7 /
  // 3.9, 3000 5.0 / 4.8, 8192 9.7 / 7.9. fp32, written channel by channel: 4 x 64
  // 1024 4.3 / 4.4, 3000 8.0 / 7.4, 8192 17.4 / 21.1.
  a.per = elem_size == 2 && T >= (HKV * a.chunks <= 96 ? 2048 : 4096) ? 8 : 1;
  const int64_t blocks = (T + a.per - 1) / a.per;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  const dim3 grid((uint32_t)blocks, 2), block(256);
  if (elem_size == 2)
    paged_append_kernel<uint16_t><<<grid, block, 0, stream>>>(a);
  else if (elem_size == 4)
    paged_append_kernel<uint32_t><<<grid, block, 0, stream>>>(a);
  else
    return hipErrorInvalidValue;
  HIP_CHECK_LAST();
  return hipSuccess;
}

// ===========================================================================
// Copying pages: pool[l, dst[i]] = pool[l, src[i]] for every layer l, for up to
// two pools at once. The page numbers travel in the kernel's arguments, so a
// call copies nothing to the device and may be captured. A workgroup moves
// COPY_PIECE bytes of one page. Bound by bytes: 301 pages of 32 layers x 8 x 64 x
// 128, keys and values, 5.0 GB: 970 us, 5.2 TB/s (a plain copy of as much 5.5 to
// 5.9); 3 pages of 31 layers x 4 x 16 x 160: 5.0 us, the launch.
// ===========================================================================
#define COPY_PAIRS 256
#define COPY_PIECE 16384

struct CopyPagesArgs {
  char* pool[2];
  int64_t layer_bytes[2], page_stride[2];   // strides in bytes
  int64_t page_bytes;
  int layers, pieces, n;
  int src[COPY_PAIRS], dst[COPY_PAIRS];
};

template <typename V>
__global__ __launch_bounds__(256)
void copy_pages_kernel(const CopyPagesArgs a) {
  const int which = blockIdx.z;
  const int pair = blockIdx.y;
  const int layer = blockIdx.x / a.pieces;
  const int piece = blockIdx.x - layer * a.pieces;
  char* base = a.pool[which] + layer * a.layer_bytes[which];
  const char* src = base + a.src[pair] * a.page_stride[which];
  char* dst = base + a.dst[pair] * a.page_stride[which];
  const int64_t at = (int64_t)piece * COPY_PIECE;
  const int64_t left = a.page_bytes - at;
  const int bytes = left < COPY_PIECE ? (int)left : COPY_PIECE;
  const V* s = reinterpret_cast<const V*>(src + at);
  V* d = reinterpret_cast<V*>(dst + at);
  const int nv = bytes / (int)sizeof(V);
  constexpr int U = 4;
  for (int i = threadIdx.x; i < nv; i += 256 * U) {
    V v[U];
    #pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + 256 * u < nv) v[u] = __builtin_nontemporal_load(s + i + 256 * u);
    #pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + 256 * u < nv) __builtin_nontemporal_store(v[u], d + i + 256 * u);
  }
}

// src and dst are host arrays of n page numbers that the caller has checked.
extern "C" hipError_t lumina_copy_pages(
    void* const* pools, int n_pools, const int64_t* layer_bytes,
    const int64_t* page_stride, int layers, int64_t page_bytes,
    const int* src, const int* dst, int64_t n, hipStream_t stream) {
  CopyPagesArgs a;
  if (n_pools < 1 || n_pools > 2) return hipErrorInvalidValue;
  a.page_bytes = page_bytes;
  a.layers = layers;
  const int64_t pieces = (page_bytes + COPY_PIECE - 1) / COPY_PIECE;
  if (pieces * layers > 0x7fffffff) return hipErrorInvalidValue;
  a.pieces = (int)pieces;
  bool wide = page_bytes % 16 == 0;
  for (int i = 0; i < n_pools; ++i) {
    a.pool[i] = (char*)pools[i];
    a.layer_bytes[i] = layer_bytes[i];
    a.page_stride[i] = page_stride[i];
    wide = wide && (uintptr_t)pools[i] % 16 == 0 && layer_bytes[i] % 16 == 0
           && page_stride[i] % 16 == 0;
  }
  for (int64_t at = 0; at < n; at += COPY_PAIRS) {
    a.n = (int)(n - at < COPY_PAIRS ? n - at : COPY_PAIRS);
    for (int i = 0; i < a.n; ++i) {
      a.src[i] = src[at + i];
      a.dst[i] = dst[at + i];
    }
    const dim3 grid((uint32_t)(pieces * layers), a.n, n_pools), block(256);
    if (wide)
      copy_pages_kernel<uintx4><<<grid, block, 0, stream>>>(a);
    else
      copy_pages_kernel<uint8_t><<<grid, block, 0, stream>>>(a);
    HIP_CHECK_LAST();
  }
  return hipSuccess;
}
