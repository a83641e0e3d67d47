// Causal GQA attention over packed sequences, forward and backward, for CDNA4
// (gfx950).
//
// q [T, H, D], k and v [T, HKV, D] bf16 in any strides with contiguous
// channels; sequence b is the tokens cu[b] .. cu[b+1]. 8 <= D <= 192 is padded to a
// multiple of 32 (DP) while a tile is staged, not in memory.
//
//   forward   S = scale Q K^T, P = softmax(S), O = P V, lse2 = log2 sum 2^S2
//   backward  dP = dO V^T, delta = rowsum(dO O), dS = P (dP - delta)
//             dV = P^T dO, dK = scale dS^T Q, dQ = scale dS K
//
// Bound by the matrix pipe, and beside it by the exponentials and the LDS reads
// of the operands. What carries all three kernels:
// - mfma 32x32x16 bf16 (C: column = lane & 31, row = 8 (r >> 2) + 4 (lane >> 5)
//   + (r & 3) for register r). The softmax index runs along the lanes' columns
//   where it can (forward, dQ), so maximum, sum and rescaling are lane-local.
// - A product that contracts over C's rows takes them in the order they lie in:
//   registers 8s .. 8s+7 are already the B fragment of step s, if the other
//   operand supplies rows 16s + 4 hi + {0..3} and 16s + 8 + 4 hi + {0..3}. Two
//   transposing LDS reads (ds_read_b64_tr_b16) at those rows do; P and dS never
//   cross lanes.
// - One LDS image per tile serves both row reads (16 bytes of a row) and
//   transposing reads (4 rows x 64 bytes per half wave): row stride = 16 or 48
//   mod 64 dwords and the 16-byte piece index xor (row >> 2) & 3, which keeps
//   both free of bank conflicts.
// - Tiles go global -> registers -> LDS, loaded one step ahead; two LDS buffers,
//   one barrier a step. The last step loads its own tile once more: where a
//   branch skipped the loads, their registers would be waited for at its end.
#include "common.h"

#include <cfloat>

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) float floatx2;
typedef __attribute__((ext_vector_type(2))) uint32_t uintx2;
typedef __attribute__((ext_vector_type(4))) int intx4;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

#define LOG2E 1.4426950408889634f

struct PackedArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* o;           // backward: forward's result [T, H, D]
  uint16_t* rest;              // [T, H, W] what rounding o left over, or null
  const uint16_t* go;          // backward: its gradient
  uint16_t* out;               // forward: [T, H, D]
  uint16_t* dq;                // [T, H, D]
  uint16_t* dk;                // [T, HKV, D]
  uint16_t* dv;
  float* part;                 // [2 (dk, dv), splits, T, HKV, D up to 4]
  float* lse;                  // [H, T], log2 units
  float* delta;                // [H, T]
  const int* cu;               // [B + 1]
  const int* list;             // packed_list_kernel's blocks, or null
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, go_st, go_sh;
  int T, B, H, HKV, W, D;
  int splits;                  // parts of a group's heads in dK / dV
  float scale;
};

// ---- which rows a workgroup takes ------------------------------------------
struct Work {
  int start;                   // the sequence's first token
  int len;                     // its length
  int level;                   // its blocks number 1 .. n by rising work
  int tail;                    // >= 0: rows behind the last sequence start here
};

// Start and length of sequence b. cu[0] counts as 0 and the rest is cut to [0, T],
// so that no content of it leads outside the tensors; past the last one, 0.
DEV_INLINE int sequence(const int* cu, int B, int T, int b, int& s) {
  s = 0;
  if (b >= B) return 0;
  s = b ? cu[b] : 0;
  s = s < 0 ? 0 : (s > T ? T : s);
  int e = cu[b + 1];
  e = e > T ? T : e;
  return e > s ? e - s : 0;
}

// Block `id` of all sequences' blocks of `rows` rows, then the blocks of the
// rows behind the last sequence. Every wave finds its block by itself, from L2.
//
// The blocks with the most work come first, over all sequences, so that the
// launch does not end with a few long ones. A sequence of n blocks has one of each
// level 1 .. n, hence sum max(0, n - x + 1) blocks are of level x or more, and the
// level is found by bisection. That holds for the 64 sequences of a wave; more of
// them are listed beforehand by packed_list_kernel.
DEV_INLINE Work find_work(const PackedArgs& a, int id, int rows) {
  const int lane = threadIdx.x & 63, T = a.T;
  Work w = {0, 0, 0, -1};
  int all;
  if (a.list) {
    all = a.list[0];
    if (id < all) {
      const int* e = a.list + 4 + 4 * (int64_t)id;
      w.start = e[0];
      w.len = e[1];
      w.level = e[2];
      return w;
    }
  } else {
    int s;
    const int n = sequence(a.cu, a.B, T, lane, s);
    const int nb = (n + rows - 1) / rows;
    all = wave_sum(nb);
    if (id < all) {
      int lo = 1, hi = (T + rows - 1) / rows + 1, above = 0;
      while (hi - lo > 1) {                  // blocks of level lo or more: > id
        const int mid = (lo + hi) >> 1;
        const int more = wave_sum(nb >= mid ? nb - mid + 1 : 0);
        if (more > id) {
          lo = mid;
        } else {
          hi = mid;
          above = more;
        }
      }
      int rank = id - above;                 // among the sequences that have it
      unsigned long long has = __ballot(nb >= lo);
      for (int i = 0; i < rank; ++i) has &= has - 1;
      rank = __builtin_ctzll(has | (1ull << 63));
      w.start = __builtin_amdgcn_readlane(s, rank);
      w.len = __builtin_amdgcn_readlane(n, rank);
      w.level = lo;
      return w;
    }
  }
  int end = a.B > 0 ? a.cu[a.B] : 0;
  end = end < 0 ? 0 : (end > T ? T : end);
  const int64_t tail = end + (int64_t)(id - all) * rows;
  w.tail = tail < T ? (int)tail : T;
  return w;
}

// ===========================================================================
// The blocks of more than 64 sequences, those with the most work first:
// list[0] of them, entry i at list[4 + 4 i ..]: start, length, level. One
// workgroup counts the blocks of each level in LDS and then gives each block
// the next place of its level; levels from LEVELS on are not told apart. Places
// are taken in no fixed order, which moves work between workgroups and changes no
// result. Walking through cu in every workgroup instead, 16384 tokens of 32:8 heads
// x 128 took, forward: in 65 sequences 111 us, with the list 110; in 256 142 and
// 102; in 1024 533 and 312; in 16384 43.8 ms and 4.6.
// ===========================================================================
#define LEVELS 1024

__global__ __launch_bounds__(LEVELS)
void packed_list_kernel(const int* cu, int B, int T, int rows, int cap,
                        int* list) {
  __shared__ int at[LEVELS], ws[LEVELS / 64], top;
  __shared__ unsigned long long total;
  const int tid = threadIdx.x, lane = tid & 63;
  at[tid] = 0;
  if (tid == 0) {
    total = 0;
    top = 0;
  }
  __syncthreads();
  for (int b0 = 0; b0 < B; b0 += LEVELS) {   // sequences by their blocks
    int s;
    const int n = sequence(cu, B, T, b0 + tid, s);
    const int nb = (n + rows - 1) / rows;
    if (nb > 0) atomicAdd(&at[(nb < LEVELS ? nb : LEVELS) - 1], 1);
    if (nb >= LEVELS) atomicAdd(&top, nb - LEVELS + 1);
    const int sum = wave_sum(nb);
    if (lane == 0) atomicAdd(&total, (unsigned long long)sum);
  }
  __syncthreads();
  // level LEVELS - tid: the sequences that have it, then the places before it
  const int have = block_scan(at[LEVELS - 1 - tid], ws);
  const int blocks = tid == 0 ? top : have;
  const int first = block_scan(blocks, ws) - blocks;
  __syncthreads();
  at[LEVELS - 1 - tid] = first;
  __syncthreads();
  // borders that fall may make more blocks than there are rows for: none then
  const bool ok = total <= (unsigned long long)cap;
  if (tid == 0) list[0] = ok ? (int)total : 0;
  if (!ok) return;
  auto put = [&](int s, int n, int level) {
    const int i = atomicAdd(&at[(level < LEVELS ? level : LEVELS) - 1], 1);
    if (i >= 0 && i < cap)
      *reinterpret_cast<intx4*>(list + 4 + 4 * (int64_t)i) =
          intx4{s, n, level, 0};
  };
  for (int b0 = 0; b0 < B; b0 += LEVELS) {
    int s;
    const int n = sequence(cu, B, T, b0 + tid, s);
    const int nb = (n + rows - 1) / rows;
    for (int l = nb < 8 ? nb : 8; l > 0; --l) put(s, n, l);
    unsigned long long big = __ballot(nb > 8);   // by their wave together
    while (big) {
      const int j = __builtin_ctzll(big);
      big &= big - 1;
      const int sj = __builtin_amdgcn_readlane(s, j);
      const int nj = __builtin_amdgcn_readlane(n, j);
      const int bj = __builtin_amdgcn_readlane(nb, j);
      for (int l = 9 + lane; l <= bj; l += 64) put(sj, nj, l);
    }
  }
}

// Heads that share keys and values are given to one XCD (workgroups go round
// the eight of them), so that its L2 holds them once.
DEV_INLINE int head_of(int local, int heads) {
  return heads & 7 ? local : (local & 7) * (heads >> 3) + (local >> 3);
}

// ---- staging ---------------------------------------------------------------
template <int DP> struct Img {
  // dwords of a row: 16 or 48 mod 64
  static constexpr int ROW = (DP / 2) % 64 == 16 || (DP / 2) % 64 == 48
                                 ? DP / 2 : DP / 2 + 16;
  static constexpr int BYTES = ROW * 4;
  static_assert(ROW % 64 == 16 || ROW % 64 == 48, "bank layout");
  static DEV_INLINE int at(int row, int piece) {     // 16-byte pieces
    return row * BYTES + ((piece ^ ((row >> 2) & 3)) << 4);
  }
};

// 8 channels from 8 c on of a row, zero past its end
DEV_INLINE uintx4 load_piece(const uint16_t* row, int c, int W) {
  if (8 * c >= W) return uintx4{0, 0, 0, 0};
  return *reinterpret_cast<const uintx4*>(row + 8 * c);
}
// A tile of ROWS rows on its way from memory to LDS, in the registers of NT
// threads. Channels past W are not cleared: they meet zeros in the other
// operand's fragment (load_piece), or columns that are not stored. They repeat
// the row's own channels, never what lies behind it.
template <int DP, int ROWS, int NT>
struct Stage {
  static constexpr int PIECES = ROWS * DP / 8;
  static constexpr int N = (PIECES + NT - 1) / NT;
  uintx4 v[N];
  uint32_t roff[N], coff[N];                 // bytes of the row and in it

  static DEV_INLINE int piece(int i) {
    // threads past the end repeat the last piece
    const int p = threadIdx.x + i * NT;
    return PIECES % NT == 0 || p < PIECES ? p : PIECES - 1;
  }
  DEV_INLINE void init(int64_t st, int W) {
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = piece(i) / (DP / 8), c = piece(i) - row * (DP / 8);
      roff[i] = 2 * (uint32_t)(row * (int)st);
      coff[i] = 2 * (8 * c < W - 8 ? 8 * c : W - 8);
    }
  }
  // base: the tile's first row; rows past `lim` repeat that one, so that
  // nothing outside the sequence is read. No branch: a register that two paths
  // load is waited for where they meet, which lays the latency bare.
  DEV_INLINE void load(const uint16_t* base, int64_t st, int lim) {
    const char* b = reinterpret_cast<const char*>(base);
    const uint32_t most = 2 * (uint32_t)((lim < ROWS ? lim : ROWS) * (int)st);
    #pragma unroll
    for (int i = 0; i < N; ++i)
      v[i] = *reinterpret_cast<const uintx4*>(
          b + ((roff[i] < most ? roff[i] : most) + coff[i]));
  }
  DEV_INLINE void store(char* img) const {
    #pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = piece(i) / (DP / 8), c = piece(i) - row * (DP / 8);
      *reinterpret_cast<uintx4*>(img + Img<DP>::at(row, c)) = v[i];
    }
  }
};

// A or B fragment of step ks: row lane & 31, channels 16 ks + 8 hi ..
// A lane keeps two addresses, for even and odd ks; the rest is an offset that the
// instruction holds.
template <int DP>
struct RowAddr {
  uint32_t even, odd;
  DEV_INLINE void init(int lane) {
    even = Img<DP>::at(lane & 31, lane >> 5);
    odd = Img<DP>::at(lane & 31, 2 + (lane >> 5));
  }
  DEV_INLINE bf16x8 get(const char* img, int ks) const {
    return *reinterpret_cast<const bf16x8*>(img + (ks & 1 ? odd : even)
                                            + 64 * (ks >> 1));
  }
};

// A fragment of the transposed tile: channel 32 dt + (lane & 31), rows
// r0 + 4 hi + {0..3} and r0 + 8 + 4 hi + {0..3}, r0 a multiple of 16.
// ds_read_b64_tr_b16 hands lane l of 16 the l-th channel of the four rows whose
// 8-byte pieces the lanes address: lane l points at row l >> 2, channels
// 4 (l & 3) .. Two addresses again, for the two groups of rows.
template <int DP>
struct ColAddr {
  uint32_t low, high;
  DEV_INLINE void init(int lane) {
    const int l = lane & 15;
    const int row = 4 * (lane >> 5) + (l >> 2);
    const int ch = (lane & 16) + 4 * (l & 3);
    low = Img<DP>::at(row, ch >> 3) + (ch & 4) * 2;
    high = Img<DP>::at(row + 8, ch >> 3) + (ch & 4) * 2;
  }
  DEV_INLINE bf16x8 get(const char* img, int r0, int dt) const {
    const char* p = img + r0 * Img<DP>::BYTES + 64 * dt;
    union { bf16x4 h[2]; bf16x8 v; } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(p + low));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(p + high));
    return u.v;
  }
};

DEV_INLINE uint32_t pack2(float lo, float hi) {
  floatx2 f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
}

// C's registers 8 s .. 8 s + 7 as the B fragment of step s
DEV_INLINE bf16x8 pack_frag(const float* p) {
  const uintx4 u = {pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]),
                    pack2(p[6], p[7])};
  return __builtin_bit_cast(bf16x8, u);
}

// what rounding two numbers to u left over
DEV_INLINE uint32_t left_over(float lo, float hi, uint32_t u) {
  return pack2(lo - __builtin_bit_cast(float, u << 16),
               hi - __builtin_bit_cast(float, u & 0xffff0000u));
}

// what pack_frag's rounding left over, as a fragment
DEV_INLINE bf16x8 pack_rest(const float* p, bf16x8 f) {
  const uintx4 u = __builtin_bit_cast(uintx4, f);
  const uintx4 v = {left_over(p[0], p[1], u[0]), left_over(p[2], p[3], u[1]),
                    left_over(p[4], p[5], u[2]), left_over(p[6], p[7], u[3])};
  return __builtin_bit_cast(bf16x8, v);
}

DEV_INLINE f32x16 zero16() {
  f32x16 z;
  #pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

DEV_INLINE f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Order of the N products of a block whose operands come from LDS, READS reads
// each: four products' reads ahead, then one more with each product. Left to
// itself the compiler keeps one read in flight, whose latency is two products.
template <int N, int READS>
DEV_INLINE void reads_ahead() {
  constexpr int AHEAD = N < 4 ? N : 4;
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);   // LDS reads
  #pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);             // products
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// A column of a transposed result: this lane's row of memory has channels
// 8 g + 4 hi + {0..3}, g = 0 .. 4 DT - 1, in this lane and the rest in the lane
// 32 away. They swap halves, and each stores 8 channels at once. `rest`, if not
// null, takes what the rounding left over.
DEV_INLINE void store8(uint16_t* row, uint32_t a0, uint32_t a1, uint32_t b0,
                       uint32_t b1, int d, int D, bool live) {
  const auto x = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
  const auto y = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
  if (!live) return;
  const uint32_t u[4] = {x[0], y[0], x[1], y[1]};
  if (d + 8 <= D) {
    *reinterpret_cast<uintx4_any*>(row + d) = uintx4{u[0], u[1], u[2], u[3]};
  } else {
    #pragma unroll
    for (int j = 0; j < 7; ++j)
      if (d + j < D) row[d + j] = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
  }
}

template <int DT>
DEV_INLINE void store_col(uint16_t* row, uint16_t* rest, const f32x16* acc,
                          float f, int hi, int D, int W, bool live) {
  #pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    #pragma unroll
    for (int g = 0; g < 4; g += 2) {
      float x[8];
      uint32_t u[4];
      #pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = acc[dt][4 * g + j] * f;
      #pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = pack2(x[2 * j], x[2 * j + 1]);
      const int d = 32 * dt + 8 * g + 8 * hi;
      store8(row, u[0], u[1], u[2], u[3], d, D, live);
      if (rest)
        store8(rest, left_over(x[0], x[1], u[0]), left_over(x[2], x[3], u[1]),
               left_over(x[4], x[5], u[2]), left_over(x[6], x[7], u[3]), d, W,
               live);
    }
}

// Rows behind the last sequence belong to nothing: zero.
DEV_INLINE void zero_rows(uint16_t* out, int heads, int head, int D, int from,
                          int T, int rows) {
  const int n = T - from < rows ? T - from : rows;
  for (int i = threadIdx.x; i < n * D; i += blockDim.x) {
    const int r = i / D;
    out[((int64_t)(from + r) * heads + head) * D + i - r * D] = 0;
  }
}

// ===========================================================================
// Forward: a workgroup takes Q rows of one head, a wave 32 of them. Two
// workgroups of four waves on a unit are better than one of eight: one's
// exponentials run under the other's products, and causal blocks of half the
// length are levelled better. 8192 tokens, four / eight waves: 32:8 heads x 128
// 257 / 268 us (780 TFLOP/s), 12:4 x 159 95 / 105; 483 tokens of 8:4 x 64
// 7.4 / 9.7. At 192 the images of two do not fit into LDS. Where there are few
// blocks, a second set of waves takes the other half of a step's keys (PARTS = 2)
// and both sets' maximum, sum and result are joined at the end.
//
// P enters P V as bf16: its roundings, up to 2^-8 each and independent from key to
// key, leave an error of 1.9e-3 of the result where the result's own rounding
// leaves 1.6e-3 (483 tokens of 8:4 x 64). Keeping 16 bits as run_bwd's FINE does
// would make three products of two. The sum l is of the unrounded P, in fp32.
// ===========================================================================
template <int DP, int PARTS> struct Fwd {
  static constexpr int W = DP <= 160 ? 4 * PARTS : 8;    // waves
  static constexpr int Q = 32 * W / PARTS;               // rows of a workgroup
  static constexpr int K = DP <= 160 ? 64 * PARTS : 64;  // keys of a step
};

template <int DP, int PARTS>
__global__ __launch_bounds__((64 * Fwd<DP, PARTS>::W), 2)
void packed_fwd_kernel(const PackedArgs a) {
  constexpr int DT = DP / 32, KS = DP / 16;
  constexpr int FQ = Fwd<DP, PARTS>::Q, NT = 64 * Fwd<DP, PARTS>::W;
  constexpr int FK = Fwd<DP, PARTS>::K, KEYS = FK / PARTS;  // of a step, a wave's
  constexpr int IMG = FK * Img<DP>::BYTES;
  constexpr int JOIN = PARTS == 1 ? 0 : 256 * FQ / 32 * (16 * DT + 2);
  __shared__ char lds[4 * IMG > JOIN ? 4 * IMG : JOIN];  // [2][K, V image]
  const int h = head_of(blockIdx.x % a.H, a.H);
  const Work w = find_work(a, blockIdx.x / a.H, FQ);
  if (w.tail >= 0) {
    zero_rows(a.out, a.H, h, a.D, w.tail, a.T, FQ);
    return;
  }
  const int lane = threadIdx.x & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = h / (a.H / a.HKV);
  const int group = wave % (FQ / 32), part = wave / (FQ / 32);
  const int q0 = (w.level - 1) * FQ, qw = q0 + 32 * group;
  const int last = w.len - 1;
  const uint16_t* kb = a.k + w.start * a.k_st + hk * a.k_sh;
  const uint16_t* vb = a.v + w.start * a.v_st + hk * a.v_sh;
  const int qi = qw + (lane & 31);           // this lane's query

  RowAddr<DP> rows;
  ColAddr<DP> cols;
  rows.init(lane);
  cols.init(lane);
  bf16x8 qf[KS];
  {
    const uint16_t* qr = a.q + (int64_t)(w.start + (qi < last ? qi : last))
                         * a.q_st + h * a.q_sh;
    #pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[ks] = __builtin_bit_cast(bf16x8, load_piece(qr, 2 * ks + hi, a.W));
  }
  f32x16 o[DT];
  #pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = zero16();
  float m = -FLT_MAX, l = 0.f;               // below every score
  const float c2 = a.scale * LOG2E;

  // keys up to the last query of the workgroup, or of the sequence
  const int kend = q0 + FQ < w.len ? q0 + FQ : w.len;
  const int steps = (kend + FK - 1) / FK;
  Stage<DP, FK, NT> sk, sv;
  sk.init(a.k_st, a.W);
  sv.init(a.v_st, a.W);
  sk.load(kb, a.k_st, last);
  sv.load(vb, a.v_st, last);
  sk.store(lds);
  sv.store(lds + IMG);
  __syncthreads();
  for (int t = 0; t < steps; ++t) {
    const char* ki = lds + (t & 1) * 2 * IMG + KEYS * part * Img<DP>::BYTES;
    const char* vi = ki + IMG;
    {
      const int64_t r = (int64_t)(t + 1 < steps ? t + 1 : t) * FK;
      sk.load(kb + r * a.k_st, a.k_st, last - (int)r);
      sv.load(vb + r * a.v_st, a.v_st, last - (int)r);
    }
    const int k0 = t * FK + KEYS * part;
    if (k0 <= qw + 31) {                     // else all masked for this wave
      float p[KEYS / 32][16];
      #pragma unroll
      for (int kk = 0; kk < KEYS / 32; ++kk) {
        f32x16 s = zero16();
        #pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          s = mfma(rows.get(ki + 32 * kk * Img<DP>::BYTES, ks), qf[ks], s);
        #pragma unroll
        for (int r = 0; r < 16; ++r) p[kk][r] = s[r];
      }
      if (k0 + KEYS - 1 > qw) {                // touches the diagonal
        #pragma unroll
        for (int kk = 0; kk < KEYS / 32; ++kk)
          #pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int kt = k0 + 32 * kk + 8 * (r >> 2) + 4 * hi + (r & 3);
            if (kt > qi) p[kk][r] = -INFINITY;
          }
      }
      float pm = p[0][0];
      #pragma unroll
      for (int kk = 0; kk < KEYS / 32; ++kk)
        #pragma unroll
        for (int r = 0; r < 16; ++r) pm = fmaxf(pm, p[kk][r]);
      pm *= c2;                              // c2 > 0
      // the maximum follows only when it grew by more than 2^8: sums and
      // products of up to 2^8 lose nothing
      if (__any(pm > m + 8.f)) {
        pm = fmaxf(pm, __shfl_xor(pm, 32, 64));
        const float mn = fmaxf(m, pm);
        const float f = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= f;
        #pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
      }
      #pragma unroll
      for (int kk = 0; kk < KEYS / 32; ++kk) {
        #pragma unroll
        for (int r = 0; r < 16; ++r) {
          p[kk][r] = __builtin_amdgcn_exp2f(
              __builtin_fmaf(p[kk][r], c2, -m));
          l += p[kk][r];
        }
        #pragma unroll
        for (int s = 0; s < 2; ++s) {
          const bf16x8 pf = pack_frag(&p[kk][8 * s]);
          #pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            o[dt] = mfma(cols.get(vi, 32 * kk + 16 * s, dt), pf, o[dt]);
        }
      }
    }
    char* next = lds + ((t + 1) & 1) * 2 * IMG;
    sk.store(next);
    sv.store(next + IMG);
    __syncthreads();
  }
  if (PARTS == 2) {                          // the second part's state joins
    float* other = reinterpret_cast<float*>(lds) + group * 64 * (16 * DT + 2)
                   + lane;
    if (part == 1) {
      #pragma unroll
      for (int i = 0; i < 16 * DT; ++i) other[64 * i] = o[i / 16][i & 15];
      other[64 * 16 * DT] = m;
      other[64 * (16 * DT + 1)] = l;
    }
    __syncthreads();
    if (part == 1) return;
    const float m1 = other[64 * 16 * DT], mn = fmaxf(m, m1);
    const float f0 = __builtin_amdgcn_exp2f(m - mn);
    const float f1 = __builtin_amdgcn_exp2f(m1 - mn);
    m = mn;
    l = l * f0 + other[64 * (16 * DT + 1)] * f1;
    #pragma unroll
    for (int i = 0; i < 16 * DT; ++i)
      o[i / 16][i & 15] = o[i / 16][i & 15] * f0 + other[64 * i] * f1;
  }
  // l is 0 where all of a query's scores are -inf: 0 / 0, as it has no softmax
  l += __shfl_xor(l, 32, 64);
  const int64_t tok = w.start + qi;
  const int64_t at = tok * a.H + h;
  store_col<DT>(a.out + at * a.D, a.rest ? a.rest + at * a.W : nullptr, o,
                1.f / l, hi, a.D, a.W, qi < w.len);
  if (a.lse && hi == 0 && qi < w.len)
    a.lse[(int64_t)h * a.T + tok] = m + __builtin_amdgcn_logf(l);
}

// ===========================================================================
// dQ, and delta for the next kernel: the forward's arrangement, with P from the
// saved lse2. K's image serves S (rows) and dQ (columns). 8192 tokens of 32:8
// heads x 128: 390 us (770 TFLOP/s), of 12:4 x 159: 148, where the few long
// blocks that end last cost a third; the keys of a block shared by two sets of
// four waves in one workgroup took 188 and 467, since all eight then wait for
// each other at every step.
// ===========================================================================
#define BW 4                   // waves
#define BQ (32 * BW)
#define BK 32                  // keys of a step

template <int DP, bool FINE>
__global__ __launch_bounds__(64 * BW, DP <= 160 ? 2 : 1)
void packed_dq_kernel(const PackedArgs a) {
  constexpr int DT = DP / 32, KS = DP / 16, NT = 64 * BW;
  constexpr int IMG = BK * Img<DP>::BYTES;
  // Two waves a SIMD have 256 registers: at DP = 160 that leaves no room for
  // dO's fragments, which go through an image of the wave's own instead. At 192
  // the images would not fit twice; one wave a SIMD then has 512 registers.
  constexpr bool GO_LDS = DP == 160;
  constexpr int OWN = GO_LDS ? 32 * Img<DP>::BYTES : 0;
  __shared__ char lds[4 * IMG + BW * OWN];
  const int h = head_of(blockIdx.x % a.H, a.H);
  const Work w = find_work(a, blockIdx.x / a.H, BQ);
  if (w.tail >= 0) {
    zero_rows(a.dq, a.H, h, a.D, w.tail, a.T, BQ);
    return;
  }
  const int lane = threadIdx.x & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hk = h / (a.H / a.HKV);
  const int q0 = (w.level - 1) * BQ, qw = q0 + 32 * wave;
  const int last = w.len - 1;
  const uint16_t* kb = a.k + w.start * a.k_st + hk * a.k_sh;
  const uint16_t* vb = a.v + w.start * a.v_st + hk * a.v_sh;
  const int qi = qw + (lane & 31);
  const int64_t tok = w.start + (qi < last ? qi : last);

  RowAddr<DP> rows;
  ColAddr<DP> cols;
  rows.init(lane);
  cols.init(lane);
  bf16x8 qf[KS], gf[GO_LDS ? 1 : KS];
  char* own = lds + 4 * IMG + wave * OWN;
  float delta = 0.f;
  {
    const uint16_t* qr = a.q + tok * a.q_st + h * a.q_sh;
    const uint16_t* gr = a.go + tok * a.go_st + h * a.go_sh;
    // delta from o with what its rounding left over: without, the error of dQ and
    // dK is 2.5e-3 to 2.6e-3 for 2.4e-3
    const uint16_t* orow = a.o + (tok * a.H + h) * a.D;
    const uint16_t* rrow = a.rest + (tok * a.H + h) * a.W;
    #pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = __builtin_bit_cast(bf16x8, load_piece(qr, 2 * ks + hi, a.W));
      const bf16x8 gk = __builtin_bit_cast(bf16x8,
                                           load_piece(gr, 2 * ks + hi, a.W));
      if (GO_LDS)
        *reinterpret_cast<bf16x8*>(own + Img<DP>::at(lane & 31, 2 * ks + hi)) =
            gk;
      else
        gf[ks] = gk;
      const bf16x8 of = __builtin_bit_cast(
          bf16x8, load8_ragged(orow, 2 * ks + hi, a.D));
      const bf16x8 rf = __builtin_bit_cast(
          bf16x8, load_piece(rrow, 2 * ks + hi, a.W));
      #pragma unroll
      for (int j = 0; j < 8; ++j)
        delta = __builtin_fmaf((float)gk[j], (float)of[j] + (float)rf[j],
                               delta);
    }
    delta += __shfl_xor(delta, 32, 64);
  }
  const float lse = a.lse[(int64_t)h * a.T + tok];
  if (hi == 0 && qi < w.len) a.delta[(int64_t)h * a.T + tok] = delta;
  f32x16 dq[DT];
  #pragma unroll
  for (int dt = 0; dt < DT; ++dt) dq[dt] = zero16();
  const float c2 = a.scale * LOG2E;

  const int kend = q0 + BQ < w.len ? q0 + BQ : w.len;
  const int steps = (kend + BK - 1) / BK;
  Stage<DP, BK, NT> sk, sv;
  sk.init(a.k_st, a.W);
  sv.init(a.v_st, a.W);
  sk.load(kb, a.k_st, last);
  sv.load(vb, a.v_st, last);
  sk.store(lds);
  sv.store(lds + IMG);
  __syncthreads();
  for (int t = 0; t < steps; ++t) {
    const char* ki = lds + (t & 1) * 2 * IMG;
    const char* vi = ki + IMG;
    {
      const int64_t r = (int64_t)(t + 1 < steps ? t + 1 : t) * BK;
      sk.load(kb + r * a.k_st, a.k_st, last - (int)r);
      sv.load(vb + r * a.v_st, a.v_st, last - (int)r);
    }
    const int k0 = t * BK;
    if (k0 <= qw + 31) {
      f32x16 s = zero16(), dp = zero16();
      #pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = mfma(rows.get(ki, ks), qf[ks], s);
        dp = mfma(rows.get(vi, ks),
                  GO_LDS ? rows.get(own, ks) : gf[GO_LDS ? 0 : ks], dp);
      }
      reads_ahead<2 * KS, 1>();
      float ds[16];
      #pragma unroll
      for (int r = 0; r < 16; ++r) {
        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -lse));
        const int kt = k0 + 8 * (r >> 2) + 4 * hi + (r & 3);
        if (kt > qi) p = 0.f;
        ds[r] = p * (dp[r] - delta);
      }
      #pragma unroll
      for (int st = 0; st < 2; ++st) {
        const bf16x8 f = pack_frag(&ds[8 * st]);
        const bf16x8 rest = pack_rest(&ds[8 * st], f);
        #pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const bf16x8 c = cols.get(ki, 16 * st, dt);
          if (FINE) dq[dt] = mfma(c, rest, dq[dt]);
          dq[dt] = mfma(c, f, dq[dt]);
        }
      }
    }
    char* next = lds + ((t + 1) & 1) * 2 * IMG;
    sk.store(next);
    sv.store(next + IMG);
    __syncthreads();
  }
  store_col<DT>(a.dq + (tok * a.H + h) * a.D, nullptr, dq, a.scale, hi, a.D,
                0, qi < w.len);
}

// ===========================================================================
// dK and dV: a workgroup takes BKV keys of one kv head and goes over the queries
// of the heads that share it, so the sum over those heads stays in registers
// and has one order. S has rows = queries (registers), columns = keys (lanes): P
// and dS are then B fragments of dV^T = dO^T P and dK^T = Q^T dS, and the images
// of Q and dO serve rows and columns.
//
// Two waves share 32 keys: one computes S, P and dV, the other dP, dS and dK,
// a step behind, with P handed over in LDS (fp32, as it lies in the
// registers). Each then holds one accumulator and one of K and V, which leaves
// two waves a SIMD for every head_dim, and one's exponentials run under the
// other's products: 546 us for 8192 tokens of 32:8 heads x 128 (735 TFLOP/s) and
// 185 of 12:4 x 159. One wave for all of it took 1015 us for the former (410
// registers, one wave a SIMD).
//
// Where T * HKV / BKV workgroups of uneven length would not fill the chip, a
// group's heads are split over `splits` workgroups, whose fp32 results
// packed_join_kernel adds in order.
// ===========================================================================
#define BKV 128
#define BQT 32                 // queries of a step
#define BKW 8                  // waves: 4 of each kind

template <int DP, bool FINE>
__global__ __launch_bounds__(64 * BKW, 2)
void packed_dkdv_kernel(const PackedArgs a) {
  constexpr int DT = DP / 32, KS = DP / 16, NT = 64 * BKW;
  constexpr int IMG = BQT * Img<DP>::BYTES;
  constexpr int BUF = 2 * IMG + 2 * BQT * 4;   // Q, dO, lse2, delta
  constexpr int PB = 32 * 32 * 4;              // P of one pair of waves
  __shared__ char lds[3 * BUF + 2 * 4 * PB];
  int id = blockIdx.x;
  const int hk = head_of(id % a.HKV, a.HKV);
  id /= a.HKV;
  const int split = id % a.splits;
  const Work w = find_work(a, id / a.splits, BKV);
  if (w.tail >= 0) {
    if (split == 0) {
      zero_rows(a.dk, a.HKV, hk, a.D, w.tail, a.T, BKV);
      zero_rows(a.dv, a.HKV, hk, a.D, w.tail, a.T, BKV);
    }
    return;
  }
  const int lane = threadIdx.x & 63, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool first = wave < 4;                 // S, P, dV; else dP, dS, dK
  const int pair = wave & 3;
  const int G = a.H / a.HKV, heads = G / a.splits;
  const int h0 = hk * G + split * heads;
  // the first keys have the most queries
  const int kv0 = ((w.len + BKV - 1) / BKV - w.level) * BKV;
  const int kw = kv0 + 32 * pair;
  const int last = w.len - 1;
  const int ki = kw + (lane & 31);             // this lane's key
  const int64_t tok = w.start + (ki < last ? ki : last);

  RowAddr<DP> rows;
  ColAddr<DP> cols;
  rows.init(lane);
  cols.init(lane);
  bf16x8 kvf[KS];                              // K's or V's rows
  {
    const uint16_t* r = first ? a.k + tok * a.k_st + hk * a.k_sh
                              : a.v + tok * a.v_st + hk * a.v_sh;
    #pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      kvf[ks] = __builtin_bit_cast(bf16x8, load_piece(r, 2 * ks + hi, a.W));
  }
  f32x16 acc[DT];                              // dV^T or dK^T
  #pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();
  const float c2 = a.scale * LOG2E;

  const int per = (w.len - kv0 + BQT - 1) / BQT;   // steps of one head
  const int steps = per * heads;
  Stage<DP, BQT, NT> sq, sg;
  float slab = 0.f;
  // the tile to load: its first query and where its rows lie
  int lq = kv0;
  const uint16_t* qp = a.q + (int64_t)(w.start + kv0) * a.q_st + h0 * a.q_sh;
  const uint16_t* gp = a.go + (int64_t)(w.start + kv0) * a.go_st + h0 * a.go_sh;
  const int si = threadIdx.x & (BQT - 1);
  const float* sp = (threadIdx.x & BQT ? a.delta : a.lse)
                    + (int64_t)h0 * a.T + w.start;
  const int64_t q_next = BQT * a.q_st, g_next = BQT * a.go_st;
  const int64_t q_head = a.q_sh - (per - 1) * q_next;
  const int64_t g_head = a.go_sh - (per - 1) * g_next;
  auto load = [&]() {
    sq.load(qp, a.q_st, last - lq);
    sg.load(gp, a.go_st, last - lq);
    // lse2 = +inf makes P zero for rows past the end
    const int row = lq + si;
    slab = sp[row < last ? row : last];
    if (row > last) slab = threadIdx.x & BQT ? 0.f : INFINITY;
  };
  auto advance = [&]() {
    const bool wrap = lq + BQT > last;
    lq = wrap ? kv0 : lq + BQT;
    qp += wrap ? q_head : q_next;
    gp += wrap ? g_head : g_next;
    sp += wrap ? a.T : 0;
  };
  auto store = [&](char* buf) {
    sq.store(buf);
    sg.store(buf + IMG);
    if (threadIdx.x < 2 * BQT)
      reinterpret_cast<float*>(buf + 2 * IMG)[threadIdx.x] = slab;
  };
  sq.init(a.q_st, a.W);
  sg.init(a.go_st, a.W);
  load();
  store(lds);
  __syncthreads();
  int qt = kv0;                                // the step's first query
  int buf = 0;
  // step t: the first kind takes tile t, the second tile t - 1, and tile t + 1
  // is loaded; three buffers go round
  for (int t = 0; t <= steps; ++t) {
    if (t + 1 < steps) advance();
    load();
    const int mine = first ? buf : (buf == 0 ? 2 : buf - 1);
    const char* qi = lds + mine * BUF;
    const char* gi = qi + IMG;
    const float* ls = reinterpret_cast<const float*>(qi + 2 * IMG);
    const bool live = first ? t < steps : t > 0;
    if (live && qt + BQT - 1 >= kw) {          // else all masked for this pair
      char* pb = lds + 3 * BUF + ((first ? t : t - 1) & 1) * 4 * PB + pair * PB
                 + lane * 16;
      const char* ri = first ? qi : gi;        // rows, then columns
      const char* ci = first ? gi : qi;
      f32x16 s = zero16();
      // products go before the other waves' exponentials (8192 tokens of 12:4 x
      // 159: 190 -> 185 us, of 32:8 x 128: 556 -> 546; forward and dQ, whose
      // waves are all of one kind, lose by it)
      __builtin_amdgcn_s_setprio(1);
      #pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s = mfma(rows.get(ri, ks), kvf[ks], s);
      reads_ahead<KS, 1>();
      __builtin_amdgcn_s_setprio(0);
      float p[16];
      if (first) {
        #pragma unroll
        for (int g = 0; g < 4; ++g) {
          const floatx4 le = *reinterpret_cast<const floatx4*>(ls + 8 * g
                                                               + 4 * hi);
          #pragma unroll
          for (int j = 0; j < 4; ++j)
            p[4 * g + j] = __builtin_amdgcn_exp2f(
                __builtin_fmaf(s[4 * g + j], c2, -le[j]));
        }
        if (qt < kw + 31) {                    // touches the diagonal
          #pragma unroll
          for (int r = 0; r < 16; ++r)
            if (ki > qt + 8 * (r >> 2) + 4 * hi + (r & 3)) p[r] = 0.f;
        }
        #pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<floatx4*>(pb + 1024 * g) =
              floatx4{p[4 * g], p[4 * g + 1], p[4 * g + 2], p[4 * g + 3]};
      } else {
        #pragma unroll
        for (int g = 0; g < 4; ++g) {
          const floatx4 de = *reinterpret_cast<const floatx4*>(
              ls + BQT + 8 * g + 4 * hi);
          const floatx4 x = *reinterpret_cast<const floatx4*>(pb + 1024 * g);
          #pragma unroll
          for (int j = 0; j < 4; ++j)
            p[4 * g + j] = x[j] * (s[4 * g + j] - de[j]);
        }
      }
      #pragma unroll
      for (int st = 0; st < 2; ++st) {
        const bf16x8 pf = pack_frag(&p[8 * st]);
        const bf16x8 rest = pack_rest(&p[8 * st], pf);
        __builtin_amdgcn_s_setprio(1);
        #pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const bf16x8 c = cols.get(ci, 16 * st, dt);
          if (FINE) acc[dt] = mfma(c, rest, acc[dt]);
          acc[dt] = mfma(c, pf, acc[dt]);
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }
    buf = buf == 2 ? 0 : buf + 1;
    store(lds + buf * BUF);
    if (live) qt = qt + BQT > last ? kv0 : qt + BQT;
    __syncthreads();
  }
  const float f = first ? 1.f : a.scale;
  if (a.splits == 1) {
    store_col<DT>((first ? a.dv : a.dk) + (tok * a.HKV + hk) * a.D, nullptr,
                  acc, f, hi, a.D, 0, ki < w.len);
  } else if (ki < w.len) {
    const int pw = (a.D + 3) & ~3;
    float* row = a.part + ((((int64_t)(first ? 1 : 0) * a.splits + split) * a.T
                            + tok) * a.HKV + hk) * pw;
    #pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      #pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * dt + 8 * g + 4 * hi;
        if (d < pw)
          *reinterpret_cast<floatx4*>(row + d) =
              floatx4{acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f,
                      acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f};
      }
  }
}

// Adds the splits' results in order, for the rows of the sequences. A thread
// takes four channels of a row; bound by bytes (two parts of 8192 x 8 x 128 twice
// over, 168 MB: 25 us, 6.7 TB/s, much of it from the last-level cache).
__global__ __launch_bounds__(256)
void packed_join_kernel(const PackedArgs a) {
  int end = a.B > 0 ? a.cu[a.B] : 0;
  end = end < 0 ? 0 : (end > a.T ? a.T : end);
  const int pw = (a.D + 3) & ~3, q = pw / 4;
  const int64_t n = (int64_t)a.T * a.HKV * pw;
  const int64_t live = (int64_t)end * a.HKV * q;
  const float* part = a.part + blockIdx.y * a.splits * n;
  uint16_t* out = blockIdx.y ? a.dv : a.dk;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < live;
       i += (int64_t)gridDim.x * 256) {
    floatx4 x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s)
      x += *reinterpret_cast<const floatx4*>(part + s * n + 4 * i);
    const int64_t row = i / q;
    const int d = 4 * (int)(i - row * q);
    uint16_t* p = out + row * a.D + d;
    const uintx2 u = {pack2(x[0], x[1]), pack2(x[2], x[3])};
    if (d + 4 <= a.D) {
      __builtin_memcpy(p, &u, 8);
    } else {
      #pragma unroll
      for (int j = 0; j < 3; ++j)
        if (d + j < a.D) p[j] = (uint16_t)(u[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// Blocks of `rows` rows that any cu can need: a partial one for each sequence
// and one for the rows behind them.
static int64_t max_blocks(const PackedArgs& a, int rows) {
  return a.T / rows + a.B + 1;
}

// Lists the blocks if there are more sequences than a wave has lanes.
static hipError_t list_blocks(PackedArgs& a, int* list, int rows,
                              hipStream_t stream) {
  a.list = list;
  if (!list) return hipSuccess;
  const int64_t cap = max_blocks(a, rows);
  packed_list_kernel<<<dim3(1), dim3(LEVELS), 0, stream>>>(
      a.cu, a.B, a.T, rows, (int)cap, list);
  HIP_CHECK_LAST();
  return hipSuccess;
}

template <int DP, int PARTS>
static hipError_t launch_fwd(PackedArgs& a, int* list, hipStream_t stream) {
  constexpr int Q = Fwd<DP, PARTS>::Q;
  const hipError_t err = list_blocks(a, list, Q, stream);
  if (err != hipSuccess) return err;
  const int64_t n = max_blocks(a, Q) * a.H;
  if (n > 0x7fffffff) return hipErrorInvalidValue;
  packed_fwd_kernel<DP, PARTS><<<dim3((uint32_t)n),
                                 dim3(64 * Fwd<DP, PARTS>::W), 0, stream>>>(a);
  HIP_CHECK_LAST();
  return hipSuccess;
}

template <int DP>
static hipError_t run_fwd(PackedArgs& a, int* list, hipStream_t stream) {
  // Two parts where few blocks leave units idle and a block's time is its chain of
  // steps: there it is halved, while the wider steps and the join cost about 1 us. One
  // / two parts, us:
  //   1 sequence: 2048 tokens of 12:4 x 160 61.7 / 50.3, of 8:4 x 64 30.0 / 25.4, of
  //     32:8 x 128 53.0 / 52.2, 8000 of 8:4 x 64 114 / 102
  //   256 tokens each: 1024 of 12:4 x 160 13.3 / 13.3, of 32:8 x 128 11.3 / 11.8
  //   338 each: 2708 of 2:1 x 64 9.3 / 8.6, of 2:2 x 128 12.4 / 12.2
  //   512 each: 1024 of 32:8 x 128 16.1 / 15.9, 2048 of it 19.9 / 24.9
  //   1000 each: 4000 of 12:4 x 160 37.7 / 35.5, 8000 of 8:4 x 64 19.4 / 21.8
  //   64 each: 1024 of 8:4 x 64 5.2 / 6.4, of 32:8 x 128 8.8 / 17.2
  // At 192 two parts are eight waves for 128 rows instead of 256 (4:4 heads): 125
  // each 8000 15.7 / 15.2, 62 each 4000 11.0 / 11.5; 1000 each 16000 48.5 / 44.9, 500
  // each 31.2 / 34.8.
  // More than 64 sequences may be mostly empty ones, which fill up borders of a
  // fixed size: then as long as one round of workgroups takes them (100 short ones
  // of 2:1 x 64 8.6 / 9.6, of 4:2 x 64, 436 workgroups, 9.2 / 13.5).
  const int64_t size = (int64_t)a.T * a.H;
  const int each = a.T / (a.B > 1 ? a.B : 1);
  const bool fits = a.B > 64 ? max_blocks(a, 128) * a.H <= 256
      : (size <= 32768 && each >= (DP <= 160 ? 320 : 128))
        || (size <= 65536 && each >= (DP <= 160 ? 1536 : 1000));
  if (a.T > 512 && fits)
    return launch_fwd<DP, 2>(a, list, stream);
  return launch_fwd<DP, 1>(a, list, stream);
}

template <int DP, bool FINE>
static hipError_t launch_bwd(PackedArgs& a, int* list, hipStream_t stream) {
  static_assert(BQ == BKV, "one list for both kernels");
  const hipError_t err = list_blocks(a, list, BQ, stream);
  if (err != hipSuccess) return err;
  const int64_t n = max_blocks(a, BQ) * a.H;
  if (n > 0x7fffffff) return hipErrorInvalidValue;
  packed_dq_kernel<DP, FINE><<<dim3((uint32_t)n), dim3(64 * BW), 0, stream>>>(a);
  HIP_CHECK_LAST();
  const int64_t m = max_blocks(a, BKV) * a.HKV * a.splits;
  if (m > 0x7fffffff) return hipErrorInvalidValue;
  packed_dkdv_kernel<DP, FINE><<<dim3((uint32_t)m), dim3(64 * BKW), 0,
                                 stream>>>(a);
  HIP_CHECK_LAST();
  if (a.splits > 1) {
    const int64_t each = (int64_t)a.T * a.HKV * ((a.D + 3) / 4);
    packed_join_kernel<<<dim3(elementwise_grid(each, 256, 2), 2), dim3(256), 0,
                         stream>>>(a);
    HIP_CHECK_LAST();
  }
  return hipSuccess;
}

template <int DP>
static hipError_t run_bwd(PackedArgs& a, int* list, hipStream_t stream) {
  // P and dS enter dV, dK and dQ as bf16; FINE adds what that rounding left over, in
  // a second product. Small calls take it, as the roundings of few terms do not
  // average out and an eager call is bound by the host's 70 us. Forward and gradient,
  // without / with it: 52 tokens of 2:1 x 64 18.7 / 19.6 us with an error of dQ of
  // 2.6e-3 / 1.9e-3 (the result's own rounding is 1.7e-3), 256 of 32:8 x 128 49.8 /
  // 53.1, which a captured graph does pay, 2048 262 / 295, 8192 1084 / 1270 (2.4e-3
  // without). So a sequence's gradients are rounded differently in a larger batch.
  if ((int64_t)a.T * a.H <= 8192) return launch_bwd<DP, true>(a, list, stream);
  return launch_bwd<DP, false>(a, list, stream);
}

static void fill(PackedArgs& a, const int64_t* st, const int* cu, int T, int B,
                 int H, int HKV, int W, int D, float scale) {
  a.q_st = st[0]; a.q_sh = st[1]; a.k_st = st[2]; a.k_sh = st[3];
  a.v_st = st[4]; a.v_sh = st[5]; a.go_st = st[6]; a.go_sh = st[7];
  a.cu = cu; a.T = T; a.B = B; a.H = H; a.HKV = HKV; a.W = W; a.D = D;
  a.scale = scale;
}

#define DISPATCH_DP(W, FN)                                                   \
  if ((W) <= 64) return FN<64>(a, list, stream);                                   \
  if ((W) <= 96) return FN<96>(a, list, stream);                                   \
  if ((W) <= 128) return FN<128>(a, list, stream);                                 \
  if ((W) <= 160) return FN<160>(a, list, stream);                                 \
  if ((W) <= 192) return FN<192>(a, list, stream);                                 \
  return hipErrorInvalidValue;

extern "C" hipError_t lumina_packed_attn_fwd(
    const void* q, const void* k, const void* v, void* out, void* rest,
    float* lse, const int* cu, int* list, const int64_t* strides, int T, int B,
    int H, int HKV, int W, int D, float scale, hipStream_t stream) {
  PackedArgs a = {};
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.out = (uint16_t*)out; a.rest = (uint16_t*)rest; a.lse = lse;
  fill(a, strides, cu, T, B, H, HKV, W, D, scale);
  DISPATCH_DP(W, run_fwd)
}

extern "C" hipError_t lumina_packed_attn_bwd(
    const void* q, const void* k, const void* v, const void* o,
    const void* rest, const void* go, const float* lse, float* delta, void* dq,
    void* dk, void* dv, float* part, int splits, const int* cu, int* list,
    const int64_t* strides, int T, int B, int H, int HKV, int W, int D,
    float scale, hipStream_t stream) {
  PackedArgs a = {};
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.o = (const uint16_t*)o; a.go = (const uint16_t*)go;
  a.rest = (uint16_t*)const_cast<void*>(rest);
  a.lse = const_cast<float*>(lse); a.delta = delta;
  a.part = part; a.splits = splits;
  a.dq = (uint16_t*)dq; a.dk = (uint16_t*)dk; a.dv = (uint16_t*)dv;
  fill(a, strides, cu, T, B, H, HKV, W, D, scale);
  DISPATCH_DP(W, run_bwd)
}

// ===========================================================================
// Rows of D channels anywhere -> rows of W, zero past D, for up to three tensors
// [T, heads, .] at once; a thread moves 8 channels. Rows that start between 16
// bytes cost the kernels above more than this copy: at D = 159 they took 563 us
// together for 8192 tokens of 12:4 heads, and 430 at D = 160, while q, k, v and
// dO are copied in 34.
// ===========================================================================
struct PackRowsArgs {
  const uint16_t* src[3];
  uint16_t* dst[3];
  int64_t st[3], sh[3];        // strides of tokens and heads
  int64_t T;
  int heads[3];
  int D, pieces, per;          // per: tokens of a workgroup
};

// A workgroup's pieces are counted in 32 bits: two 64-bit divisions a piece took
// longer than its bytes.
__global__ __launch_bounds__(256)
void pack_rows_kernel(const PackRowsArgs a) {
  const int w = blockIdx.y;
  const int64_t t0 = (int64_t)blockIdx.x * a.per;
  const int64_t left = a.T - t0;
  const uint32_t heads = a.heads[w], pieces = a.pieces;
  const uint32_t n = (uint32_t)(left < a.per ? left : a.per) * heads * pieces;
  const uint16_t* src = a.src[w] + t0 * a.st[w];
  uint16_t* dst = a.dst[w] + t0 * heads * pieces * 8;
  #pragma unroll 4
  for (uint32_t i = threadIdx.x; i < n; i += 256) {
    const uint32_t row = i / pieces, c = i - row * pieces;
    const uint32_t t = row / heads, h = row - t * heads;
    *reinterpret_cast<uintx4*>(dst + 8 * (int64_t)i) =
        load8_ragged(src + t * a.st[w] + h * a.sh[w], c, a.D);
  }
}

extern "C" hipError_t lumina_pack_rows(const void* const* src, void* const* dst,
                                       const int64_t* strides,
                                       const int* heads, int n, int64_t T,
                                       int D, hipStream_t stream) {
  PackRowsArgs a = {};
  if (n < 1 || n > 3) return hipErrorInvalidValue;
  a.T = T;
  a.D = D;
  a.pieces = (D + 7) / 8;
  // Tokens of a workgroup: one, so that small calls have enough workgroups, or eight,
  // which keep its threads busy. One / eight, with the forward behind it (sequences of
  // 32), us: 12:4 x 159 64 tokens 9.3 / 11.3, 1024 17.2 / 18.6, 2048 27.4 / 26.7, 4096
  // 40.8 / 39.5; 2:1 x 53 64 6.9 / 6.8, 1024 8.6 / 7.9, 4096 15.3 / 12.4.
  a.per = T >= 2048 ? 8 : 1;
  for (int i = 0; i < n; ++i) {
    a.src[i] = (const uint16_t*)src[i];
    a.dst[i] = (uint16_t*)dst[i];
    a.st[i] = strides[2 * i];
    a.sh[i] = strides[2 * i + 1];
    a.heads[i] = heads[i];
  }
  const int64_t blocks = (T + a.per - 1) / a.per;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  pack_rows_kernel<<<dim3((uint32_t)blocks, n), dim3(256), 0, stream>>>(a);
  HIP_CHECK_LAST();
  return hipSuccess;
}
