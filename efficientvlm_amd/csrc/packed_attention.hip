// Attention over packed sequences for gfx950: the queries of many sequences laid end to end, their keys likewise (or in the
// slots of a cache), heads in groups that share a key head, forward and backward, f32 and bf16.
//
//   row = one (query token, head).  Query i of a sequence with n queries and m keys sees the keys  j < vis(i),
//   vis(i) = m  or, causal,  m - n + i + 1  (the last query sees every key: a prompt, a chunk behind a cache and a single
//   new token are the same formula).
//   s_j = scale q.k_j,  p_j = 2^(s_j log2e - lse),  lse = log2 sum_j 2^(s_j log2e),  O = sum_j p_j v_j
//   dP_j = dO.v_j,  delta = dO.O = sum_j p_j dP_j,  dS_j = p_j (dP_j - delta)
//   dQ = scale sum_j dS_j k_j,   dK_j = scale sum_rows dS_j q,   dV_j = sum_rows p_j dO   (rows of every head of the group)
//   A row that sees no key has O = 0 and adds nothing to any gradient.
//   A row whose largest score m is far from zero, |m c| > 2^10 with c = scale log2e, has its exponents formed as (s_j - m) c - log2 sum_j
//   2^((s_j - m) c) instead: s_j c - lse would carry the rounding of m c or of lse, half a unit of numbers of that size.  (Scores of
//   3e5: probabilities of the backward pass 1 % off; from 3e9 on out of f32's range, NaN.  Up to 2^10 it is 2^-15.)
//
// All four products of a step are built from two wave-level forms over 32 x 32 blocks:
//   row_mm   C[r][c] = sum_d tile[r][d] col[c][d]     tile rows from LDS, columns held in registers for the whole loop
//   col_mm   acc[d][c] += sum_r tile[r][d] P[r][c]    the C of the first product IS the B operand of the second one (the
//            k-slots of both operands are assigned alike, so P never moves between lanes); bf16 tiles are read by columns
//            with the transposing LDS reads, f32 tiles with plain ones
// Forward and dQ hold 32 rows of Q (and dO) as columns and stream keys; dK / dV hold 32 keys as columns and stream rows.
// A softmax row then lies in two lanes: the running maximum costs one shuffle per block, the sum one at the end.
//
// Rows are packed: the gp heads of a group (the largest divisor of the group <= 32) of consecutive tokens fill a block of
// 32 rows, so one pass over the keys serves all heads that share them - also for a single token.
//
// A sequence's blocks are found on the device (find_tile): nothing about the lengths is known to the host, no copy back,
// and lengths may change between replays of a captured launch.  Every length and start is clamped to the tensors, so no
// content of cu_q / cu_k / k_lens can make a kernel leave them.  Everything is summed in a fixed order in f32: no atomics.
#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
#define PK_LOG2E 1.44269504088896341f
#define PK_FAR 1024.0f

struct PkArgs {
  const void *Q, *K, *V, *O, *dO;
  void *out, *out_lo, *dQ, *dK, *dV;
  const int32_t *cu_q, *cu_k, *k_lens;
  float *lse, *delta, *part;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, do_tok, do_head, dq_tok, dq_head, dk_tok, dk_head, dv_tok, dv_head;
  int Tq, Tk, S, H, G, dh;          // G = heads per key head
  int gp, chunks, units;            // heads packed into a row block, chunks of a group, chunks * key heads
  int per, tiles;                   // tokens (keys) of a block, grid tiles
  int far;                          // lse has a second plane, for the rows far from zero
  int splits, causal;               // splits: parts of the rows of a key block (dK / dV)
  int want;                         // chunks of keys aimed at for one chunk of heads (forward, few rows)
  unsigned inv_gp;                  // 2^16 / gp rounded up: r / gp = r * inv_gp >> 16 for r < 256
  float scale, c;                   // c = scale * log2e
};

// ---- 16-byte fragments ----------------------------------------------------------------------
template <typename T> struct Frag;
template <> struct Frag<bf16> { typedef bf16x8 type; };
template <> struct Frag<float> { typedef f32x4 type; };

__device__ __forceinline__ f32x16 mma(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const f32x4& a, const f32x4& b, f32x16 c) {      // 8 of the k-dimension: 4 products of 2
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// LDS addresses as numbers: all pieces of a row, and all column blocks of 4 rows, lie at base ^ (constant).  The compiler keeps a
// register for each of them; a LEAN kernel makes the base opaque where it is used, so that the few exclusive-ors are done again
// in every iteration.  (dK / dV at head dim 128 fits two waves a SIMD only so; the forward pass lost 7 % by it.)
typedef __attribute__((address_space(3))) const char* lds_ptr;
__device__ __forceinline__ uint32_t lds_of(const char* p) { return (uint32_t)(uintptr_t)(lds_ptr)p; }
template <bool LEAN> __device__ __forceinline__ uint32_t base_of(uint32_t x) {
  if (LEAN) asm volatile("" : "+v"(x));
  return x;
}
template <typename F> __device__ __forceinline__ F lds_read(uint32_t at) { return *(__attribute__((address_space(3))) const F*)(uintptr_t)at; }

// Row-major LDS tile [rows][D], 16-byte pieces of a row permuted so that neither the row reads (16 rows, one piece each) nor
// the column reads (4 consecutive rows, 4 consecutive pieces each) of a half-wave meet in one of the 16 piece-wide bank groups:
// the two low row bits move groups of 4 pieces, the next two the pieces within a group (128-byte rows: two rows share the
// bank groups, the lowest row bit selects the half).  SQ_LDS_BANK_CONFLICT: 0.
template <typename T, int D> struct Tile {
  typedef typename Frag<T>::type frag;
  static constexpr int RB = D * (int)sizeof(T), NC = RB / 16, NS = RB / 32, EP = 16 / (int)sizeof(T);
  static __device__ __forceinline__ int at(int row, int c) {
    const int x = NC == 8 ? ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)) : (((row & 3) << 2) | ((row >> 2) & 3));
    return row * RB + (c ^ x) * 16;
  }
  // 32 rows as columns of a product: lane -> row lane & 31, pieces 2s + (lane >> 5); null row: zeros
  static __device__ __forceinline__ void load_cols(const T* row, int dh, int hh, frag (&f)[NS]) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      f[s] = frag{};
      const int e = (2 * s + hh) * EP;
      if (row && e < dh) f[s] = *reinterpret_cast<const frag*>(row + e);
    }
  }
  // order of a product's LDS reads and MFMAs: the reads of the next two steps on their way before a step's products.  (Left alone, the
  // compiler reuses one step's registers and waits for every read; most of that wait is hidden by the SIMD's other wave.  Left alone,
  // one, two, three steps: the documents below, both directions, 777, 767, 762, 773 us; the prompts' forward 899, 900, 889, 893.)
  template <int READS, int N> static __device__ __forceinline__ void ahead() {
    constexpr int AHEAD = 2;
    if constexpr (sizeof(T) == 2) {
      __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
      for (int s = 0; s < NS - AHEAD; ++s) {
        __builtin_amdgcn_sched_group_barrier(0x008, N, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * N, 0);
    }
  }
  template <bool LEAN = false> static __device__ __forceinline__ f32x16 row_mm(const char* tile, int r0, const frag (&b)[NS], int lane) {
    f32x16 acc = {};
    const uint32_t base = base_of<LEAN>(lds_of(tile) + at(r0 + (lane & 31), lane >> 5));
#pragma unroll
    for (int s = 0; s < NS; ++s) acc = mma(lds_read<frag>(base ^ (32 * s)), b[s], acc);
    ahead<1, 1>();
    return acc;
  }
  // columns from LDS as well (32 rows of another tile)
  static __device__ __forceinline__ f32x16 row_mm(const char* tile, int r0, const char* cols, int c0, int lane) {
    f32x16 acc = {};
    const uint32_t rows = base_of<true>(lds_of(tile) + at(r0 + (lane & 31), lane >> 5)), col = base_of<true>(lds_of(cols) + at(c0 + (lane & 31), lane >> 5));
#pragma unroll
    for (int s = 0; s < NS; ++s) acc = mma(lds_read<frag>(rows ^ (32 * s)), lds_read<frag>(col ^ (32 * s)), acc);
    ahead<2, 1>();
    return acc;
  }
  // NB blocks of 32 rows against the same columns
  template <int NB> static __device__ __forceinline__ void rows_mm(const char* tile, const frag (&b)[NS], f32x16 (&acc)[NB], int lane) {
    const uint32_t base = lds_of(tile) + at(lane & 31, lane >> 5);
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[n] = f32x16{};
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[n] = mma(lds_read<frag>((base ^ (32 * s)) + 32 * n * RB), b[s], acc[n]);
    ahead<NB, NB>();
  }
};

// acc[d][c] += sum_r tile[r][d] p[r][c]
// bf16: register i of C holds tile row 8 (i >> 2) + 4 (lane >> 5) + (i & 3); registers 8kk .. 8kk + 7 are the B operand of k-step
// kk, and the A operand takes its 8 rows in that order: two transposing reads of 4 rows x 16 columns each
template <int D, bool LEAN = false> __device__ __forceinline__ void col_mm(const bf16*, const char* tile, int r0, const f32x16& p, f32x16 (&acc)[D / 32], int lane) {
  typedef Tile<bf16, D> TL;
  const int hh = lane >> 5, w = lane & 15, sub = (lane >> 4) & 1;
  const uint32_t base = base_of<LEAN>(lds_of(tile) + TL::at(r0 + 4 * hh + (w >> 2), sub * 2 + ((w & 3) >> 1)) + (w & 1) * 8);
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
    bf16x8 b;
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = (bf16)p[8 * kk + j];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      bf16x8 a;
#pragma unroll
      for (int half = 0; half < 2; ++half) {                 // rows r0 + 16 kk + 8 half + 4 (lane >> 5) .. + 3, columns 32 dt ..
        const bf16x4 t = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (bf16x4 __attribute__((address_space(3)))*)(uintptr_t)((base ^ (64 * dt + 32 * half)) + (16 * kk + 8 * half) * TL::RB));
        a[4 * half + 0] = t[0]; a[4 * half + 1] = t[1]; a[4 * half + 2] = t[2]; a[4 * half + 3] = t[3];
      }
      acc[dt] = mma(a, b, acc[dt]);
    }
  }
}
template <int D, bool LEAN = false> __device__ __forceinline__ void col_mm(const float*, const char* tile, int r0, const f32x16& p, f32x16 (&acc)[D / 32], int lane) {
  const int hh = lane >> 5, w = lane & 31;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = r0 + 8 * (i >> 2) + 4 * hh + (i & 3);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      const int e = dt * 32 + w;
      const float v = *reinterpret_cast<const float*>(tile + Tile<float, D>::at(row, e >> 2) + (e & 3) * 4);
      acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[i], acc[dt], 0, 0, 0);
    }
  }
}
// C register -> row of the 32-row block
__device__ __forceinline__ int c_row(int i, int hh) { return 8 * (i >> 2) + 4 * hh + (i & 3); }

// ---- sequences ------------------------------------------------------------------------------
struct Seq { int qs, qlen, ks, klen; };
__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }
__device__ __forceinline__ Seq load_seq(const PkArgs& a, int s) {
  Seq q;
  q.qs = clampi(a.cu_q[s], 0, a.Tq);
  q.qlen = clampi(a.cu_q[s + 1], q.qs, a.Tq) - q.qs;
  q.ks = clampi(a.cu_k[s], 0, a.Tk);
  q.klen = clampi(a.cu_k[s + 1], q.ks, a.Tk) - q.ks;
  if (a.k_lens) q.klen = clampi(a.k_lens[s], 0, q.klen);
  return q;
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
__device__ __forceinline__ Seq uniform(const Seq& x) {       // what every lane holds alike, in scalar registers
  return Seq{__builtin_amdgcn_readfirstlane(x.qs), __builtin_amdgcn_readfirstlane(x.qlen), __builtin_amdgcn_readfirstlane(x.ks),
             __builtin_amdgcn_readfirstlane(x.klen)};
}
__device__ __forceinline__ int vis_of(const PkArgs& a, const Seq& q, int tok) {
  return a.causal ? clampi(q.klen - q.qlen + tok + 1, 0, q.klen) : q.klen;
}
// ... one sequence after the other: every wave counts 64 E of them at a time, E a lane (24 tokens a sequence, 680 sequences, forward at
// heads 16/4, dim 128: E = 4 92 us, E = 1 106 us; 65 sequences of 250: backward 114 and 107 us)
template <bool KEYS, int E> __device__ __forceinline__ bool find_in_order(const PkArgs& a, int t, Seq& q, int& i, int& over, int& total) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int s0 = 0; s0 < a.S; s0 += 64 * E) {
    int n[E];
    int64_t mine = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int s = s0 + E * lane + j;
      n[j] = 0;
      if (s < a.S) {
        const Seq x = load_seq(a, s);
        n[j] = ((KEYS ? x.klen : x.qlen) + a.per - 1) / a.per;
      }
      mine += n[j];
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t up = __shfl_up(incl, o, 64);
      if (lane >= o) incl += up;
    }
    const unsigned long long hit = __ballot(before + incl > t);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      int64_t left = t - (before + incl - mine);             // (of the lane that has it: the block's index among the lane's)
      int j = 0;
#pragma unroll
      for (int e = 0; e < E - 1; ++e)
        if (j == e && left >= n[e]) { left -= n[e]; j = e + 1; }
      q = uniform(load_seq(a, s0 + E * l + __shfl(j, l, 64)));
      i = __builtin_amdgcn_readfirstlane(__shfl((int)left, l, 64));
      return true;
    }
    before += __shfl(incl, 63, 64);
  }
  over = (int)(t - before);
  total = (int)before;
  return false;
}
// Block t of all sequences' blocks (KEYS: of their keys): the sequence it belongs to and its index there.  False: t lies behind the last
// block (t - total in `over`), the block has nothing to do but the rows outside all sequences.  Up to 64 causal sequences are taken
// longest blocks first - the j-th block of queries, or the j-th block of keys from the end, of every sequence that has one, j
// descending - so that the chip does not end on a few long blocks; of more sequences, one after the other.
template <bool KEYS> __device__ __forceinline__ bool find_tile(const PkArgs& a, int t, Seq& q, int& i, int& over, int& total) {
  const int lane = threadIdx.x & 63;
  if (a.causal && a.S <= 64) {
    int n = 0;
    if (lane < a.S) {
      const Seq x = load_seq(a, lane);
      n = ((KEYS ? x.klen : x.qlen) + a.per - 1) / a.per;
    }
    auto from = [&](int j) {                                 // blocks of a level >= j
      int64_t f = max(0, n - j);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) f += __shfl_xor(f, o, 64);
      return f;
    };
    int lo = 0, hi = n;                                      // level: the largest j with from(j) > t
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) hi = max(hi, __shfl_xor(hi, o, 64));
    const int64_t all = from(0);
    if (t >= all) { over = (int)(t - all); total = (int)all; return false; }
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (from(mid) > t) lo = mid; else hi = mid;
    }
    int64_t rank = t - from(lo + 1);
    unsigned long long has = __ballot(n > lo);
    for (; rank > 0; --rank) has &= has - 1;
    const int s = __builtin_ctzll(has);
    q = uniform(load_seq(a, s));
    i = __builtin_amdgcn_readfirstlane(KEYS ? __shfl(n, s, 64) - 1 - lo : lo);
    return true;
  }
  return a.S > 128 ? find_in_order<KEYS, 4>(a, t, q, i, over, total) : find_in_order<KEYS, 1>(a, t, q, i, over, total);
}
// Few rows, many keys: the keys of every (sequence, block of tokens) are cut into chunks of one length for all, so that blocks of equal
// work fill the chip however different the sequences are.  The length follows from the sequences themselves: their keys
// (once for each block of tokens) over the number of chunks that is wanted, a multiple of 32, at least PK_CHUNK.
#define PK_CHUNK 256
struct Chunk { Seq q; int tile, chunk, n, keys; int64_t first; };       // `first`: index of the tile's first chunk among all
__device__ __forceinline__ int chunks_of(const PkArgs& a, const Seq& x, int keys) { return max(1, (x.klen + keys - 1) / keys); }
// the chunk with index g (BY_TOKEN: the first chunk of the block that holds token g); false: there is none
template <bool BY_TOKEN> __device__ __forceinline__ bool find_chunk(const PkArgs& a, int g, Chunk& c) {
  const int lane = threadIdx.x & 63;
  int64_t work = 0;
  for (int s = lane; s < a.S; s += 64) {
    const Seq x = load_seq(a, s);
    work += (int64_t)((x.qlen + a.per - 1) / a.per) * x.klen;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) work += __shfl_xor(work, o, 64);
  const int64_t even = ((work + a.want - 1) / a.want + 31) / 32 * 32;
  const int keys = even < PK_CHUNK ? PK_CHUNK : (even > (1 << 30) ? 1 << 30 : (int)even);
  int64_t before = 0;
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    Seq x = {0, 0, 0, 0};
    int64_t n = 0;
    if (s0 + lane < a.S) {
      x = load_seq(a, s0 + lane);
      n = (int64_t)((x.qlen + a.per - 1) / a.per) * chunks_of(a, x, keys);
    }
    int64_t incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t up = __shfl_up(incl, o, 64);
      if (lane >= o) incl += up;
    }
    const unsigned long long hit = __ballot(BY_TOKEN ? (g >= x.qs && g - x.qs < x.qlen) : before + incl > g);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int64_t first = before + __shfl(incl - n, l, 64);
      c.q = uniform(load_seq(a, s0 + l));
      c.n = __builtin_amdgcn_readfirstlane(chunks_of(a, c.q, keys));
      c.keys = __builtin_amdgcn_readfirstlane(keys);
      const int64_t rest = BY_TOKEN ? (int64_t)((g - c.q.qs) / a.per) * c.n : g - first;
      c.tile = __builtin_amdgcn_readfirstlane((int)(rest / c.n));
      c.chunk = __builtin_amdgcn_readfirstlane((int)(rest % c.n));
      c.first = uniform64(first + rest - rest % c.n);
      return true;
    }
    before += __shfl(incl, 63, 64);
  }
  return false;
}
// rows outside all sequences ([0, first start), [last end, T)): zeros.  `per_row(row)` by every wave of the surplus blocks
template <typename F> __device__ __forceinline__ void outside_rows(const int32_t* cu, int S, int T, int index, int count, F per_row) {
  const int head = S > 0 ? clampi(cu[0], 0, T) : T, tail = S > 0 ? clampi(cu[S], 0, T) : T;
  const int wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  const int n = head + (T - tail);
  for (int64_t r = (int64_t)index * nw + wave; r < n; r += (int64_t)count * nw) per_row(r < head ? (int)r : tail + (int)(r - head));
}

// ---- staging: `ROWS` rows of a [token][head][dh] tensor -> LDS tile, in two halves (load into registers, store into LDS) ----
template <typename T, int D, int ROWS, int NT> struct Stage {
  typedef Tile<T, D> TL;
  static constexpr int N = ROWS * TL::NC / NT;
  static_assert(ROWS * TL::NC % NT == 0, "whole pieces per thread");
  typename TL::frag v[N];
  // (no branch around a load: pieces behind the head dim read the row's first piece and are zeroed in registers)
  __device__ __forceinline__ void pad(int dh, int tid) {
    if (dh == D) return;
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (((tid + k * NT) % TL::NC) * TL::EP >= dh) v[k] = typename TL::frag{};
  }
  // rows first .. first + ROWS - 1 of `base` (row stride `stride` elements, everything the same in all lanes): a scalar address for
  // each piece plus one 32-bit offset of the thread.  Rows >= n repeat row n - 1 (their scores are masked)
  __device__ __forceinline__ void load(const T* base, int64_t stride, int first, int n, int dh, int tid) {
    constexpr int RP = NT / TL::NC;                          // rows of one piece of the block
    const int r = tid / TL::NC, e0 = (tid % TL::NC) * TL::EP, e = e0 < dh ? e0 : 0;
    if (first + ROWS <= n) {
      const uint32_t off = (uint32_t)(r * (int)stride + e) * (uint32_t)sizeof(T);
#pragma unroll
      for (int k = 0; k < N; ++k)
        v[k] = *reinterpret_cast<const typename TL::frag*>((const char*)(base + (int64_t)(first + k * RP) * stride) + off);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
        v[k] = *reinterpret_cast<const typename TL::frag*>(base + min(first + k * RP + r, n - 1) * stride + e);
    }
  }
  // packed rows: row r = (token first + r / gp, head r % gp); rows behind the last token repeat it, unused rows are those of the
  // tokens that follow (the row's lse of +inf makes its probabilities zero).  Where gp divides the rows of a piece, every piece
  // is a scalar address plus the thread's one offset
  __device__ __forceinline__ void load_rows(const T* base, int64_t tok_stride, int64_t head_stride, int first, int qlen, int gp,
                                            unsigned inv_gp, int dh, int tid) {
    constexpr int RP = NT / TL::NC;
    const int r0 = tid / TL::NC, e0 = (tid % TL::NC) * TL::EP, e = e0 < dh ? e0 : 0;
    if ((gp & (gp - 1)) == 0 && gp <= RP && first + (int)((ROWS - 1) * inv_gp >> 16) < qlen) {
      const int rt = (int)(r0 * inv_gp >> 16), step = (int)(RP * inv_gp >> 16);
      const uint32_t off = (uint32_t)(rt * (int)tok_stride + (r0 - rt * gp) * (int)head_stride + e) * (uint32_t)sizeof(T);
#pragma unroll
      for (int k = 0; k < N; ++k)
        v[k] = *reinterpret_cast<const typename TL::frag*>((const char*)(base + (int64_t)(first + k * step) * tok_stride) + off);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int r = r0 + k * RP, rt = (int)(r * inv_gp >> 16), tok = min(first + rt, qlen - 1);
        v[k] = *reinterpret_cast<const typename TL::frag*>(base + tok * tok_stride + (r - rt * gp) * head_stride + e);
      }
    }
  }
  __device__ __forceinline__ void store(char* tile, int tid) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int id = tid + k * NT;
      *reinterpret_cast<typename TL::frag*>(tile + TL::at(id / TL::NC, id % TL::NC)) = v[k];
    }
  }
};

// one block of NB * 32 keys for 32 rows: scores, running maximum, probabilities, context.  m is kept as a raw score; it follows
// the true maximum only when that has grown by more than 2^8 (p then stays <= 2^8, far from any overflow of the f32 sums, and
// bf16 keeps the same relative precision), so the rescaling of the context is rare.  p is rounded to bf16 for the second
// product (its sum is not): half a step, 2^-8 relative to each p (a product in f32 has a sixteenth of the rate, p as a sum of two bf16
// would cost it twice).  The backward pass rounds p and dS = p (dP - delta) likewise, as operands of dV, dK and dQ.  The products of inputs that are bf16 already
// are exact in f32, so these are the only roundings beside the outputs': errors against 64 bits are 1.1 - 1.5 x those of a form in
// f32 that rounds its outputs alone (1.1 for short rows, whose p are few; 1.5 for the gradients of short sequences).
template <typename T, int D, int NB>
__device__ __forceinline__ void attend(const char* Ks, const char* Vs, int kt0, int vis, bool mask,
                                       const typename Frag<T>::type (&qf)[Tile<T, D>::NS], float c, float& m, float& l,
                                       f32x16 (&o)[D / 32], int lane) {
  const int hh = lane >> 5;
  f32x16 s[NB];
  Tile<T, D>::template rows_mm<NB>(Ks, qf, s, lane);
  if (mask) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = kt0 + 32 * b + c_row(i, hh) < vis ? s[b][i] : -INFINITY;
  }
  float mx = s[0][0];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
  const float mn = fmaxf(m, mx);
  float mc = m == -INFINITY ? 0.f : m * c;
  if (__any((mn - m) * c > 8.0f || fabsf(mc) > PK_FAR)) {
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * c);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
    mc = m == -INFINITY ? 0.f : m * c;
    if (__any(fabsf(mc) > PK_FAR)) {
      const float base = fabsf(mc) > PK_FAR ? m : 0.f;
      mc = fabsf(mc) > PK_FAR ? 0.f : mc;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][i] -= base;
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], c, -mc));
      l += s[b][i];
    }
    col_mm<D>((const T*)nullptr, Vs, 32 * b, s[b], o, lane);
  }
}

// context / gradient of 32 rows held transposed (lane -> row, registers -> head dim), times `mul`
template <typename T, int D> __device__ __forceinline__ void store_cols(T* row, int dh, const f32x16 (&o)[D / 32], float mul, int hh) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = dt * 32 + 8 * j + 4 * hh;
      if (d < dh) {
        const float v[4] = {o[dt][4 * j] * mul, o[dt][4 * j + 1] * mul, o[dt][4 * j + 2] * mul, o[dt][4 * j + 3] * mul};
        Vec4<T>::store(row + d, v);
      }
    }
}
// ... and what the rounding to bf16 took from it, in bf16 as well: O = out + out_lo to 2^-17
template <typename T, int D> __device__ __forceinline__ void store_rest(T* row, int dh, const f32x16 (&o)[D / 32], float mul, int hh) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = dt * 32 + 8 * j + 4 * hh;
      if (d < dh) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) { const float x = mul_rn(o[dt][4 * j + e], mul); v[e] = x - to_f(from_f<T>(x)); }
        Vec4<T>::store(row + d, v);
      }
    }
}
// a row's log-sum-exp for the backward pass, from its maximum and its sum relative to it.  A row far from zero keeps its maximum in the
// second plane, and the log of that sum so that it shows: (log + 1) 2^100, where the others are at most 2^11
__device__ __forceinline__ void store_lse(const PkArgs& a, int h, int64_t t, float m, float l, int vis) {
  const int64_t at = (int64_t)h * a.Tq + t;
  const float logl = __builtin_amdgcn_logf(l);
  const bool far = a.far && vis > 0 && fabsf(m * a.c) > PK_FAR;
  a.lse[at] = vis > 0 ? (far ? (logl + 1.0f) * 0x1p100f : fmaf(m, a.c, logl)) : INFINITY;
  if (far) a.lse[(int64_t)a.H * a.Tq + at] = m;
}
// ... read: the maximum of a row far from zero (and its lse relative to it), 0 for any other
__device__ __forceinline__ float far_base(const PkArgs& a, int64_t at, float& lse) {
  if (!(a.far && fabsf(lse) > 0x1p64f && fabsf(lse) < INFINITY)) return 0.f;
  lse = lse * 0x1p-100f - 1.0f;
  return a.lse[(int64_t)a.H * a.Tq + at];
}
template <typename T> __device__ __forceinline__ void zero_row(T* row, int dh) {
  for (int d = threadIdx.x & 63; d < dh; d += 64) row[d] = from_f<T>(0.f);
}

// the surplus blocks of a launch over query blocks: rows outside all sequences are zero
template <typename T> __device__ __forceinline__ void fwd_outside(const PkArgs& a, int h0, int over, int total) {
  outside_rows(a.cu_q, a.S, a.Tq, over, a.tiles - total, [&](int r) {
    for (int h = h0; h < h0 + a.gp; ++h) {
      zero_row<T>((T*)a.out + ((int64_t)r * a.H + h) * a.dh, a.dh);
      if (a.lse && (threadIdx.x & 63) == 0) a.lse[(int64_t)h * a.Tq + r] = INFINITY;
    }
  });
}

// ---------------------------------------------------------------------------------------------
// forward, rows split over the waves: NW * 32 rows of one (sequence, chunk of heads), keys in shared blocks of BN.
// 6 causal sequences of 1 653 - 4 965 (22 492 tokens), heads 32/8 of 128, bf16: 890 us = 0.89 PF/s.  No unit is the bound by itself: MFMA are busy
// 39 % of the cycles, vector instructions 40 % (1.8 - 1.9 GHz); of the waves' cycles 21 % wait for memory, LDS and barriers, 41 % for their
// turn to issue.  Within a wave the exponentials of its scores wait for the product and the next product for them, and two waves a
// SIMD overlap that in part: a loop without the maximum, a quarter fewer vector instructions, took the same time, so it is the
// chain and not the instructions' number.  Two blocks of 64 keys in flight a wave spilled: 1 075 us.
// ---------------------------------------------------------------------------------------------
template <typename T, int D, int NW, int BN>
__global__ __launch_bounds__(64 * NW, sizeof(T) * D == 512 ? 1 : 2) void pk_fwd_rows_kernel(PkArgs a) {
  typedef Tile<T, D> TL;
  __shared__ __attribute__((aligned(512))) char sm[2 * BN * TL::RB];
  char *Ks = sm, *Vs = sm + BN * TL::RB;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const int unit = blockIdx.x % a.units, kh = unit / a.chunks, h0 = kh * a.G + (unit % a.chunks) * a.gp;
  Seq q; int ti, over, total;
  if (!find_tile<false>(a, blockIdx.x / a.units, q, ti, over, total)) { fwd_outside<T>(a, h0, over, total); return; }
  const int r = wave * 32 + (lane & 31), tok0 = ti * a.per, tok = tok0 + r / a.gp, h = h0 + r % a.gp;
  const bool valid = r < a.per * a.gp && tok < q.qlen;
  const int vis = valid ? vis_of(a, q, tok) : 0;
  const int last = min(tok0 + a.per, q.qlen) - 1;
  const int nk = vis_of(a, q, last);                                                    // keys any row of the block sees
  const int w_lo = tok0 + (int)(wave * 32 * a.inv_gp >> 16), w_hi = tok0 + (int)((wave * 32 + 31) * a.inv_gp >> 16);      // the wave's tokens
  const int w_min = vis_of(a, q, min(w_lo, last)), w_max = vis_of(a, q, min(w_hi, last));
  const bool w_any = w_lo <= last;
  typename TL::frag qf[TL::NS];
  TL::load_cols(valid ? (const T*)a.Q + (q.qs + tok) * a.q_tok + h * a.q_head : nullptr, a.dh, hh, qf);
  const T* Kb = (const T*)a.K + q.ks * a.k_tok + kh * a.k_head;
  const T* Vb = (const T*)a.V + q.ks * a.v_tok + kh * a.v_head;
  float m = -INFINITY, l = 0.f;
  f32x16 o[D / 32] = {};
  Stage<T, D, BN, 64 * NW> ks, vs;
  if (nk > 0) { ks.load(Kb, a.k_tok, 0, q.klen, a.dh, tid); vs.load(Vb, a.v_tok, 0, q.klen, a.dh, tid); }
  for (int kt = 0; kt < nk; kt += BN) {
    __syncthreads();
    ks.pad(a.dh, tid); vs.pad(a.dh, tid);
    ks.store(Ks, tid); vs.store(Vs, tid);
    __syncthreads();
    if (kt + BN < nk) { ks.load(Kb, a.k_tok, kt + BN, q.klen, a.dh, tid); vs.load(Vb, a.v_tok, kt + BN, q.klen, a.dh, tid); }
    if (w_any && kt < w_max) attend<T, D, BN / 32>(Ks, Vs, kt, vis, kt + BN > w_min, qf, a.c, m, l, o, lane);
  }
  l += __shfl_xor(l, 32, 64);
  if (!valid) return;
  const int64_t t = q.qs + tok;
  const float inv = vis > 0 ? 1.0f / l : 0.f;
  store_cols<T, D>((T*)a.out + (t * a.H + h) * a.dh, a.dh, o, inv, hh);
  if (sizeof(T) == 2 && a.out_lo) store_rest<T, D>((T*)a.out_lo + (t * a.H + h) * a.dh, a.dh, o, inv, hh);
  if (a.lse && hh == 0) store_lse(a, h, t, m, l, vis);
}

// ---------------------------------------------------------------------------------------------
// forward, keys split over the waves: 32 rows of one (sequence, chunk of heads) - single tokens and very short sequences, where
// there are too few rows to fill a block of waves but perhaps many keys.  Every wave walks its own 32-key blocks through its own
// LDS tile (no barrier in the loop) and the waves' sums are joined at the end.  CH: a block takes one chunk of the keys (find_chunk)
// and leaves its part for pk_join_kernel, unless the chunk is all there is.
// Bound by HBM for long caches: 12 single tokens on 6 000 - 40 000 keys, heads 32/8 of 128, bf16: 652 MB in 126 us (5.2 TB/s) and 10 us
// for the join; by one block's chain of loads for short ones (24 on 6 - 40 keys, 12 heads of 64: 6.8 us).
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// part of chunk g, chunk of heads `unit`: 32 x dh context (not divided by the sum), then 32 x (maximum, sum)
__device__ __forceinline__ float* part_of(const PkArgs& a, int64_t g, int unit) {
  return a.part + (g * a.units + unit) * (32 * (a.dh + 2));
}
template <typename T, int D, int NW, bool CH>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 ? 1 : 2) void pk_fwd_keys_kernel(PkArgs a) {
  typedef Tile<T, D> TL;
  constexpr int WB = 2 * 32 * TL::RB > 32 * D * 4 ? 2 * 32 * TL::RB : 32 * D * 4;       // one wave's tiles, later its context
  __shared__ __attribute__((aligned(512))) char sm[NW * WB];
  __shared__ float sml[NW][2][32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const int unit = blockIdx.x % a.units, kh = unit / a.chunks, h0 = kh * a.G + (unit % a.chunks) * a.gp, g = blockIdx.x / a.units;
  Seq q; int ti;
  Chunk c;
  if constexpr (CH) {
    if (!find_chunk<false>(a, g, c)) return;                 // (rows outside all sequences: pk_join_kernel)
    q = c.q; ti = c.tile;
  } else {
    int over, total;
    if (!find_tile<false>(a, g, q, ti, over, total)) { fwd_outside<T>(a, h0, over, total); return; }
  }
  const int r = lane & 31, tok0 = ti * a.per, tok = tok0 + r / a.gp, h = h0 + r % a.gp;
  const bool valid = r < a.per * a.gp && tok < q.qlen;
  const int vis = valid ? vis_of(a, q, tok) : 0;
  const int last = min(tok0 + a.per, q.qlen) - 1;
  const int nk = vis_of(a, q, last), w_min = vis_of(a, q, tok0);
  const int nb = (nk + 31) / 32, b0 = CH ? c.chunk * (c.keys / 32) : 0, b1 = CH ? min(nb, b0 + c.keys / 32) : nb;   // 32-key blocks
  char* Ks = sm + wave * WB;
  char* Vs = Ks + 32 * TL::RB;
  typename TL::frag qf[TL::NS];
  TL::load_cols(valid ? (const T*)a.Q + (q.qs + tok) * a.q_tok + h * a.q_head : nullptr, a.dh, hh, qf);
  const T* Kb = (const T*)a.K + q.ks * a.k_tok + kh * a.k_head;
  const T* Vb = (const T*)a.V + q.ks * a.v_tok + kh * a.v_head;
  float m = -INFINITY, l = 0.f;
  f32x16 o[D / 32] = {};
  Stage<T, D, 32, 64> ks, vs;
  int kb = b0 + wave;
  if (kb < b1) { ks.load(Kb, a.k_tok, kb * 32, q.klen, a.dh, lane); vs.load(Vb, a.v_tok, kb * 32, q.klen, a.dh, lane); }
  for (; kb < b1; kb += NW) {
    wave_lds_fence();
    ks.pad(a.dh, lane); vs.pad(a.dh, lane);
    ks.store(Ks, lane); vs.store(Vs, lane);
    wave_lds_fence();
    if (kb + NW < b1) {
      ks.load(Kb, a.k_tok, (kb + NW) * 32, q.klen, a.dh, lane);
      vs.load(Vb, a.v_tok, (kb + NW) * 32, q.klen, a.dh, lane);
    }
    attend<T, D, 1>(Ks, Vs, kb * 32, vis, kb * 32 + 32 > w_min, qf, a.c, m, l, o, lane);
  }
  l += __shfl_xor(l, 32, 64);
  const int64_t t = q.qs + tok;
  if constexpr (NW > 1) {
    // join the waves: wave w sums the row block's columns d = w * D / NW .. of every wave, rescaled to the common maximum
    wave_lds_fence();
    float* mine = (float*)(sm + wave * WB);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[(dt * 32 + c_row(i, hh)) * 32 + r] = o[dt][i];
    if (hh == 0) { sml[wave][0][r] = m; sml[wave][1][r] = l; }
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[w][0][r]);
    float L = 0.f, f[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = sml[w][0][r];
      f[w] = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - M) * a.c);
      L += sml[w][1][r] * f[w];
    }
    if (!valid) return;
    const bool whole = !CH || c.n == 1;
    const float inv = vis > 0 ? 1.0f / L : 0.f;
    float* part = CH ? part_of(a, c.first + c.chunk, unit) : nullptr;
    // thread -> (row r, 4 consecutive d): the 2 NW half-waves take them in turn
    for (int d = (wave * 2 + hh) * 4; d < a.dh; d += NW * 8) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = fmaf(((float*)(sm + w * WB))[(d + j) * 32 + r], f[w], v[j]);
      if (!whole) {
        Vec4<float>::store(part + r * a.dh + d, v);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] *= inv;
        Vec4<T>::store((T*)a.out + (t * a.H + h) * a.dh + d, v);
        if (sizeof(T) == 2 && a.out_lo) {
          float lo[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) lo[j] = v[j] - to_f(from_f<T>(v[j]));
          Vec4<T>::store((T*)a.out_lo + (t * a.H + h) * a.dh + d, lo);
        }
      }
    }
    if (wave == 0 && hh == 0) {
      if (!whole) {
        part[32 * a.dh + 2 * r] = M; part[32 * a.dh + 2 * r + 1] = L;
      } else if (a.lse) {
        store_lse(a, h, t, M, L, vis);
      }
    }
  } else {
    if (!valid) return;
    const float inv = vis > 0 ? 1.0f / l : 0.f;
    store_cols<T, D>((T*)a.out + (t * a.H + h) * a.dh, a.dh, o, inv, hh);
    if (sizeof(T) == 2 && a.out_lo) store_rest<T, D>((T*)a.out_lo + (t * a.H + h) * a.dh, a.dh, o, inv, hh);
    if (a.lse && hh == 0) store_lse(a, h, t, m, l, vis);
  }
}

// v += f_i part_i for N parts, all on their way at a time (of the parts behind n the last is read again, their f is 0)
template <int N> __device__ __forceinline__ void join_parts(const float* p, int64_t next, int n, unsigned d0, unsigned d1, float f, int i0, float& v0, float& v1) {
  float x0[N], x1[N];
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const float* pi = p + min(u, n - 1) * next;
    x0[u] = pi[d0]; x1[u] = pi[d1];
  }
#pragma unroll
  for (int u = 0; u < N; ++u) {
    const float fi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), (i0 + u) & 63));      // (0 in the lanes behind the last part)
    v0 = fmaf(x0[u], fi, v0);
    v1 = fmaf(x1[u], fi, v1);
  }
}
// join of the chunks: one wave per (token, head), lanes over the head dim, 4 heads a block.  Rows of one chunk are done; a token
// outside all sequences is zero.  The parts' maxima and sums are read 64 chunks at a time, the parts themselves eight or four at once
template <typename T> __global__ __launch_bounds__(256) void pk_join_kernel(PkArgs a) {
  const unsigned per = (a.H + 3) / 4;
  const int t = blockIdx.x / per, h = __builtin_amdgcn_readfirstlane((int)(blockIdx.x % per * 4 + (threadIdx.x >> 6)));
  if (h >= a.H) return;
  const int lane = threadIdx.x & 63;
  Chunk c;
  const bool inside = find_chunk<true>(a, t, c);
  if (inside && c.n == 1) return;
  T* o = (T*)a.out + ((int64_t)t * a.H + h) * a.dh;
  float M = -INFINITY, L = 0.f, v0 = 0.f, v1 = 0.f;
  const int vis = inside ? vis_of(a, c.q, t - c.q.qs) : 0;
  if (vis > 0) {                                             // (a maximum of -inf is no row without keys: its scores may all be NaN)
    const int unit = h / a.gp, r = (t - c.q.qs - c.tile * a.per) * a.gp + h % a.gp;      // (heads of a unit are consecutive)
    const int n = __builtin_amdgcn_readfirstlane((int)min((int64_t)c.n, a.tiles - c.first));                             // (never past the workspace)
    for (int i = lane; i < n; i += 64) M = fmaxf(M, part_of(a, c.first + i, unit)[32 * a.dh + 2 * r]);
    M = wave_max(M);
    const unsigned d0 = min(lane, a.dh - 1), d1 = min(lane + 64, a.dh - 1);
    const int64_t next = (int64_t)a.units * (32 * (a.dh + 2));
    for (int i0 = 0; i0 < n; i0 += 64) {
      float f = 0.f;
      if (i0 + lane < n) {
        const float* ml = part_of(a, c.first + i0 + lane, unit) + 32 * a.dh + 2 * r;
        f = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml[0] - M) * a.c);
        L = fmaf(ml[1], f, L);
      }
      const int e = min(64, n - i0);
      const float* p = (const float*)uniform64((int64_t)(part_of(a, c.first + i0, unit) + r * a.dh));
      int i = 0;
      for (; i + 8 <= e; i += 8) join_parts<8>(p + i * next, next, 8, d0, d1, f, i, v0, v1);
      for (; i < e; i += 4) join_parts<4>(p + i * next, next, e - i, d0, d1, f, i, v0, v1);
    }
    L = wave_sum(L);
  }
  const float inv = vis > 0 ? 1.0f / L : 0.f;
  v0 *= inv; v1 *= inv;
  if (lane < a.dh) o[lane] = from_f<T>(v0);
  if (lane + 64 < a.dh) o[lane + 64] = from_f<T>(v1);
  if (sizeof(T) == 2 && a.out_lo) {
    T* lo = (T*)a.out_lo + ((int64_t)t * a.H + h) * a.dh;
    if (lane < a.dh) lo[lane] = from_f<T>(v0 - to_f(from_f<T>(v0)));
    if (lane + 64 < a.dh) lo[lane + 64] = from_f<T>(v1 - to_f(from_f<T>(v1)));
  }
  if (a.lse && lane == 0) store_lse(a, h, t, M, L, vis);
}

// ---------------------------------------------------------------------------------------------
// backward, dQ: NW * 32 rows as in the forward (KS: 32 rows, every wave with keys of its own, the waves' sums joined at the end);
// delta = dO.O of the block's rows is formed here and kept for dK / dV.  Two waves a SIMD; the joined one at head dim 128 is faster
// with one and no spills (32 sequences of 8 queries and 500 keys, heads 16/4, both directions: 73 and 83 us).
// 5 causal sequences of 1 148 - 4 956 (10 156 tokens), heads 16/4 of 128, bf16 (193 GF): 247 us = 0.78 PF/s (median of 23, shortest 235), MFMA busy
// 38 % of the cycles at 2.0 GHz.  45 % of the waves' cycles are waits: one buffer of keys between two barriers a step, filled through
// registers.
// Spills at bf16, head dim 128 (256 registers): 2 of the 128-row form, each half of a step reads one again; 59 of the one-wave form, 8 reads a
// step - it still is the faster one for short sequences (171 us, 224 with 128-row blocks, below).
// ---------------------------------------------------------------------------------------------
template <typename T, int D, int NW, int BN, bool KS>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 4 || (KS && NW > 1 && D == 128) ? 1 : 2) void pk_bwd_dq_kernel(PkArgs a) {
  typedef Tile<T, D> TL;
  constexpr int WB = 2 * BN * TL::RB, NT = KS ? 64 : 64 * NW;                   // KS: a wave has keys of its own, staged by itself
  __shared__ __attribute__((aligned(512))) char sm[(KS ? NW : 1) * WB];
  const int own = KS ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  char *Ks = sm + own * WB, *Vs = Ks + BN * TL::RB;
  const int tid = threadIdx.x & (NT - 1), lane = tid & 63, wave = KS ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5;
  const int unit = blockIdx.x % a.units, kh = unit / a.chunks, h0 = kh * a.G + (unit % a.chunks) * a.gp;
  Seq q; int ti, over, total;
  if (!find_tile<false>(a, blockIdx.x / a.units, q, ti, over, total)) {
    outside_rows(a.cu_q, a.S, a.Tq, over, a.tiles - total, [&](int r) {
      for (int h = h0; h < h0 + a.gp; ++h) zero_row<T>((T*)a.dQ + r * a.dq_tok + h * a.dq_head, a.dh);
    });
    return;
  }
  const int r = wave * 32 + (lane & 31), tok0 = ti * a.per, tok = tok0 + r / a.gp, h = h0 + r % a.gp;
  const bool valid = r < a.per * a.gp && tok < q.qlen;
  const int vis = valid ? vis_of(a, q, tok) : 0;
  const int last = min(tok0 + a.per, q.qlen) - 1;
  const int nk = vis_of(a, q, last);
  const int w_lo = tok0 + (int)(wave * 32 * a.inv_gp >> 16), w_hi = tok0 + (int)((wave * 32 + 31) * a.inv_gp >> 16);      // the wave's tokens
  const int w_min = vis_of(a, q, min(w_lo, last)), w_max = vis_of(a, q, min(w_hi, last));
  const bool w_any = w_lo <= last;
  const int64_t t = q.qs + tok;
  typename TL::frag qf[TL::NS], df[TL::NS];
  TL::load_cols(valid ? (const T*)a.Q + t * a.q_tok + h * a.q_head : nullptr, a.dh, hh, qf);
  TL::load_cols(vis > 0 ? (const T*)a.dO + t * a.do_tok + h * a.do_head : nullptr, a.dh, hh, df);      // (a row that sees no key: 0 whatever its dO)
  float delta = 0.f;
  {
    typename TL::frag of[TL::NS];
    TL::load_cols(valid ? (const T*)a.O + (t * a.H + h) * a.dh : nullptr, a.dh, hh, of);
#pragma unroll
    for (int s = 0; s < TL::NS; ++s)
#pragma unroll
      for (int j = 0; j < TL::EP; ++j) delta = fmaf((float)df[s][j], (float)of[s][j], delta);
    if (sizeof(T) == 2) {                                    // O to f32 precision: a rounded O would shift every dS of the row
      TL::load_cols(valid ? (const T*)a.out_lo + (t * a.H + h) * a.dh : nullptr, a.dh, hh, of);
#pragma unroll
      for (int s = 0; s < TL::NS; ++s)
#pragma unroll
        for (int j = 0; j < TL::EP; ++j) delta = fmaf((float)df[s][j], (float)of[s][j], delta);
    }
    delta += __shfl_xor(delta, 32, 64);
    if (valid && hh == 0 && own == 0) a.delta[(int64_t)h * a.Tq + t] = delta;
  }
  float lse = valid ? a.lse[(int64_t)h * a.Tq + t] : INFINITY;
  const float base = far_base(a, (int64_t)h * a.Tq + t, lse);
  const bool far = __any(base != 0.f);
  const T* Kb = (const T*)a.K + q.ks * a.k_tok + kh * a.k_head;
  const T* Vb = (const T*)a.V + q.ks * a.v_tok + kh * a.v_head;
  f32x16 acc[D / 32] = {};
  Stage<T, D, BN, NT> ks, vs;
  constexpr int STEP = KS ? NW * BN : BN;
  int kt = own * BN;
  if (kt < nk) { ks.load(Kb, a.k_tok, kt, q.klen, a.dh, tid); vs.load(Vb, a.v_tok, kt, q.klen, a.dh, tid); }
  for (; kt < nk; kt += STEP) {
    if constexpr (KS) wave_lds_fence(); else __syncthreads();
    ks.pad(a.dh, tid); vs.pad(a.dh, tid);
    ks.store(Ks, tid); vs.store(Vs, tid);
    if constexpr (KS) wave_lds_fence(); else __syncthreads();
    if (kt + STEP < nk) { ks.load(Kb, a.k_tok, kt + STEP, q.klen, a.dh, tid); vs.load(Vb, a.v_tok, kt + STEP, q.klen, a.dh, tid); }
    if (w_any && kt < w_max) {
      const bool mask = kt + BN > w_min;
#pragma unroll
      for (int b = 0; b < BN / 32; ++b) {
        f32x16 s = TL::row_mm(Ks, 32 * b, qf, lane);
        const f32x16 dp = TL::row_mm(Vs, 32 * b, df, lane);
        if (mask | far) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[i] = kt + 32 * b + c_row(i, hh) < vis ? s[i] - base : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.c, -lse)) * (dp[i] - delta);
        col_mm<D>((const T*)nullptr, Ks, 32 * b, s, acc, lane);
      }
    }
  }
  T* out = (T*)a.dQ + t * a.dq_tok + h * a.dq_head;
  if constexpr (KS && NW > 1) {                              // join the waves, thread -> (row, 4 consecutive d)
    wave_lds_fence();
    float* mine = (float*)(sm + own * WB);
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[(dt * 32 + c_row(i, hh)) * 32 + r] = acc[dt][i];
    __syncthreads();
    if (!valid) return;
    for (int d = (own * 2 + hh) * 4; d < a.dh; d += NW * 8) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += ((float*)(sm + w * WB))[(d + j) * 32 + r];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= a.scale;
      Vec4<T>::store(out + d, v);
    }
  } else {
    if (valid) store_cols<T, D>(out, a.dh, acc, a.scale, hh);
  }
}

// ---------------------------------------------------------------------------------------------
// backward, dK / dV.  A wave holds 32 keys as columns; the NW waves are NW / RG groups of keys x RG groups of rows, whose sums are
// joined at the end.  The rows of every head of the group stream through LDS, RG * 32 at a time.  `splits` blocks share the rows of
// a key block and leave f32 parts (joined by pk_bwd_join_kernel) where there are few key blocks.
// VL: V is read from LDS as well.  At head dim 128 the two accumulators take 128 registers, K and V as columns 64, two blocks of
// scores 32: without V two waves fit a SIMD, and they hide what one wave with all of it in registers (512) had to wait for.
// One register too many is worse than either: a spill's reload waits for the loads of the next rows (base of rows far from zero kept in a
// register between the loads and the barrier: 3 spilled, 768 us for the documents' both directions; read where it is needed: 753).
// The same documents (257 GF): 376 us = 0.68 PF/s (median of 23, shortest 354), MFMA busy 33 % at 2.0 GHz, 46 % of the waves' cycles waits, and
// 36 us for the join of 208 MB of parts (5.8 TB/s).  The one-wave form at bf16, head dim 128 spills 13 registers beside 512 in use.
// ---------------------------------------------------------------------------------------------
template <typename T, int D, int NW, int RG, bool VL>
__global__ __launch_bounds__(64 * NW, sizeof(T) * D == 128 || NW == 8 ? 2 : 1) void pk_bwd_dkv_kernel(PkArgs a) {
  typedef Tile<T, D> TL;
  constexpr int BR = 32 * RG, KG = NW / RG, JOIN = KG * (RG - 1) * 32 * D * 4;
  constexpr int VB = VL ? KG * 32 * TL::RB : 0, SM = VB + 2 * BR * TL::RB > JOIN ? VB + 2 * BR * TL::RB : JOIN;
  __shared__ __attribute__((aligned(512))) char sm[SM];
  __shared__ __attribute__((aligned(16))) float Ls[BR], Ds[BR], Bs[BR];
  __shared__ __attribute__((aligned(16))) int Vis[BR];
  __shared__ int Far[RG];                                    // does any of 32 rows have a base?
  char *Vs = sm, *Qs = sm + VB, *Os = Qs + BR * TL::RB;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, kg = wave / RG, rg = wave % RG;
  const int nkh = a.H / a.G, kh = blockIdx.x % nkh;
  const int rest = blockIdx.x / nkh, part = rest % a.splits;
  Seq q; int ti, over, total;
  if (!find_tile<true>(a, rest / a.splits, q, ti, over, total)) {
    if (a.splits == 1)
      outside_rows(a.cu_k, a.S, a.Tk, over, a.tiles - total, [&](int r) {
        zero_row<T>((T*)a.dK + r * a.dk_tok + kh * a.dk_head, a.dh);
        zero_row<T>((T*)a.dV + r * a.dv_tok + kh * a.dv_head, a.dh);
      });
    return;
  }
  const int k0 = ti * a.per, w0 = k0 + kg * 32, key = w0 + (lane & 31);       // first key of the block, of the wave; the lane's
  typename TL::frag kf[TL::NS], vf[TL::NS];
  TL::load_cols(key < q.klen ? (const T*)a.K + (q.ks + (int64_t)key) * a.k_tok + kh * a.k_head : nullptr, a.dh, hh, kf);
  TL::load_cols(key < q.klen ? (const T*)a.V + (q.ks + (int64_t)key) * a.v_tok + kh * a.v_head : nullptr, a.dh, hh, vf);
  if constexpr (VL) {                                        // (the row groups of a key group write the same)
#pragma unroll
    for (int s = 0; s < TL::NS; ++s) *reinterpret_cast<typename TL::frag*>(Vs + TL::at(key - k0, 2 * s + hh)) = vf[s];
  }
  f32x16 dk[D / 32] = {}, dv[D / 32] = {};
  const int btok = (int)(BR * a.inv_gp >> 16), used = btok * a.gp;
  // row blocks: the tokens from the first that sees key k0, for one chunk of heads after the other
  const int first = a.causal ? max(0, k0 - (q.klen - q.qlen)) : 0;
  const int per_chunk = first < q.qlen ? (q.qlen - first + btok - 1) / btok : 0;
  const int64_t blocks = (int64_t)per_chunk * a.chunks;
  const int b0 = (int)(blocks * part / a.splits), b1 = (int)(blocks * (part + 1) / a.splits);
  int ch = per_chunk ? b0 / per_chunk : 0, tok0 = first + (b0 - ch * per_chunk) * btok;
  Stage<T, D, BR, 64 * NW> qs, os;
  float lv = INFINITY, dl = 0.f;
  auto load = [&](int c, int t0) {
    const int h0 = kh * a.G + c * a.gp;
    qs.load_rows((const T*)a.Q + q.qs * a.q_tok + h0 * a.q_head, a.q_tok, a.q_head, t0, q.qlen, a.gp, a.inv_gp, a.dh, tid);
    os.load_rows((const T*)a.dO + q.qs * a.do_tok + h0 * a.do_head, a.do_tok, a.do_head, t0, q.qlen, a.gp, a.inv_gp, a.dh, tid);
    if (tid < BR) {
      const int rt = (int)(tid * a.inv_gp >> 16), tok = t0 + rt;
      const bool in = tid < used && tok < q.qlen;
      const int64_t at = (int64_t)(h0 + tid - rt * a.gp) * a.Tq + q.qs + tok;
      lv = in ? a.lse[at] : INFINITY;
      dl = in ? a.delta[at] : 0.f;
    }
  };
  if (b0 < b1) load(ch, tok0);
  for (int b = b0; b < b1; ++b) {
    __syncthreads();
    qs.pad(a.dh, tid); os.pad(a.dh, tid);
    qs.store(Qs, tid); os.store(Os, tid);
    if (tid < BR) {
      const int rt = (int)(tid * a.inv_gp >> 16), tok = tok0 + rt;
      const float bs = far_base(a, (int64_t)(kh * a.G + ch * a.gp + tid - rt * a.gp) * a.Tq + q.qs + tok, lv);
      Ls[tid] = lv; Ds[tid] = dl; Bs[tid] = bs; Vis[tid] = tid < used && tok < q.qlen ? vis_of(a, q, tok) : 0;
      const unsigned long long any = __ballot(bs != 0.f);
      if ((tid & 31) == 0) Far[tid >> 5] = (uint32_t)(any >> (tid & 32)) != 0u;
    }
    __syncthreads();
    const bool far = __builtin_amdgcn_readfirstlane(Far[rg]) != 0;      // (asked for ahead of the products, whose reads cover it)
    const int now = tok0;
    tok0 += btok;
    if (tok0 >= q.qlen) { tok0 = first; ++ch; }
    if (b + 1 < b1) load(ch, tok0);
    // this wave's rows: tokens t_lo .. t_hi of the block.  Nothing to do if the last of them sees none of the wave's keys; masked
    // if the first does not see all of them (columns behind the last key are not stored)
    const int r_lo = 32 * rg;
    const int t_lo = now + (int)(r_lo * a.inv_gp >> 16), t_hi = min(now + (int)((r_lo + 31) * a.inv_gp >> 16), q.qlen - 1);
    if (t_lo >= q.qlen || vis_of(a, q, t_hi) <= w0) continue;
    const bool mask = a.causal && vis_of(a, q, t_lo) < w0 + 32;
    f32x16 p = TL::template row_mm<VL>(Qs, r_lo, kf, lane), ds;
    if constexpr (VL) ds = TL::row_mm(Os, r_lo, Vs, w0 - k0, lane);
    else ds = TL::row_mm(Os, r_lo, vf, lane);
    if (far) {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] -= Bs[r_lo + c_row(i, hh)];
    }
    if (mask) {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = key < Vis[r_lo + c_row(i, hh)] ? p[i] : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r0 = r_lo + 8 * j + 4 * hh;
      const f32x4 l4 = *reinterpret_cast<const f32x4*>(Ls + r0), d4 = *reinterpret_cast<const f32x4*>(Ds + r0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * j + e;
        const float x = __builtin_amdgcn_exp2f(fmaf(p[i], a.c, -l4[e]));
        ds[i] = x * (ds[i] - d4[e]);
        p[i] = x;
      }
    }
    col_mm<D, VL>((const T*)nullptr, Os, r_lo, p, dv, lane);
    col_mm<D, VL>((const T*)nullptr, Qs, r_lo, ds, dk, lane);
  }
  if constexpr (RG > 1) {                                     // join the row groups, dK first, then dV
    auto join = [&](f32x16 (&acc)[D / 32]) {
      float* buf = (float*)sm + (size_t)kg * (RG - 1) * (D / 32) * 16 * 64;
      __syncthreads();
      if (rg > 0) {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) buf[(((rg - 1) * (D / 32) + dt) * 16 + i) * 64 + lane] = acc[dt][i];
      }
      __syncthreads();
      if (rg == 0) {
#pragma unroll
        for (int g = 0; g < RG - 1; ++g)
#pragma unroll
          for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] += buf[((g * (D / 32) + dt) * 16 + i) * 64 + lane];
      }
    };
    join(dk);
    join(dv);
    if (rg > 0) return;
  }
  if (key >= q.klen) return;
  const int64_t kr = q.ks + (int64_t)key;
  if (a.splits > 1) {
    float* o = a.part + ((((int64_t)part * 2) * a.Tk + kr) * nkh + kh) * a.dh;
    store_cols<float, D>(o, a.dh, dk, a.scale, hh);
    store_cols<float, D>(o + (int64_t)a.Tk * nkh * a.dh, a.dh, dv, 1.0f, hh);
  } else {
    store_cols<T, D>((T*)a.dK + kr * a.dk_tok + kh * a.dk_head, a.dh, dk, a.scale, hh);
    store_cols<T, D>((T*)a.dV + kr * a.dv_tok + kh * a.dv_head, a.dh, dv, 1.0f, hh);
  }
}
// sum of the parts, in order; one block of 256 threads per key (all heads, dK and dV).  Keys of no sequence: zeros
template <typename T> __global__ __launch_bounds__(256) void pk_bwd_join_kernel(PkArgs a) {
  const int64_t key = blockIdx.x;
  const int nkh = a.H / a.G, row = nkh * a.dh;
  // last sequence that starts at or before this key
  int s = -1;
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    const int i = s0 + (threadIdx.x & 63);
    const int n = __popcll(__ballot(i < a.S && a.cu_k[i] <= key));
    s += n;
    if (n < 64) break;
  }
  s = __builtin_amdgcn_readfirstlane(s);
  bool inside = false, room = false;
  if (s >= 0) {
    const Seq q = load_seq(a, s);
    inside = key >= q.ks && key < (int64_t)q.ks + q.klen;
    room = !inside && key < a.cu_k[s + 1];                    // (the unfilled part of a slot is left as it is)
  }
  if (room) return;
  const int64_t plane = (int64_t)a.Tk * row;
  for (int e = threadIdx.x * 4; e < 2 * row; e += 1024) {
    const int which = e >= row, c = e - which * row, kh = c / a.dh, d = c - kh * a.dh;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (inside)
      for (int p = 0; p < a.splits; ++p) {
        float x[4];
        Vec4<float>::load(a.part + (int64_t)(2 * p + which) * plane + key * row + c, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += x[j];
      }
    T* o = which ? (T*)a.dV + key * a.dv_tok + kh * a.dv_head : (T*)a.dK + key * a.dk_tok + kh * a.dk_head;
    Vec4<T>::store(o + d, v);
  }
}

// ---------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------
#define PK_BLOCKS 1536
static int largest_divisor(int n, int most) {
  for (int d = n < most ? n : most; d > 1; --d)
    if (n % d == 0) return d;
  return 1;
}
static bool pk_few_rows(const evlm_packed_attn_args* x, int gp) {
  // rows of a sequence and chunk of heads, on average: one wave's worth -> keys are split over the waves instead of rows
  return (int64_t)x->Tq * gp <= (int64_t)48 * x->S;
}
// chunks of keys aimed at for each chunk of heads; 0: every block of rows walks all its keys.  Worth it where the rows alone are too few
// blocks for the chip, or are of very different lengths and long enough to pay for the second kernel.  Single tokens, heads 32/8 of 128,
// lengths between a third and five thirds of the mean, us with / without chunks: 800 keys, 72 blocks 34 / 33, 288: 37 / 28; 2000 keys,
// 144: 43 / 38, 576: 122 / 124; 8000 keys, 144: 126 / 185, 576: 438 / 487, 1152: 903 / 928.  12 sequences of 6 000 - 40 000 keys (104
// blocks): 137 / 400.  30 rows on 577 keys, heads 12/12 of 64, 1488: 61 / 34
static int pk_want(const evlm_packed_attn_args* x, int gp) {
  if (x->S == 0 || x->Tq == 0 || !pk_few_rows(x, gp) || (int64_t)x->Tk <= (int64_t)2 * PK_CHUNK * x->S) return 0;
  const int64_t units = x->H / gp, blocks = ((int64_t)x->Tq * gp / 32 + x->S) * units;
  const bool wanted = blocks < 128 || (blocks < 1024 && (int64_t)x->Tk >= (int64_t)4096 * x->S);
  return wanted ? (int)((PK_BLOCKS + units - 1) / units) : 0;
}
static int64_t pk_chunk_slots(const evlm_packed_attn_args* x, int gp) {     // an upper bound of the chunks, whatever the lengths
  return pk_want(x, gp) + (int64_t)x->Tq / (32 / gp) + x->S;
}
// dK / dV, the shape of a block: waves, groups of rows among them; the other factor are groups of 32 keys
template <typename T, int D> struct DkvShape { static constexpr int NW = 4, RG = sizeof(T) == 4 ? 1 : 4, KEYS = 32 * NW / RG; static constexpr bool VL = D > 64; };
template <> struct DkvShape<bf16, 128> { static constexpr int NW = 8, RG = 1, KEYS = 256; static constexpr bool VL = true; };
// ... blocks of one wave, 32 keys, for short key ranges.  16 384 tokens, heads 8/8, backward in us, one wave against a full block:
// bf16 dim 64, 24 keys a sequence 85 / 201, 72: 77 / 117, 150: 76 / 105, 250: 77 / 108 (heads 16/4: 150: 96 / 104, 250: 119 / 117);
// bf16 dim 128, 24: 172 / 293, 44: 145 / 195 (100 keys, blocks of four waves that share 32 keys: 297 / 156).  f32 at dim 128 has
// no such kernel: with all of K, V and both sums in one wave's registers it spilled (4096 tokens, heads 16/4, 44 keys: 311 / 234)
template <typename T, int D> static bool pk_few_keys(int Tk, int S) {
  if (D > 64 && sizeof(T) == 4) return false;
  return (int64_t)Tk <= (int64_t)(D <= 64 ? 160 : 48) * S;
}
// ... parts of the rows of a key block, where there are too few key blocks for the chip; each part still has some hundred rows.
// 256-key blocks are long and (causal) of very different lengths: they want three a CU (5 x 176 blocks of the documents' 10 156
// keys and 4 key heads: 607 us backward; 3 x 176: 670; undivided 64-key blocks of 4 waves: 715), shorter ones just the CUs filled
template <typename T, int D> static int pk_parts_of(const evlm_packed_attn_args* x) {
  typedef DkvShape<T, D> SH;
  if (pk_few_keys<T, D>(x->Tk, x->S)) return 1;
  const int64_t blocks = ((int64_t)x->Tk / SH::KEYS + x->S) * x->Hkv, rows = (int64_t)x->Tq * (x->H / x->Hkv) / x->S;
  int64_t n = ((SH::KEYS == 256 ? 768 : 256) + blocks - 1) / blocks;
  if (n > rows / 512) n = rows / 512;
  return n < 1 ? 1 : (n > 8 ? 8 : (int)n);
}
static int pk_parts(const evlm_packed_attn_args* x) {
  if (x->S == 0 || x->Tk == 0) return 1;
  return x->dtype == EVLM_BF16 ? (x->dh <= 64 ? pk_parts_of<bf16, 64>(x) : pk_parts_of<bf16, 128>(x))
                               : (x->dh <= 64 ? pk_parts_of<float, 64>(x) : pk_parts_of<float, 128>(x));
}
static int pk_check(const evlm_packed_attn_args* x, const char* name) {
  EVLM_REQUIRE(x->dtype == EVLM_F32 || x->dtype == EVLM_BF16, "%s: bad dtype %d", name, x->dtype);
  EVLM_REQUIRE(x->Tq >= 0 && x->Tk >= 0 && x->S >= 0 && x->H > 0 && x->Hkv > 0 && x->H % x->Hkv == 0, "%s: bad sizes", name);
  EVLM_REQUIRE(x->Tq <= (1 << 30) && x->Tk <= (1 << 30) && x->S <= (1 << 30), "%s: more than 2^30 tokens or sequences", name);
  EVLM_REQUIRE(x->dh > 0 && x->dh <= 128 && x->dh % 8 == 0, "%s: head dim %d is not a multiple of 8 up to 128", name, x->dh);
  EVLM_REQUIRE(x->scale > 0.f && x->scale < 1e30f, "%s: the scale must be positive and finite", name);
  EVLM_REQUIRE(x->S == 0 || (x->cu_q && x->cu_k), "%s: no sequence starts", name);
  const int64_t st[6] = {x->q_tok, x->q_head, x->k_tok, x->k_head, x->v_tok, x->v_head};
  const int unit = x->dtype == EVLM_BF16 ? 8 : 4;
  for (int i = 0; i < 6; ++i) EVLM_REQUIRE(st[i] >= 0 && st[i] % unit == 0, "%s: strides must be whole 16-byte pieces", name);
  EVLM_REQUIRE(x->k_tok < (1 << 22) && x->v_tok < (1 << 22), "%s: token strides of K and V must stay below 2^22 elements", name);
  EVLM_REQUIRE(x->q_tok < (1 << 22) && x->q_head < (1 << 22), "%s: strides of Q must stay below 2^22 elements", name);
  EVLM_REQUIRE((((uintptr_t)x->Q | (uintptr_t)x->K | (uintptr_t)x->V) & 15) == 0, "%s: tensors must be 16-byte aligned", name);
  return 0;
}
static PkArgs pk_args(const evlm_packed_attn_args* x) {
  PkArgs a = {};
  a.Q = x->Q; a.K = x->K; a.V = x->V; a.out = x->O; a.O = x->O; a.out_lo = x->O_lo; a.lse = x->lse;
  a.far = x->lse_planes == 2;
  a.cu_q = x->cu_q; a.cu_k = x->cu_k; a.k_lens = x->k_lens;
  a.q_tok = x->q_tok; a.q_head = x->q_head; a.k_tok = x->k_tok; a.k_head = x->k_head; a.v_tok = x->v_tok; a.v_head = x->v_head;
  a.Tq = x->Tq; a.Tk = x->Tk; a.S = x->S; a.H = x->H; a.G = x->H / x->Hkv; a.dh = x->dh;
  a.gp = largest_divisor(a.G, 32);
  a.inv_gp = (65536u + a.gp - 1) / a.gp;
  a.chunks = a.G / a.gp; a.units = a.chunks * x->Hkv;
  a.causal = x->causal != 0; a.scale = x->scale; a.c = x->scale * PK_LOG2E;
  a.splits = 1;
  return a;
}
// grid: `units` x (upper bound of the number of blocks + 1, so that there always is a surplus block for the rows outside)
static int pk_grid(PkArgs& a, int64_t T, int per, int units, const char* name, unsigned* grid) {
  a.per = per;
  const int64_t tiles = T / per + a.S + 1, n = tiles * units * a.splits;
  if (n > 0x7fffffffll) return evlm_set_error("%s: too many blocks", name);
  a.tiles = (int)tiles;
  *grid = (unsigned)n;
  return 0;
}

extern "C" int evlm_packed_attention_workspace(const evlm_packed_attn_args* x, int backward) {
  if (!x || pk_check(x, "evlm_packed_attention_workspace")) return 0;       // (the call itself refuses such arguments)
  const int gp = largest_divisor(x->H / x->Hkv, 32);
  if (backward) {
    const int parts = pk_parts(x);
    return parts > 1 ? (int)((int64_t)parts * 2 * x->Tk * x->Hkv * x->dh) : 0;
  }
  return pk_want(x, gp) ? (int)(pk_chunk_slots(x, gp) * (x->H / gp) * 32 * (x->dh + 2)) : 0;
}

template <typename T, int D> static int pk_fwd_launch(PkArgs& a, bool few, int64_t slots, hipStream_t stream) {
  unsigned grid;
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  if (a.want) {
    a.per = 32 / a.gp;
    a.tiles = (int)slots;
    hipLaunchKernelGGL((pk_fwd_keys_kernel<T, D, 4, true>), dim3((unsigned)(slots * a.units)), dim3(256), 0, stream, a);
    EVLM_LAUNCH_CHECK("evlm_packed_attention_fwd");
    const int64_t blocks = (int64_t)a.Tq * ((a.H + 3) / 4);
    hipLaunchKernelGGL((pk_join_kernel<T>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  } else if (few) {
    if (int rc = pk_grid(a, a.Tq, 32 / a.gp, a.units, "evlm_packed_attention_fwd", &grid)) return rc;
    if (a.S > 0 && a.Tk / a.S <= 64)
      hipLaunchKernelGGL((pk_fwd_keys_kernel<T, D, 1, false>), dim3(grid), dim3(64), 0, stream, a);
    else
      hipLaunchKernelGGL((pk_fwd_keys_kernel<T, D, 4, false>), dim3(grid), dim3(256), 0, stream, a);
  } else {
    if (int rc = pk_grid(a, a.Tq, 128 / a.gp, a.units, "evlm_packed_attention_fwd", &grid)) return rc;
    hipLaunchKernelGGL((pk_fwd_rows_kernel<T, D, 4, BN>), dim3(grid), dim3(256), 0, stream, a);
  }
  EVLM_LAUNCH_CHECK("evlm_packed_attention_fwd");
  return 0;
}

// Head dims run the code of the next of 64 and 128, the pieces behind them zero: 32 pays for products and LDS of 64 (20 causal sequences of
// 42 - 884, heads 12/4, both directions: 89 us, 95 at 64), 72 - 120 for those of 128.
#define PK_DISPATCH(x, CALL)                                                                                   \
  ((x)->dtype == EVLM_BF16 ? ((x)->dh <= 64 ? CALL<bf16, 64> : CALL<bf16, 128>)                                \
                           : ((x)->dh <= 64 ? CALL<float, 64> : CALL<float, 128>))

extern "C" int evlm_packed_attention_fwd(const evlm_packed_attn_args* x, void* stream_) {
  EVLM_REQUIRE(x, "evlm_packed_attention_fwd: no arguments");
  if (int rc = pk_check(x, "evlm_packed_attention_fwd")) return rc;
  if (x->Tq == 0) return 0;
  EVLM_REQUIRE(x->Q && x->O && (x->Tk == 0 || (x->K && x->V)), "evlm_packed_attention_fwd: null tensor");
  PkArgs a = pk_args(x);
  const bool few = x->S > 0 && pk_few_rows(x, a.gp);
  a.want = pk_want(x, a.gp);
  const int64_t slots = a.want ? pk_chunk_slots(x, a.gp) : 0;
  if (a.want) {
    EVLM_REQUIRE(x->workspace, "evlm_packed_attention_fwd: this many keys for so few rows need a workspace");
    a.part = (float*)x->workspace;
  }
  return PK_DISPATCH(x, pk_fwd_launch)(a, few, slots, (hipStream_t)stream_);
}

template <typename T, int D> static int pk_bwd_launch(PkArgs& a, bool few, int parts, hipStream_t stream) {
  unsigned grid;
  constexpr int BN = sizeof(T) == 2 ? 64 : 32;
  const char* name = "evlm_packed_attention_bwd";
  const int nkh = a.H / a.G;
  if (a.Tq > 0) {
    // few rows: one wave a block (16 384 tokens, heads 8/8, 24 a sequence, bf16 dim 128: backward 171 us, 224 with 128-row blocks), but
    // not at dim 128 in f32, where it spilled (4096 tokens, heads 16/4, 24 a sequence: 267 us, 227 with 128-row blocks).  Its keys
    // split over four waves where they are many and the blocks would not give every SIMD a wave (both directions, 9 sequences of 47
    // queries and 210 keys, 12 heads of 64 in f32: 60 us, 83 with one wave; 64 sequences of 30 and 577 in bf16, 768 blocks: 270, 264)
    constexpr bool kOneWave = D <= 64 || sizeof(T) == 2;
    const bool split = few && a.Tk / a.S > 64 && ((int64_t)a.Tq * a.gp / 32 + a.S) * a.units <= 1024;
    if (few && kOneWave) {
      if constexpr (kOneWave) {
        if (int rc = pk_grid(a, a.Tq, 32 / a.gp, a.units, name, &grid)) return rc;
        if (split) hipLaunchKernelGGL((pk_bwd_dq_kernel<T, D, 4, 32, true>), dim3(grid), dim3(256), 0, stream, a);
        else hipLaunchKernelGGL((pk_bwd_dq_kernel<T, D, 1, 32, true>), dim3(grid), dim3(64), 0, stream, a);
      }
    } else {
      if (int rc = pk_grid(a, a.Tq, 128 / a.gp, a.units, name, &grid)) return rc;
      hipLaunchKernelGGL((pk_bwd_dq_kernel<T, D, 4, BN, false>), dim3(grid), dim3(256), 0, stream, a);
    }
    EVLM_LAUNCH_CHECK(name);
  }
  if (a.Tk > 0) {
    a.splits = parts;
    if (pk_few_keys<T, D>(a.Tk, a.S)) {
      if constexpr (D <= 64 || sizeof(T) == 2) {
        if (int rc = pk_grid(a, a.Tk, 32, nkh, name, &grid)) return rc;
        hipLaunchKernelGGL((pk_bwd_dkv_kernel<T, D, 1, 1, false>), dim3(grid), dim3(64), 0, stream, a);
      }
    } else {
      typedef DkvShape<T, D> SH;
      if (int rc = pk_grid(a, a.Tk, SH::KEYS, nkh, name, &grid)) return rc;
      hipLaunchKernelGGL((pk_bwd_dkv_kernel<T, D, SH::NW, SH::RG, SH::VL>), dim3(grid), dim3(64 * SH::NW), 0, stream, a);
    }
    if (a.splits > 1) {
      EVLM_LAUNCH_CHECK(name);
      hipLaunchKernelGGL((pk_bwd_join_kernel<T>), dim3((unsigned)a.Tk), dim3(256), 0, stream, a);
    }
    EVLM_LAUNCH_CHECK(name);
  }
  return 0;
}

extern "C" int evlm_packed_attention_bwd(const evlm_packed_attn_args* x, void* stream_) {
  EVLM_REQUIRE(x, "evlm_packed_attention_bwd: no arguments");
  const char* name = "evlm_packed_attention_bwd";
  if (int rc = pk_check(x, name)) return rc;
  EVLM_REQUIRE(x->Tq == 0 || (x->Q && x->O && x->dO && x->dQ && x->lse && x->delta), "%s: null tensor", name);
  EVLM_REQUIRE(x->Tq == 0 || x->dtype == EVLM_F32 || x->O_lo, "%s: bf16 needs O_lo", name);
  EVLM_REQUIRE(x->Tk == 0 || (x->K && x->V && x->dK && x->dV), "%s: null tensor", name);
  const int64_t st[8] = {x->do_tok, x->do_head, x->dq_tok, x->dq_head, x->dk_tok, x->dk_head, x->dv_tok, x->dv_head};
  const int unit = x->dtype == EVLM_BF16 ? 8 : 4;
  for (int i = 0; i < 8; ++i) EVLM_REQUIRE(st[i] >= 0 && st[i] % unit == 0, "%s: strides must be whole 16-byte pieces", name);
  EVLM_REQUIRE((((uintptr_t)x->dO | (uintptr_t)x->dQ | (uintptr_t)x->dK | (uintptr_t)x->dV) & 15) == 0, "%s: tensors must be 16-byte aligned", name);
  EVLM_REQUIRE(x->do_tok < (1 << 22) && x->do_head < (1 << 22), "%s: strides of dO must stay below 2^22 elements", name);
  PkArgs a = pk_args(x);
  a.dO = x->dO; a.dQ = x->dQ; a.dK = x->dK; a.dV = x->dV; a.delta = x->delta;
  a.do_tok = x->do_tok; a.do_head = x->do_head; a.dq_tok = x->dq_tok; a.dq_head = x->dq_head;
  a.dk_tok = x->dk_tok; a.dk_head = x->dk_head; a.dv_tok = x->dv_tok; a.dv_head = x->dv_head;
  const bool few = x->S > 0 && pk_few_rows(x, a.gp);
  const int parts = pk_parts(x);
  if (parts > 1) {
    EVLM_REQUIRE(x->workspace, "%s: %d row parts need a workspace", name, parts);
    a.part = (float*)x->workspace;
  }
  return PK_DISPATCH(x, pk_bwd_launch)(a, few, parts, (hipStream_t)stream_);
}
