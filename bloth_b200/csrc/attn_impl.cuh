// Attention over [B, S, H, D] head tensors, forward and backward: the
// arguments, the sequences they describe and the tiles of a sequence that see
// one another, shared by every attention kernel.
//
// Mathematics, per query row i and the keys j it sees (see_keys below):
//   s_ij = scale * q_i . k_j,  lse_i = log sum_j exp(s_ij),
//   p_ij = exp(s_ij - lse_i),  o_i = sum_j p_ij v_j;
// backward, which recomputes p from lse instead of reading it:
//   delta_i = do_i . o_i,  dp_ij = do_i . v_j,  ds_ij = p_ij (dp_ij - delta_i),
//   dv_j = sum_i p_ij do_i,  dq_i = scale sum_j ds_ij k_j,
//   dk_j = scale sum_i ds_ij q_i.
// delta takes o to twice the precision of 16-bit tensors (o and `rest`): with
// o as rounded, rows of few keys, whose dp nearly equal delta, would get twice
// the error.
// A row that sees no key has o = 0, lse = -inf and no gradient. Query heads
// h of a group of G = Hq / Hk share key head h / G, whose gradients sum over
// the group inside one CTA, in a fixed order: no atomics anywhere.
// A row that sees one key has p = 1 and dp = delta whatever they are: its ds is
// set to the 0 it is (the difference of the two sums would be their noise).
#pragma once

#include "common.cuh"
#include "heads_impl.cuh"

namespace bloth {

struct AttnArgs {
  HT q, k, v, o, dout, dq, dk, dv;
  void* rest;         // what rounding took off o, times kRestUp, laid out as o (16-bit
                      // tensors), or NULL
  float* lse;         // [B, Hq, Sq] natural logarithm (forward writes, backward reads)
  float* lse2;        // backward workspace: [Hq, R] lse * log2(e) - kBwdShift, +inf where
                      // nothing is seen
  float* delta;       // backward workspace: [Hq, R]
  int64_t R;          // rows per head of lse2 and delta (attn_stat_rows)
  // backward workspace of fp16 tensors, what bounds ds (ds_scale):
  float* donorm;      // [Hq, R] |do_i|
  float2* qtop;       // [Hq, stat_tiles(R)] of 128 query rows, largest |do_i| and |delta_i|
  float* vtop;        // [Hk, stat_tiles(RK)] of 128 key rows, largest |v_j|
  int64_t RK;         // as R, for key rows
  const void* qseq;   // dense: [B] query lengths or NULL; packed: [n + 1] offsets
  const void* kseq;   // the same for keys
  int seq_dt;
  int packed;         // 0: dense, else the number of packed sequences n
  int B, Sq, Sk, Hq, Hk, G;
  float scale, scale_log2;
  int causal;
  int window;         // 0: none
  unsigned int* fault;
};

// Tiles whose rows see at most this many keys each have P and dS as two terms of
// 16 bits: where few terms are summed, a gradient of two nearly equal ones lost up
// to six times what rounding the result takes (bf16, two keys); with two terms no
// more than that rounding. A tile is what a CTA or a group of warps works on, in
// the rows of one sequence: 128 query rows for o and dq, 128 keys with every query
// that sees them for dk and dv, the call's few rows over a cache. The tensors'
// extents do not count.
// It costs a product for each of P and dS: 4 x 8192 rows of 32/8 heads of 128 (bf16),
// forward and backward, 1405 us with a window of 128, 1272 us with one of 129; 8192
// rows as 128 sequences 606 us, with one term 575; 64 x 129 rows, of which the first
// 128 have two terms in o and dq, 480 us, with one term 459.
constexpr int kFineKeys = 128;

// Powers of two that probabilities are held times where they enter a product, so
// that fp16 holds small ones: its normal range starts at 2^-14. In the forward they
// are at most 2^8 (attn_fwd.cuh), in the backward at most 1. They cost nothing: they
// are added to the exponent, and leave with the sum of exponentials or the store.
template <typename T>
constexpr float kFwdShift = std::is_same<T, __half>::value ? 7.f : 0.f;
template <typename T>
constexpr float kBwdShift = std::is_same<T, __half>::value ? 15.f : 0.f;

// The power of two that ds, at most `bound` in size, is held times in fp16, whose
// largest number is 65504: it brings the bound to between 2^14 and 2^15. What it
// leaves above fp16's normal range is 2^29 below the bound.
__device__ __forceinline__ float ds_scale(float bound) {
  const int x = max((__float_as_int(bound) >> 23) - 127, -100);  // floor(log2(bound)), or -100
  return __int_as_float((127 + 14 - x) << 23);
}
// The largest of non-negative numbers, over the lanes of a warp.
__device__ __forceinline__ float warp_top(float x) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x)));
}

// What rounding takes off o is 2^-11 of it in fp16, or less: as it is it would leave
// fp16's range where o is small.
template <typename T>
constexpr int kRestUp = std::is_same<T, __half>::value ? 2048 : 1;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// One sequence: its rows in the tensors and its lengths.
struct AttnSeq {
  int b;           // batch row of the tensors
  int q0, qlen;    // first query row and their number
  int k0, klen;
  int64_t stat0;   // first row of its lse2 and delta rows
  int64_t kstat0;  // the same for rows of keys
  int tile;        // tile of the sequence this CTA works on; < 0: none
};

__device__ __forceinline__ int seq_at(const void* p, int dt, int i, int limit) {
  const int64_t v = dt == BLOTH_I64 ? __ldg(reinterpret_cast<const long long*>(p) + i)
                                    : (int64_t)__ldg(reinterpret_cast<const int*>(p) + i);
  return (int)(v < 0 ? 0 : (v > limit ? limit : v));
}

// Rows of lse2 and delta a packed sequence starts at: 16-byte units, and room
// for its last tile of 128 rows in full.
__host__ __device__ __forceinline__ int64_t attn_stat_base(int64_t cu, int64_t s) {
  return (cu + 3) / 4 * 4 + 132 * s;
}
inline int64_t attn_stat_rows(int64_t B, int64_t Sq, int64_t packed) {
  return packed ? attn_stat_base(Sq, packed + 2) + 128 : B * ((Sq + 127) / 128 * 128);
}
// Tile t of 128 rows of a sequence is entry stat0 / 128 + t of an array with an
// entry for each tile; sequences start more than 128 rows apart.
__host__ __device__ __forceinline__ int64_t stat_tiles(int64_t R) { return R / 128 + 1; }
// Tiles of `tile` rows that cover every sequence, at most (the offsets of
// packed sequences are known on the device only). The rows before the first
// sequence and those past the last are two more, which see nothing.
inline int64_t attn_tiles(int64_t S, int64_t packed, int tile) {
  return (S + tile - 1) / tile + (packed ? packed + 2 : 0);
}

// The sequence and tile of flat tile index `t` (BY_Q: tiles of query rows,
// else of key rows). Called by whole warps; every warp finds the same.
// A step of 32 sequences costs about 150 cycles: sums of their tiles, with scans
// only where the tile is found or the offsets decrease (8192 rows as 2048
// sequences, 32/8 heads of 128, forward: 7.7 ms with scans in each, 5.6 without).
// Packed offsets are clamped to the tensors and to be non-decreasing, so no
// content of the offsets leads outside of them.
template <bool BY_Q>
__device__ __forceinline__ AttnSeq find_seq(const AttnArgs& a, int b, int t, int tile) {
  AttnSeq s;
  if (!a.packed) {
    s.b = b;
    s.q0 = s.k0 = 0;
    s.qlen = a.qseq ? seq_at(a.qseq, a.seq_dt, b, a.Sq) : a.Sq;
    s.klen = a.kseq ? seq_at(a.kseq, a.seq_dt, b, a.Sk) : a.Sk;
    s.stat0 = (int64_t)b * ((a.Sq + 127) / 128 * 128);
    s.kstat0 = (int64_t)b * ((a.Sk + 127) / 128 * 128);
    s.tile = t;
    return s;
  }
  s.b = 0;
  s.tile = -1;
  const int lane = threadIdx.x & 31;
  const int n = a.packed;
  int before = 0;
  int last_q = 0, last_k = 0;  // ends of the pieces before this step of 32
  // piece i = base + lane ends at offset i: the rows before the first sequence,
  // the n sequences, the rows past the last one
  auto end_q = [&](int i) { return i <= n ? seq_at(a.qseq, a.seq_dt, i, a.Sq) : a.Sq; };
  auto end_k = [&](int i) { return i <= n ? seq_at(a.kseq, a.seq_dt, i, a.Sk) : a.Sk; };
  int next_q = end_q(lane), next_k = end_k(lane);
  for (int base = 0; base <= n + 1; base += 32) {
    const int i = base + lane;
    int q1 = max(next_q, last_q), k1 = max(next_k, last_k);
    next_q = end_q(i + 32);
    next_k = end_k(i + 32);
    int q0 = __shfl_up_sync(0xffffffffu, q1, 1), k0 = __shfl_up_sync(0xffffffffu, k1, 1);
    if (lane == 0) {
      q0 = last_q;
      k0 = last_k;
    }
    if (!__all_sync(0xffffffffu, q1 >= q0 && k1 >= k0)) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {  // running maxima: non-decreasing ends
        const int uq = __shfl_up_sync(0xffffffffu, q1, o), uk = __shfl_up_sync(0xffffffffu, k1, o);
        if (lane >= o) {
          q1 = max(q1, uq);
          k1 = max(k1, uk);
        }
      }
      const int uq = __shfl_up_sync(0xffffffffu, q1, 1), uk = __shfl_up_sync(0xffffffffu, k1, 1);
      q0 = lane == 0 ? last_q : uq;
      k0 = lane == 0 ? last_k : uk;
    }
    const int rows = BY_Q ? q1 - q0 : k1 - k0;
    const int tiles = i <= n + 1 ? (rows + tile - 1) / tile : 0;
    const int all = (int)__reduce_add_sync(0xffffffffu, (unsigned)tiles);
    if (t < before + all) {
      int upto = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, t < before + upto);
      const int src = __ffs(hit) - 1;
      s.q0 = __shfl_sync(0xffffffffu, q0, src);
      s.qlen = __shfl_sync(0xffffffffu, q1, src) - s.q0;
      s.k0 = __shfl_sync(0xffffffffu, k0, src);
      s.klen = __shfl_sync(0xffffffffu, k1, src) - s.k0;
      s.tile = t - before - __shfl_sync(0xffffffffu, upto - tiles, src);
      s.stat0 = attn_stat_base(s.q0, base + src);
      s.kstat0 = attn_stat_base(s.k0, base + src);
      // rows outside of the sequences: nothing is seen from or by them
      if (base + src == 0 || base + src == n + 1) (BY_Q ? s.klen : s.qlen) = 0;
      return s;
    }
    before += all;
    last_q = __shfl_sync(0xffffffffu, q1, 31);
    last_k = __shfl_sync(0xffffffffu, k1, 31);
  }
  return s;
}

// Whether every query of a sequence before row m1 sees at most kFineKeys keys.
__device__ __forceinline__ bool few_keys(const AttnArgs& a, const AttnSeq& s, int m1) {
  const int n = a.causal ? min(s.klen, m1 + s.klen - s.qlen) : s.klen;
  return (a.window ? min(n, a.window) : n) <= kFineKeys;
}

// Query i of a sequence sees key j when j < klen and, causal, j <= i + klen -
// qlen (the last query sees the last key), and, with a window, j > i + klen -
// qlen - window.
__device__ __forceinline__ bool see_keys(const AttnArgs& a, const AttnSeq& s, int i, int j) {
  const int at = i + s.klen - s.qlen;
  return i < s.qlen && j < s.klen && (!a.causal || j <= at) && (!a.window || j > at - a.window);
}

// Whether query i, which sees a key, sees no other.
__device__ __forceinline__ bool sees_one(const AttnArgs& a, const AttnSeq& s, int i) {
  const int at = i + s.klen - s.qlen;
  const int hi = a.causal ? min(s.klen, at + 1) : s.klen;
  return hi - (a.window ? max(0, at - a.window + 1) : 0) == 1;
}

// Keys [lo, hi) seen by any of the query rows [m0, m1) (m1 <= qlen).
__device__ __forceinline__ void key_range(const AttnArgs& a, const AttnSeq& s, int m0, int m1,
                                          int& lo, int& hi) {
  const int off = s.klen - s.qlen;
  hi = a.causal ? min(s.klen, m1 + off) : s.klen;
  lo = a.window ? max(0, m0 + off - a.window + 1) : 0;
  if (m1 <= m0 || hi <= lo) lo = hi = 0;
}

// Queries [lo, hi) that see any of the key rows [n0, n1) (n1 <= klen).
__device__ __forceinline__ void query_range(const AttnArgs& a, const AttnSeq& s, int n0, int n1,
                                            int& lo, int& hi) {
  const int off = s.klen - s.qlen;
  lo = a.causal ? max(0, n0 - off) : 0;
  hi = a.window ? min(s.qlen, n1 - off + a.window - 1) : s.qlen;
  if (n1 <= n0 || hi <= lo) lo = hi = 0;
}

// The first query of a sequence that sees a key, and the first key that a query
// sees. The ones before are used by nobody: where a tile holds some beside others,
// they are cleared in shared memory, since a probability of 0 times a NaN is a NaN.
__device__ __forceinline__ int first_query(const AttnArgs& a, const AttnSeq& s) {
  return a.causal ? max(0, s.qlen - s.klen) : 0;
}
__device__ __forceinline__ int first_key(const AttnArgs& a, const AttnSeq& s) {
  return a.window ? max(0, s.klen - s.qlen - a.window + 1) : 0;
}

// CW columns of a warp's 32 rows, thread = row, as 16-bit pairs w, to global
// memory: row r (< n) at dst + r * ss. Through 64 CW bytes of shared memory `sm`
// of the warp's own, so that a store instruction writes 32 / (CW / 8) rows'
// pieces of 2 CW bytes, not 16 bytes of each of 32 rows, which take it a cycle
// apiece (dQ of 8192 causal rows of 32/8 heads of 128: 620 us without, 585 with).
template <int CW, typename T>
__device__ __forceinline__ void store_rows(unsigned char* sm, const uint32_t (&w)[CW / 2], T* dst,
                                           int64_t ss, int n) {
  static_assert(CW == 64 || CW == 32, "a row is one line of shared memory, or half of one");
  constexpr int CH = CW / 8;  // 16-byte chunks of a row
  // where chunk c of row r lies: eight rows' fall in different banks
  auto at = [&](int r, int c) {
    return sm + r * (CW * 2) + ((c ^ (CH == 8 ? r & 7 : (r >> 1) & 3)) * 16);
  };
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    *reinterpret_cast<uint4*>(at(lane, c)) =
        make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int r = i * (32 / CH) + lane / CH, c = lane % CH;
    if (r < n)
      *reinterpret_cast<uint4*>(dst + r * ss + c * 8) = *reinterpret_cast<const uint4*>(at(r, c));
  }
  __syncwarp();
}

// Host launchers.
// attn_tc_*: 16-bit tensors, on the tensor cores.
template <typename T>
int attn_tc_fwd(const AttnArgs& a, int D, cudaStream_t st);
template <typename T>
int attn_tc_bwd(const AttnArgs& a, int D, cudaStream_t st);
// attn_rows_*: 16-bit dense tensors with few query rows; the workspace of
// `rows` rows (16 or 32) per key head, fp32 as well.
bool attn_rows_take(int64_t Sq, int64_t G, int64_t D, int64_t packed);
size_t attn_rows_workspace(int64_t B, int64_t Sk, int64_t Hk, int64_t D, int rows);
template <typename T>
int attn_rows_fwd(const AttnArgs& a, int D, void* ws, cudaStream_t st);
// attn_simt_*: fp32 tensors. attn_simt_rows_take: few query rows (16 rows in
// the workspace). simt_split: the backward takes fp32 partial sums of dk and
// dv, [2][B, Hq, Sk, D].
bool attn_simt_rows_take(int64_t Sq, int64_t G, int64_t packed);
bool simt_split(int64_t B, int64_t Sk, int64_t Hk, int64_t G, int64_t packed);
template <typename T>
int attn_simt_fwd(const AttnArgs& a, int D, void* ws, cudaStream_t st);
template <typename T>
int attn_simt_bwd(const AttnArgs& a, int D, void* partial, cudaStream_t st);
template <typename T>
int attn_stats(const AttnArgs& a, int D, cudaStream_t st);
// Floats of workspace that fp16's bounds of ds take.
inline int64_t attn_top_floats(int64_t B, int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hk,
                               int64_t packed) {
  const int64_t R = attn_stat_rows(B, Sq, packed);
  return Hq * (R + 2 * stat_tiles(R)) + Hk * stat_tiles(attn_stat_rows(B, Sk, packed));
}

template <typename F>
int attn_head_dim(int D, F&& f) {
  switch (D) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 256: return f(std::integral_constant<int, 256>{});
    default: return BLOTH_ERR_SHAPE;
  }
}

}  // namespace bloth
