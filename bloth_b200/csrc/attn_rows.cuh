// Attention forward for few query rows over many keys (single tokens, drafts,
// short tails): 16-bit dense tensors whose group of Hq / Hk heads and queries
// make at most 32 rows per key head.
//
// The rows of a key head (row r = query r / G of head h*G + r % G) are one
// operand of 16 or 32 rows, so K and V are read once for the whole group. The
// keys are split over CTAs in chunks of `chunk` keys and over the four warps
// of a CTA in strips of 16, each warp with its own ring of copies, running
// maximum and sums; nothing in the loop waits for another warp. The warps'
// results are joined in shared memory, the chunks' (fp32 sums, maximum and
// sum of exponentials in the workspace) by attn_join_kernel, in chunk order.
//
// Products are mma.sync m16n8k16: a strip of 16 keys of D = 128 is 8 KB and 32
// of them, while the strip's share of HBM time is 0.2 us of an SM. Bound: HBM,
// K and V once.
//
// Rows of K and V past the sequence's end, or below every query's window, are
// not read (zeros stand for them).
#pragma once

#include "attn_impl.cuh"
#include "tc.cuh"

namespace bloth {

constexpr int kRowsWarps = 4;
constexpr int kStrip = 16;

template <int D, int MT>
struct RowsCfg {
  static constexpr int ROWS = 16 * MT;
  static constexpr int STRIPB = kStrip * D * 2;  // bytes of a strip of K or of V
  // strips in flight per warp: 24 KB, or two of D = 256
  static constexpr int ST = D == 64 ? 6 : D == 128 ? 3 : 2;
  static constexpr int RING = kRowsWarps * ST * 2 * STRIPB;
  // the join of the warps: sums, maxima and sums of exponentials
  static constexpr int JOIN = kRowsWarps * ROWS * (D + 2) * 4;
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
  const int n = in ? 16 : 0;  // n < 16: the rest is filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The split of a call: chunks of `chunk` keys, `splits` of them; the partial
// results of chunk c of (b, h) are rows (c * B * Hk + b * Hk + h) * ROWS of
// `sums` [.][D] and of `stat` [.][2] (maximum in base 2, sum).
struct RowsPlan {
  int chunk, splits;
  float* sums;
  float* stat;
};

// Two neighbouring elements of one row of the result, and the row's lse.
template <typename T>
__device__ __forceinline__ void rows_out(const AttnArgs& a, int b, int h, int r, int c, float y0,
                                         float y1) {
  const int64_t at = (int64_t)b * a.o.sb + (int64_t)(h * a.G + r % a.G) * a.o.sh +
                     (int64_t)(r / a.G) * a.o.ss + c;
  T* out = reinterpret_cast<T*>(const_cast<void*>(a.o.p)) + at;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float2*>(out) = f2(y0, y1);
  } else {
    uint32_t hi, lo;
    split2<T, kRestUp<T>>(y0, y1, hi, lo);
    *reinterpret_cast<uint32_t*>(out) = hi;
    if (a.rest != nullptr) *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.rest) + at) = lo;
  }
}
__device__ __forceinline__ void rows_lse(const AttnArgs& a, int b, int h, int r, float m, float l) {
  if (a.lse != nullptr)
    a.lse[((int64_t)b * a.Hq + h * a.G + r % a.G) * a.Sq + r / a.G] =
        l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kRowsWarps * 32)
    attn_rows_kernel(const AttnArgs a, const RowsPlan pl) {
  using C = RowsCfg<D, MT>;
  constexpr int NC = D / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) unsigned char smem[];
  allow_dependent_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int bh = blockIdx.x % (a.B * a.Hk), split = blockIdx.x / (a.B * a.Hk);
  const int b = bh / a.Hk, h = bh % a.Hk;
  const AttnSeq s = find_seq<true>(a, b, 0, 1);
  const int off = s.klen - s.qlen, rows = a.Sq * a.G;
  int lo, hi;
  key_range(a, s, 0, s.qlen, lo, hi);
  const int seen0 = lo;  // the first key that a query sees
  lo = max(lo, split * pl.chunk) / kStrip * kStrip;
  hi = min(hi, (split + 1) * pl.chunk);
  const int strips = hi > lo ? (hi - lo + kStrip - 1) / kStrip : 0;
  const int mine = strips > warp ? (strips - warp + kRowsWarps - 1) / kRowsWarps : 0;

  const uint32_t ring = smem_addr(smem) + warp * C::ST * 2 * C::STRIPB;
  const T* kb = reinterpret_cast<const T*>(a.k.p) + (int64_t)b * a.k.sb + (int64_t)h * a.k.sh;
  const T* vb = reinterpret_cast<const T*>(a.v.p) + (int64_t)b * a.v.sb + (int64_t)h * a.v.sh;
  // strip i of this warp into slot i % ST; 16-byte chunk c of row r lies at
  // chunk c ^ (r & 7), so that eight rows' chunks fall in different banks
  auto issue = [&](int i) {
    if (i < mine) {
      const int j0 = lo + (warp + i * kRowsWarps) * kStrip;
      const uint32_t at = ring + (i % C::ST) * 2 * C::STRIPB;
#pragma unroll
      for (int u = 0; u < kStrip * NC / 32; ++u) {
        const int x = u * 32 + lane, r = x / NC, c = x % NC;
        const bool in = j0 + r < s.klen && j0 + r >= seen0;
        const int64_t row = in ? j0 + r : j0;  // j0 < klen: a row of this sequence
        const uint32_t d = at + r * (D * 2) + ((c ^ (r & 7)) * 16);
        cp16(d, kb + row * a.k.ss + c * 8, in);
        cp16(d + C::STRIPB, vb + row * a.v.ss + c * 8, in);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < C::ST - 1; ++i) issue(i);

  // the group's query rows, and each row's last key and first
  uint32_t qf[MT][D / 16][4];
  int to[MT][2], from[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = mt * 16 + g + u * 8;
      const bool in = r < rows;
      const int qi = in ? r / a.G : 0;
      const T* qp = reinterpret_cast<const T*>(a.q.p) + (int64_t)b * a.q.sb +
                    (int64_t)(h * a.G + (in ? r % a.G : 0)) * a.q.sh + (int64_t)qi * a.q.ss + 2 * t;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[mt][kk][u] = in ? __ldg(reinterpret_cast<const uint32_t*>(qp + kk * 16)) : 0u;
        qf[mt][kk][u + 2] = in ? __ldg(reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8)) : 0u;
      }
      to[mt][u] = qi < s.qlen ? (a.causal ? min(s.klen, qi + off + 1) : s.klen) : 0;
      from[mt][u] = a.window ? qi + off - a.window + 1 : 0;
    }
  const int all_to = a.causal ? min(s.klen, off + 1) : s.klen;  // seen by every query
  const int all_from = a.window ? a.Sq - 1 + off - a.window + 1 : 0;

  float m[MT][2], l[MT][2], acc[MT][D / 8][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt][0] = m[mt][1] = -INFINITY;
    l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[mt][n][e] = 0.f;
  }

  auto strip_loop = [&](auto few) {  // P as one term or two: see attn_fwd.cuh
    constexpr bool FINE = decltype(few)::value;
    for (int i = 0; i < mine; ++i) {
      issue(i + C::ST - 1);
      cp_wait<C::ST - 1>();
      __syncwarp();
      const int j0 = lo + (warp + i * kRowsWarps) * kStrip;
      const uint32_t at = ring + (i % C::ST) * 2 * C::STRIPB;
      float x[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[mt][n][e] = 0.f;
      {
        const int id = lane >> 3, r = (lane & 7) + 8 * (id >> 1);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          ldm4(at + r * (D * 2) + (((kk * 2 + (id & 1)) ^ (r & 7)) * 16), kf);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16<T>(x[mt][0], qf[mt][kk], kf[0], kf[1]);
            mma16<T>(x[mt][1], qf[mt][kk], kf[2], kf[3]);
          }
        }
      }
      const bool masked = j0 + kStrip > all_to || j0 < all_from || s.qlen < a.Sq;
      uint32_t pf[MT][4], rest[MT][4];
      bool move = false;
      float top[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& y = x[mt][n][2 * u + e];
              const int j = j0 + n * 8 + 2 * t + e;
              y = masked && (j >= to[mt][u] || j < from[mt][u]) ? -INFINITY : y * a.scale_log2;
              mx = fmaxf(mx, y);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          top[mt][u] = mx;
          move = move || mx > m[mt][u] + 8.f;  // as in the tile kernel: see attn_fwd.cuh
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float mn = fmaxf(m[mt][u], top[mt][u]);
            const float w = mn == m[mt][u] ? 1.f : ex2(m[mt][u] - mn);
            m[mt][u] = mn;
            l[mt][u] *= w;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              acc[mt][n][2 * u] *= w;
              acc[mt][n][2 * u + 1] *= w;
            }
          }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float base = m[mt][u] == -INFINITY ? 0.f : m[mt][u] - kFwdShift<T>;
          float p[4];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) p[2 * n + e] = ex2(x[mt][n][2 * u + e] - base);
          l[mt][u] += (p[0] + p[1]) + (p[2] + p[3]);
          split2<T>(p[0], p[1], pf[mt][u], rest[mt][u]);
          split2<T>(p[2], p[3], pf[mt][u + 2], rest[mt][u + 2]);
        }
      {
        const int id = lane >> 3, r = (lane & 7) + 8 * (id & 1);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          uint32_t vf[4];
          ldm4t(at + C::STRIPB + r * (D * 2) + (((dt * 2 + (id >> 1)) ^ (r & 7)) * 16), vf);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            mma16<T>(acc[mt][2 * dt], pf[mt], vf[0], vf[1]);
            mma16<T>(acc[mt][2 * dt + 1], pf[mt], vf[2], vf[3]);
            if (FINE) {
              mma16<T>(acc[mt][2 * dt], rest[mt], vf[0], vf[1]);
              mma16<T>(acc[mt][2 * dt + 1], rest[mt], vf[2], vf[3]);
            }
          }
        }
      }
      __syncwarp();  // the slot is free for the copy issued next
    }
  };
  if (few_keys(a, s, s.qlen)) strip_loop(std::true_type{});
  else strip_loop(std::false_type{});
  cp_wait<0>();

  // the four warps' rows through shared memory: [warp][row][D], then
  // [warp][row][2]; a lane's partial sum of exponentials is its quad's share
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
  float* stat = sums + kRowsWarps * C::ROWS * D;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = mt * 16 + g + u * 8;
      float q = l[mt][u];
      q += __shfl_xor_sync(0xffffffffu, q, 1);
      q += __shfl_xor_sync(0xffffffffu, q, 2);
      float* row = sums + (warp * C::ROWS + r) * D;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2*>(row + n * 8 + 2 * t) =
            f2(acc[mt][n][2 * u], acc[mt][n][2 * u + 1]);
      if (t == 0) {
        stat[(warp * C::ROWS + r) * 2] = m[mt][u] - kFwdShift<T>;
        stat[(warp * C::ROWS + r) * 2 + 1] = q;
      }
    }
  __syncthreads();
  const int64_t part = ((int64_t)split * a.B * a.Hk + bh) * C::ROWS;
  for (int r = warp; r < rows; r += kRowsWarps) {
    float mm = -INFINITY, w[kRowsWarps], ll = 0.f;
#pragma unroll
    for (int i = 0; i < kRowsWarps; ++i) mm = fmaxf(mm, stat[(i * C::ROWS + r) * 2]);
#pragma unroll
    for (int i = 0; i < kRowsWarps; ++i) {
      const float mi = stat[(i * C::ROWS + r) * 2];
      w[i] = mi == -INFINITY ? 0.f : ex2(mi - mm);
      ll = fmaf(stat[(i * C::ROWS + r) * 2 + 1], w[i], ll);
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;
    for (int c = lane * 2; c < D; c += 64) {
      float2 y = f2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kRowsWarps; ++i) {
        const float2 v = *reinterpret_cast<const float2*>(sums + (i * C::ROWS + r) * D + c);
        y = f2_fma(v, f2s(w[i]), y);
      }
      if (pl.splits == 1)
        rows_out<T>(a, b, h, r, c, y.x * inv, y.y * inv);
      else
        *reinterpret_cast<float2*>(pl.sums + (part + r) * D + c) = y;
    }
    if (lane == 0) {
      if (pl.splits == 1) {
        rows_lse(a, b, h, r, mm, ll);
      } else {
        pl.stat[(part + r) * 2] = mm;
        pl.stat[(part + r) * 2 + 1] = ll;
      }
    }
  }
}

// The chunks' partial rows to one row: a CTA per row, whose four warps take the
// chunks in turn, their sums then added in warp order.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a, const RowsPlan pl,
                                                        int part_rows) {
  constexpr int V = D / 32;
  __shared__ float sums[4][D + 1];
  const int rows = a.Sq * a.G, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int bh = (int)(blockIdx.x / rows), r = (int)(blockIdx.x % rows);
  const int64_t step = (int64_t)a.B * a.Hk * part_rows;
  const int64_t p0 = (int64_t)bh * part_rows + r;
  wait_for_prior_grid();
  float mm = -INFINITY;
  for (int c = lane; c < pl.splits; c += 32) mm = fmaxf(mm, pl.stat[(p0 + c * step) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  float y[V], ll = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) y[e] = 0.f;
#pragma unroll 4
  for (int c = warp; c < pl.splits; c += 4) {
    const int64_t p = p0 + c * step;
    const float2 st = *reinterpret_cast<const float2*>(pl.stat + p * 2);
    const float w = st.x == -INFINITY ? 0.f : ex2(st.x - mm);
    ll = fmaf(st.y, w, ll);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(pl.sums + p * D + lane * V + e);
      y[e] = fmaf(v.x, w, y[e]);
      y[e + 1] = fmaf(v.y, w, y[e + 1]);
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) sums[warp][lane * V + e] = y[e];
  if (lane == 0) sums[warp][D] = ll;
  __syncthreads();
  const float l = (sums[0][D] + sums[1][D]) + (sums[2][D] + sums[3][D]);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int c = 2 * threadIdx.x; c < D; c += 256) {
    const float y0 = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
    const float y1 = (sums[0][c + 1] + sums[1][c + 1]) + (sums[2][c + 1] + sums[3][c + 1]);
    rows_out<T>(a, bh / a.Hk, bh % a.Hk, r, c, y0 * inv, y1 * inv);
  }
  if (threadIdx.x == 0) rows_lse(a, bh / a.Hk, bh % a.Hk, r, mm, l);
}

// Keys per chunk and chunks: as many CTAs as fill the device twice over (two
// are resident per SM), but at least 256 keys each, a ring's worth of strips for
// every warp several times over. 16 tokens over caches of 2048 to 8192 rows of
// 8 heads of 128: once over 90 us, twice 77, four times 85 (more partial rows
// to write and join); one token over 65536 rows: 54, 60 and 70 us.
inline void rows_split(int64_t pairs, int64_t Sk, int64_t& chunk, int64_t& splits) {
  const int64_t want = (4 * (int64_t)device_sm_count() + pairs - 1) / pairs;
  chunk = ((Sk + want - 1) / want + 63) / 64 * 64;
  if (chunk < 256) chunk = 256;
  splits = Sk > 0 ? (Sk + chunk - 1) / chunk : 1;
}

// The plan of a call whose key heads have `rows` rows each.
inline RowsPlan rows_plan(const AttnArgs& a, int rows, int D, void* ws) {
  int64_t chunk, splits;
  const int64_t pairs = (int64_t)a.B * a.Hk;
  rows_split(pairs, a.Sk, chunk, splits);
  RowsPlan pl;
  pl.chunk = (int)chunk;
  pl.splits = (int)splits;
  pl.sums = reinterpret_cast<float*>(ws);
  pl.stat = pl.sums + splits * pairs * rows * D;
  return pl;
}

template <typename T, int D>
int launch_attn_join(const AttnArgs& a, const RowsPlan& pl, int rows, cudaStream_t st) {
  const int64_t n = (int64_t)a.B * a.Hk * a.Sq * a.G;
  if (n > 0x7fffffff) return BLOTH_ERR_SHAPE;
  return launched(
      launch_dependent(attn_join_kernel<T, D>, (unsigned)n, 128u, 0, st, a, pl, rows));
}

template <typename T, int D, int MT>
int launch_attn_rows(const AttnArgs& a, void* ws, cudaStream_t st) {
  using C = RowsCfg<D, MT>;
  const RowsPlan pl = rows_plan(a, C::ROWS, D, ws);
  auto kern = attn_rows_kernel<T, D, MT>;
  int rc = prepare_smem((const void*)kern, C::SMEM);
  if (rc != BLOTH_OK) return rc;
  const int64_t grid = (int64_t)pl.splits * a.B * a.Hk;
  if (grid > 0x7fffffff) return BLOTH_ERR_SHAPE;
  rc = launched(launch_ex(kern, (unsigned)grid, kRowsWarps * 32, C::SMEM, st, a, pl));
  if (rc != BLOTH_OK || pl.splits == 1) return rc;
  return launch_attn_join<T, D>(a, pl, C::ROWS, st);
}

}  // namespace bloth
