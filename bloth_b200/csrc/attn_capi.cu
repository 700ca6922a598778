// extern "C" attention entry points declared in include/bloth_b200.h:
// argument validation, element-type dispatch, and which kernel takes a call.
#include <cmath>
#include <cstring>

#include "attn_impl.cuh"

using namespace bloth;

namespace {

// Rows of one sequence side: positions inside a sequence, window and lengths
// are held in 32 bits, and their sums must not overflow.
constexpr int64_t kMaxSeq = (int64_t)1 << 29;

int elem_bytes(int dt) { return dt == BLOTH_F32 ? 4 : 2; }

template <typename F>
int by_dtype(int dt, F&& f) {
  switch (dt) {
    case BLOTH_F32: return f(float{});
    case BLOTH_BF16: return f(__nv_bfloat16{});
    case BLOTH_F16: return f(__half{});
    default: return BLOTH_ERR_DTYPE;
  }
}

int check_sizes(int64_t B, int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hk, int64_t D,
                int64_t packed, int dtype) {
  if (dtype != BLOTH_F32 && dtype != BLOTH_BF16 && dtype != BLOTH_F16) return BLOTH_ERR_DTYPE;
  if (D != 64 && D != 128 && D != 256) return BLOTH_ERR_SHAPE;
  if (B < 0 || Sq < 0 || Sk < 0 || Hq < 1 || Hk < 1 || Hq % Hk != 0) return BLOTH_ERR_SHAPE;
  if (Sq > kMaxSeq || Sk > kMaxSeq || B > (1 << 20) || Hq > (1 << 16)) return BLOTH_ERR_SHAPE;
  if (packed < 0 || packed > (1 << 24) || (packed > 0 && B != 1)) return BLOTH_ERR_SHAPE;
  return BLOTH_OK;
}

// A head tensor of B x S x H rows that the kernels can address, filled into t.
// The stride of a single element, on which no address depends, may be anything.
int fill(HT& t, const void* p, const int64_t* st, int64_t B, int64_t S, int64_t H, int dtype) {
  if (p == nullptr || st == nullptr) return BLOTH_ERR_NULL;
  const int vec = 16 / elem_bytes(dtype);
  if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return BLOTH_ERR_ALIGN;
  const int64_t n[3] = {B, S, H};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && st[i] % vec != 0) return BLOTH_ERR_ALIGN;
  t.p = p;
  t.sb = B > 1 ? st[0] : 0;
  t.ss = S > 1 ? st[1] : 0;
  t.sh = H > 1 ? st[2] : 0;
  return BLOTH_OK;
}

int fill_common(AttnArgs& a, const void* q_seq, const void* k_seq, int seq_dtype, int64_t packed,
                int64_t B, int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hk, float scale, int causal,
                int64_t window) {
  if (!(scale > 0.f) || std::isinf(scale)) return BLOTH_ERR_ARG;
  if (window < 0 || (window > 0 && !causal)) return BLOTH_ERR_ARG;
  if ((q_seq || k_seq) && seq_dtype != BLOTH_I32 && seq_dtype != BLOTH_I64) return BLOTH_ERR_DTYPE;
  if (packed > 0 && (!q_seq || !k_seq)) return BLOTH_ERR_NULL;
  a.qseq = q_seq;
  a.kseq = k_seq;
  a.seq_dt = seq_dtype;
  a.packed = (int)packed;
  a.B = (int)B;
  a.Sq = (int)Sq;
  a.Sk = (int)Sk;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.G = (int)(Hq / Hk);
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  a.causal = causal ? 1 : 0;
  a.window = window > kMaxSeq ? 0 : (int)window;  // wider than any sequence: no window
  a.fault = nullptr;
  return BLOTH_OK;
}

cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

size_t bloth_attention_fwd_workspace_bytes(int64_t B, int64_t Sq, int64_t Sk, int64_t Hq,
                                           int64_t Hk, int64_t D, int64_t packed, int dtype) {
  if (check_sizes(B, Sq, Sk, Hq, Hk, D, packed, dtype)) return 0;
  const int64_t G = Hq / Hk;
  if (dtype == BLOTH_F32)
    return attn_simt_rows_take(Sq, G, packed) ? attn_rows_workspace(B, Sk, Hk, D, 16) : 0;
  if (attn_rows_take(Sq, G, D, packed))
    return attn_rows_workspace(B, Sk, Hk, D, Sq * G <= 16 ? 16 : 32);
  return 0;
}

int bloth_attention_fwd(const void* q, const int64_t* q_strides, const void* k,
                        const int64_t* k_strides, const void* v, const int64_t* v_strides,
                        void* out, const int64_t* out_strides, void* out_rest, float* lse,
                        const void* q_seq, const void* k_seq, int seq_dtype, int64_t packed,
                        int64_t B, int64_t Sq, int64_t Sk, int64_t Hq, int64_t Hk, int64_t D,
                        float scale, int causal, int64_t window, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
  int rc = check_sizes(B, Sq, Sk, Hq, Hk, D, packed, dtype);
  if (rc) return rc;
  AttnArgs a;
  std::memset(&a, 0, sizeof(a));
  if ((rc = fill_common(a, q_seq, k_seq, seq_dtype, packed, B, Sq, Sk, Hq, Hk, scale, causal,
                        window)))
    return rc;
  if (B == 0 || Sq == 0) return BLOTH_OK;
  if ((rc = fill(a.q, q, q_strides, B, Sq, Hq, dtype))) return rc;
  if (Sk > 0) {
    if ((rc = fill(a.k, k, k_strides, B, Sk, Hk, dtype))) return rc;
    if ((rc = fill(a.v, v, v_strides, B, Sk, Hk, dtype))) return rc;
  }
  if ((rc = fill(a.o, out, out_strides, B, Sq, Hq, dtype))) return rc;
  if (reinterpret_cast<uintptr_t>(out_rest) % 16 != 0) return BLOTH_ERR_ALIGN;
  a.rest = dtype == BLOTH_F32 ? nullptr : out_rest;
  a.lse = lse;
  const size_t need = bloth_attention_fwd_workspace_bytes(B, Sq, Sk, Hq, Hk, D, packed, dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return BLOTH_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return BLOTH_ERR_ALIGN;
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 4) {
      return attn_simt_fwd<T>(a, (int)D, workspace, as_stream(stream));
    } else {
      if (Sk > 0 && attn_rows_take(Sq, Hq / Hk, D, packed))
        return attn_rows_fwd<T>(a, (int)D, workspace, as_stream(stream));
      return attn_tc_fwd<T>(a, (int)D, as_stream(stream));
    }
  });
}

size_t bloth_attention_bwd_workspace_bytes(int64_t B, int64_t Sq, int64_t Sk, int64_t Hq,
                                           int64_t Hk, int64_t D, int64_t packed, int dtype) {
  if (check_sizes(B, Sq, Sk, Hq, Hk, D, packed, dtype)) return 0;
  int64_t n = 2 * Hq * attn_stat_rows(B, Sq, packed);
  if (dtype == BLOTH_F16) n += attn_top_floats(B, Sq, Sk, Hq, Hk, packed);
  if (dtype == BLOTH_F32 && simt_split(B, Sk, Hk, Hq / Hk, packed)) n += 2 * B * Hq * Sk * D;
  return (size_t)n * sizeof(float);
}

int bloth_attention_bwd(const void* dout, const int64_t* dout_strides, const void* q,
                        const int64_t* q_strides, const void* k, const int64_t* k_strides,
                        const void* v, const int64_t* v_strides, const void* out,
                        const int64_t* out_strides, const void* out_rest, const float* lse,
                        void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides,
                        void* dv, const int64_t* dv_strides, const void* q_seq,
                        const void* k_seq, int seq_dtype, int64_t packed, int64_t B, int64_t Sq,
                        int64_t Sk, int64_t Hq, int64_t Hk, int64_t D, float scale, int causal,
                        int64_t window, int dtype, void* workspace, size_t workspace_bytes,
                        void* stream) {
  int rc = check_sizes(B, Sq, Sk, Hq, Hk, D, packed, dtype);
  if (rc) return rc;
  AttnArgs a;
  std::memset(&a, 0, sizeof(a));
  if ((rc = fill_common(a, q_seq, k_seq, seq_dtype, packed, B, Sq, Sk, Hq, Hk, scale, causal,
                        window)))
    return rc;
  if ((dk == nullptr) != (dv == nullptr)) return BLOTH_ERR_NULL;
  if (B == 0 || (Sq == 0 && Sk == 0)) return BLOTH_OK;
  if (Sq > 0) {
    if ((rc = fill(a.dout, dout, dout_strides, B, Sq, Hq, dtype))) return rc;
    if ((rc = fill(a.q, q, q_strides, B, Sq, Hq, dtype))) return rc;
    if ((rc = fill(a.o, out, out_strides, B, Sq, Hq, dtype))) return rc;
    if (lse == nullptr) return BLOTH_ERR_NULL;
    if (dq != nullptr && (rc = fill(a.dq, dq, dq_strides, B, Sq, Hq, dtype))) return rc;
  }
  if (Sk > 0) {
    if ((rc = fill(a.k, k, k_strides, B, Sk, Hk, dtype))) return rc;
    if ((rc = fill(a.v, v, v_strides, B, Sk, Hk, dtype))) return rc;
    if (dk != nullptr && (rc = fill(a.dk, dk, dk_strides, B, Sk, Hk, dtype))) return rc;
    if (dv != nullptr && (rc = fill(a.dv, dv, dv_strides, B, Sk, Hk, dtype))) return rc;
  }
  const size_t need = bloth_attention_bwd_workspace_bytes(B, Sq, Sk, Hq, Hk, D, packed, dtype);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return BLOTH_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return BLOTH_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(out_rest) % 16 != 0) return BLOTH_ERR_ALIGN;
  a.rest = dtype == BLOTH_F32 ? nullptr : const_cast<void*>(out_rest);
  a.lse = const_cast<float*>(lse);
  a.R = attn_stat_rows(B, Sq, packed);
  a.lse2 = reinterpret_cast<float*>(workspace);
  a.delta = a.lse2 + Hq * a.R;
  if (dtype == BLOTH_F16) {
    a.RK = attn_stat_rows(B, Sk, packed);
    a.donorm = a.delta + Hq * a.R;
    a.qtop = reinterpret_cast<float2*>(a.donorm + Hq * a.R);
    a.vtop = reinterpret_cast<float*>(a.qtop + Hq * stat_tiles(a.R));
  }
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (Sq > 0) {
      const int r = attn_stats<T>(a, (int)D, as_stream(stream));
      if (r != BLOTH_OK) return r;
    }
    if constexpr (sizeof(T) == 4)
      return attn_simt_bwd<T>(a, (int)D, a.delta + Hq * a.R, as_stream(stream));
    else
      return attn_tc_bwd<T>(a, (int)D, as_stream(stream));
  });
}

}  // extern "C"
