// seq_attn.cu -- attention of packed sequences of queries over keys in the pages of a cache (16
// bits, or 8-bit codes with a scale per token and head) or in packed rows of their own.
//
//   o[i, h] = sum_j p_j v[j, g] / sum_j p_j,   p_j = exp(scale q.k_j - max)
//
// over the L keys of the query's sequence, or with a causal mask over those up to its own
// token, j <= L - n + i for query i of n; g = h / (H / Hkv). A row that sees no key is 0.
// The softmax is one pass over the keys with a running maximum m and sum l, in fp32 and base
// 2: p = 2^(s c - m) with c = scale log2(e). seq_step.cu has the kernel of few rows,
// seq_chunk.cu that of many; this file checks the arguments.
#include "seq_attn.cuh"

namespace srdit {
namespace sattn {

// Up to 16 query rows per key head over pages go to step_kernel, which streams the cache.
static Plan make_plan(const srdit_seq_attn_args& u, int max_q, int sms) {
  if (u.pages && static_cast<long long>(max_q) * (u.H / u.Hkv) <= 16) return plan_step(u, sms);
  return plan_chunk(u, sms);
}

// the arguments with max_q as it is used: 0 is all rows
static srdit_seq_attn_args with_max_q(const srdit_seq_attn_args& u) {
  srdit_seq_attn_args v = u;
  const int most = u.cu_q ? u.T : u.T / u.B;
  if (v.max_q == 0 || v.max_q > most) v.max_q = most;
  return v;
}

// 16-byte rows: base and the strides that are used; entries of an output are one place each
static int check_view(const void* p, const long long st[2], int n, int h, bool one_place) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return SRDIT_EALIGN;
  const int dims[2] = {n, h};
  for (int i = 0; i < 2; ++i) {
    if (dims[i] <= 1) continue;
    if (st[i] < 0 || st[i] % 8) return SRDIT_EALIGN;
    if (st[i] == 0 && (one_place || i == 0)) return SRDIT_EINVAL;
  }
  return 0;
}

// argument checks; 1: nothing to do
static int check(const srdit_seq_attn_args& a) {
  if (a.B < 0 || a.T < 0 || a.H < 0 || a.Hkv <= 0 || a.H % a.Hkv || a.max_q < 0 || a.max_kv < 0)
    return SRDIT_EINVAL;
  if (a.dtype != SRDIT_BF16 && a.dtype != SRDIT_FP16) return SRDIT_EINVAL;
  const bool paged = a.pages != nullptr;
  if (paged) {
    const int rc = check_pages(*a.pages);
    if (rc) return rc;
    if (a.pages->B != a.B || a.pages->Hkv != a.Hkv || a.pages->D != a.D ||
        a.pages->dtype != a.dtype)
      return SRDIT_EINVAL;
  } else if (a.Tk < 0) {
    return SRDIT_EINVAL;
  }
  if (a.B == 0 || a.T == 0 || a.H == 0) return 1;
  // (scores are taken in base 2: its factor has to be a number too)
  if (!a.q || !a.out || !(a.scale > 0.f) || !(a.scale * kLog2e <= 3.4028234e38f)) return SRDIT_EINVAL;
  if (a.H > 1 && a.q_stride[1] == 0) return SRDIT_EINVAL;  // (of the inputs, key heads may be repeated)
  if (!a.cu_q && a.T % a.B) return SRDIT_EINVAL;
  if (paged ? !a.kv_lens : (a.Tk > 0 && (!a.k || !a.v)) || (!a.cu_k && !a.cu_q && a.Tk % a.B))
    return SRDIT_EINVAL;
  if (a.D <= 0 || a.D > 128 || a.D % 8) return SRDIT_EUNSUPPORTED;
  if (static_cast<long long>(a.B) * a.Hkv > 65535 ||
      static_cast<long long>(a.T) * a.H > (1ll << 26) || (!paged && a.Tk > 0x7fffff00))
    return SRDIT_EUNSUPPORTED;
  int rc = check_view(a.q, a.q_stride, a.T, a.H, false);
  if (!rc) rc = check_view(a.out, a.o_stride, a.T, a.H, true);
  if (!rc && !paged) rc = check_view(a.k, a.k_stride, a.Tk, a.Hkv, false);
  if (!rc && !paged) rc = check_view(a.v, a.v_stride, a.Tk, a.Hkv, false);
  if (rc) return rc;
  if ((reinterpret_cast<uintptr_t>(a.cu_q) | reinterpret_cast<uintptr_t>(a.cu_k) |
       reinterpret_cast<uintptr_t>(a.kv_lens)) & 3u)
    return SRDIT_EALIGN;
  return 0;
}

}  // namespace sattn
}  // namespace srdit

using namespace srdit;

extern "C" int srdit_seq_attn_workspace(const srdit_seq_attn_args* args) {
  if (!args || sattn::check(*args) != 0) return 0;
  const srdit_seq_attn_args u = sattn::with_max_q(*args);
  const sattn::Plan p = sattn::make_plan(u, u.max_q, num_sms(device_here()));
  return static_cast<int>((p.ws_floats + 255) / 256);
}

extern "C" int srdit_seq_attn_way(const srdit_seq_attn_args* args) {
  if (!args || sattn::check(*args) != 0) return SRDIT_WAY_NONE;
  const srdit_seq_attn_args u = sattn::with_max_q(*args);
  const sattn::Plan p = sattn::make_plan(u, u.max_q, num_sms(device_here()));
  if (p.step) return p.shared ? SRDIT_WAY_STEP_SHARES : SRDIT_WAY_STEP;
  return p.ranged == 0 ? SRDIT_WAY_CHUNK : p.ranged == 1 ? SRDIT_WAY_CHUNK_SHARES : SRDIT_WAY_CHUNK_REST;
}

extern "C" int srdit_seq_attn(const srdit_seq_attn_args* args, cudaStream_t stream) {
  if (!args) return SRDIT_EINVAL;
  const int rc = sattn::check(*args);
  if (rc) return rc < 0 ? rc : 0;
  const srdit_seq_attn_args u = sattn::with_max_q(*args);
  const sattn::Plan p = sattn::make_plan(u, u.max_q, num_sms(device_here()));
  if (p.ws_floats > 0) {
    if (!u.workspace || u.workspace_bytes < 4 * p.ws_floats) return SRDIT_EINVAL;
    if (reinterpret_cast<uintptr_t>(u.workspace) & 15u) return SRDIT_EALIGN;
  }
  sattn::Args a = {};
  a.q = u.q;
  a.out = u.out;
  if (u.pages) {
    const srdit_kv_pages& c = *u.pages;
    a.table = table_of(c);
    a.scale[0] = c.k_scale;
    a.scale[1] = c.v_scale;
    for (int d = 0; d < 3; ++d) {
      a.ss[0][d] = c.ks_stride[d];
      a.ss[1][d] = c.vs_stride[d];
    }
  } else {
    a.keys = {u.cu_k ? u.cu_k : u.cu_q, u.Tk, u.Tk / u.B};
  }
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = u.q_stride[i];
    a.os[i] = u.o_stride[i];
  }
  a.rows = {u.cu_q, u.T, u.T / u.B};
  a.by_each = Divisor::of(u.cu_q ? 1 : u.T / u.B);
  a.lens = u.kv_lens;
  a.T = u.T;
  a.B = u.B;
  a.H = u.H;
  a.Hkv = u.Hkv;
  a.D = u.D;
  a.group = u.H / u.Hkv;
  a.causal = u.causal;
  a.max_q = u.max_q;
  a.c = u.scale * kLog2e;
  a.ws = static_cast<float*>(u.workspace);
  a.status = u.status;
  return p.step ? sattn::run_step(u, a, p, stream) : sattn::run_chunk(u, a, p, stream);
}
