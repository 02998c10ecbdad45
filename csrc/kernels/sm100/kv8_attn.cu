// Attention of new tokens over 8-bit key-value pages (format: kv8.cuh): decode steps, verify blocks (causal or tree mask)
// and short prefill chunks.  Counterpart in the reference: the INT8 KV of its dense layers, which expands tiles to bf16 and
// attends to those (kernels/m1/m1_dense8.cu:65-126); here the codes go straight into the products.
//
// o = sum_j p_j vs_j vc_j / sum_j p_j,  p_j = exp(q . kc_j ks_j / sqrt(hd) - m)   over the keys that the row sees.
#include "kv8.cuh"

namespace b2 {

struct Kv8AttnArgs {
  const bf16* q; long ldq;                  // [n_tok][hq * hd], RoPE applied
  const uint8_t* pool; int n_pages;
  const int* block_table; int bt_ld, bt_cols, n_seq;
  const int* grp_tok0; const int* grp_cnt; int n_groups;   // consecutive rows of one sequence, at most 32
  const int* tok_pos; const int* tok_seq; int n_tok;
  const unsigned* tree_mask;                // optional [n_tok]: bit j set = the row sees the group's j-th row
  int hq, hkv;
  float scale_log2;                         // log2(e) / sqrt(hd)
  bf16* out; long ldo;
  int* status;
};

namespace {

// One warp per (group, q head): row by row, key by key.
template <int HD, int FMT>
__global__ void __launch_bounds__(128) kv8_attn_kernel(const Kv8AttnArgs a) {
  constexpr int PER = HD / 32;
  pdl_wait();
  pdl_launch_dependents();
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int grp = (int)(item / a.hq), head = (int)(item % a.hq), kvh = head / (a.hq / a.hkv);
  if (grp >= a.n_groups) return;
  const int tok0 = a.grp_tok0[grp], cnt = a.grp_cnt[grp];
  if (cnt < 1) return;
  bool ok = cnt <= 32 && tok0 >= 0 && tok0 <= a.n_tok - cnt;
  const int seq = ok ? a.tok_seq[tok0] : -1;
  ok = ok && seq >= 0 && seq < a.n_seq;
  const int first = ok ? a.tok_pos[tok0] : 0, last = ok ? a.tok_pos[tok0 + cnt - 1] : 0;
  ok = ok && last < a.bt_cols * kKv8Page;
  if (!ok) { if (lane == 0) atomicExch(a.status, (int)B2_ERR_BOUNDS); return; }
  for (int r = 0; r < cnt; ++r) {
    const int tok = tok0 + r, pos = min(a.tok_pos[tok], last);
    const unsigned mask = a.tree_mask ? a.tree_mask[tok] : 0u;
    float qv[PER], o[PER], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) { qv[i] = __bfloat162float(a.q[(size_t)tok * a.ldq + (size_t)head * HD + lane * PER + i]); o[i] = 0.f; }
    for (int key = 0; key <= pos; ++key) {
      if (a.tree_mask && key >= first && (key - first > 31 || !((mask >> (key - first)) & 1u))) continue;
      const int page = a.block_table[(size_t)seq * a.bt_ld + key / kKv8Page], slot = key % kKv8Page;
      if (page < 0 || page >= a.n_pages) { if (lane == 0) atomicExch(a.status, (int)B2_ERR_BOUNDS); continue; }
      const uint8_t* blk = a.pool + ((size_t)page * a.hkv + kvh) * kv8_block_bytes(HD);
      const float2 sc = reinterpret_cast<const float2*>(blk + 2 * kKv8Page * HD)[slot];
      const uint8_t* kp = blk + slot * HD + lane * PER;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) s = fmaf(qv[i], kv8_value<FMT>(kp[i]), s);
      s = warp_sum(s) * sc.x * a.scale_log2;
      const float mn = fmaxf(m, s), corr = exp2f(m - mn), p = exp2f(s - mn);
      l = l * corr + p;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = o[i] * corr + p * (kv8_value<FMT>(kp[kKv8Page * HD + i]) * sc.y);
      m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < PER; ++i) a.out[(size_t)tok * a.ldo + (size_t)head * HD + lane * PER + i] = __float2bfloat16_rn(o[i] * inv);
  }
}

}  // namespace
}  // namespace b2

using namespace b2;

B2_API int b2_kv8_attn(const Kv8AttnArgs* args, int hd, int fmt, cudaStream_t st) {
  const Kv8AttnArgs& a = *args;
  if (a.n_groups < 1 || a.n_tok < 1 || a.hkv < 1 || a.hq < 1 || a.hq % a.hkv || a.n_seq < 1 || a.bt_cols < 1 || a.n_pages < 1) return B2_ERR_ARG;
  if ((hd != 64 && hd != 128) || (fmt != KV8_INT8 && fmt != KV8_FP8) || a.ldq % 8 || a.ldo % 8) return B2_ERR_ARG;
  const long blocks = ((long)a.n_groups * a.hq + 3) / 4;
  if (blocks > 0x7fffffffl || a.bt_cols > (1 << 26)) return B2_ERR_ARG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks); cfg.blockDim = dim3(128); cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  auto k = hd == 128 ? (fmt == KV8_INT8 ? kv8_attn_kernel<128, KV8_INT8> : kv8_attn_kernel<128, KV8_FP8>)
                     : (fmt == KV8_INT8 ? kv8_attn_kernel<64, KV8_INT8> : kv8_attn_kernel<64, KV8_FP8>);
  return cudaLaunchKernelEx(&cfg, k, a) == cudaSuccess ? B2_OK : B2_ERR_LAUNCH;
}
