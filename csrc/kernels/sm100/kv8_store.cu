// Writing rows into 8-bit key-value pages and reading pages back (format: kv8.cuh).
//
// Counterparts in the reference: quant_store_k / dequant_rows_k (kernels/src/kv_tier.cu:32-86), the INT8 KV of its dense
// layers (kernels/m1/m1_dense8.cu:65-126) and qk_prep_kernel (kernels/src/rope.cu:109-189), which here is one kernel with
// the quantisation: a row goes from the fused qkv product to its page without a bf16 copy between.
#include <algorithm>

#include "kv8.cuh"

namespace b2 {

struct Kv8StoreArgs {
  const bf16* qkv; long ld;                 // [n][(hq + 2 hkv) * hd]: q heads, k heads, v heads
  int n, hq, hkv;
  const float* inv_freq;                    // [hd / 2]
  const int* tok_pos;                       // slot of the row inside its sequence
  const int* rope_pos;                      // optional rotary position (differs from the slot for tree drafts)
  const int* rope_pos3;                     // optional [3][n] (time, height, width), with
  const unsigned char* pair_axis;           // [hd / 2] the axis of every rotary pair
  const int* tok_seq; int n_seq;
  const int* block_table; int bt_ld, bt_cols;
  uint8_t* pool; int n_pages;
  bf16* q_out; long ldq;
  int* status;
};

struct Kv8ReadArgs {
  const uint8_t* pool; int n_pages, hkv;
  const int* pages; int n_out; long n_tokens;
  bf16* out;
  int* status;
};

namespace {

__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 v;
  uint32_t* w = &v.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) { const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t*>(&b); }
  return v;
}

// Rotation (pairs i, i + hd/2) by pos * inv_freq, q rounded once to bf16, k and v quantised from fp32:
//     (lo, hi) -> (lo cos - hi sin, hi cos + lo sin);    scale = max(max |x| / top, 2^-64), code = round(x / scale)
// HD / 16 lanes hold a head, eight rotary pairs each, so a warp takes 32 / (HD / 16) heads at a time ("a turn") and has the next turn's
// loads under way meanwhile.  `parts` CTAs share a token, or a CTA has `toks` (one or two); each takes a token's sines and cosines once.
// Bound by the chain of launch, positions, sines and rows for few tokens (one token of 64 q and 8 KV heads of 128: 2.4 us, 48 tokens
// 2.5 us), by memory for many: 2048 tokens 17.1 us, 80 MB at 4.7 TB/s (19.4 with a token a CTA; two turns under way were slower).
template <int HD, int FMT>
__global__ void __launch_bounds__(256) kv8_store_kernel(const Kv8StoreArgs a, int parts, int toks) {
  constexpr int LPH = HD / 16, HPW = 32 / LPH, HALF = HD / 2;
  __shared__ __align__(16) float sh_c[2][HALF], sh_s[2][HALF];
  __shared__ int sh_page[2], sh_slot[2];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, l = lane % LPH, sub = lane / LPH;
  const int tok0 = blockIdx.x / parts * toks, part = blockIdx.x % parts;
  const int heads = a.hq + 2 * a.hkv, turns = (heads + HPW - 1) / HPW, all = min(toks, a.n - tok0) * turns;
  int turn = part * 8 + (threadIdx.x >> 5);
  uint4 lo8 = make_uint4(0u, 0u, 0u, 0u), hi8 = lo8;
  auto load = [&](int t) {
    const int u = t >= turns, head = (t - u * turns) * HPW + sub;
    if (t < all && head < heads) {
      const bf16* src = a.qkv + (size_t)(tok0 + u) * a.ld + (size_t)head * HD + l * 8;
      lo8 = ld_nc_v4(src);
      hi8 = ld_nc_v4(src + HALF);
    }
  };
  load(turn);

  // The angle in turns, in 64 bits: a 32-bit product of a position of 100000 and a frequency near one is off by several
  // thousandths of a radian.  Its fraction goes to sincospi, which needs no argument reduction of its own.
  const int mine = threadIdx.x / HALF, tok1 = tok0 + mine;
  if (mine < toks && tok1 < a.n) {
    const int i = threadIdx.x % HALF;
    int p = a.rope_pos ? a.rope_pos[tok1] : a.tok_pos[tok1];
    if (a.rope_pos3) p = a.rope_pos3[(size_t)min((int)a.pair_axis[i], 2) * a.n + tok1];
    double t = (double)p * (double)a.inv_freq[i] * 0.15915494309189535;
    t -= rint(t);
    sincospif((float)(2.0 * t), &sh_s[mine][i], &sh_c[mine][i]);
  }
  if (threadIdx.x >= 254 && tok0 + (int)threadIdx.x - 254 < a.n && (int)threadIdx.x - 254 < toks) {
    const int u = threadIdx.x - 254, pos = a.tok_pos[tok0 + u], seq = a.tok_seq[tok0 + u];
    int page = -1;
    if (pos >= 0 && pos / kKv8Page < a.bt_cols && seq >= 0 && seq < a.n_seq) page = a.block_table[(size_t)seq * a.bt_ld + pos / kKv8Page];
    if (page >= a.n_pages) page = -1;
    if (page < 0 && part == 0) atomicExch(a.status, (int)B2_ERR_BOUNDS);
    sh_page[u] = page;
    sh_slot[u] = pos % kKv8Page;
  }
  __syncthreads();

  for (; turn < all; turn += 8 * parts) {
    const int u = turn >= turns, head = (turn - u * turns) * HPW + sub, tok = tok0 + u, page = sh_page[u];
    const bool stored = page >= 0;
    float lo[8], hi[8];
    unpack8(lo8, lo);
    unpack8(hi8, hi);
    load(turn + 8 * parts);
    if (head < a.hq + a.hkv) {
      const float4* c4 = reinterpret_cast<const float4*>(&sh_c[u][l * 8]);
      const float4* s4 = reinterpret_cast<const float4*>(&sh_s[u][l * 8]);
      const float4 cv[2] = {c4[0], c4[1]}, sv[2] = {s4[0], s4[1]};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = lo[i], y = hi[i], c = (&cv[i >> 2].x)[i & 3], s = (&sv[i >> 2].x)[i & 3];
        lo[i] = x * c - y * s;
        hi[i] = y * c + x * s;
      }
    }
    if (head < a.hq) {
      bf16* dst = a.q_out + (size_t)tok * a.ldq + (size_t)head * HD + l * 8;
      *reinterpret_cast<uint4*>(dst) = pack8(lo);
      *reinterpret_cast<uint4*>(dst + HALF) = pack8(hi);
    }
    if (head - sub + HPW <= a.hq) continue;            // q heads only, for the whole warp
    // the largest magnitude, compared as bits: a NaN's are above an infinity's, so neither is lost
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = max(mx, max(__float_as_uint(lo[i]) & 0x7fffffffu, __float_as_uint(hi[i]) & 0x7fffffffu));
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (head >= heads || head < a.hq || !stored) continue;
    const bool is_v = head >= a.hq + a.hkv;
    const int kvh = head - a.hq - (is_v ? a.hkv : 0), slot = sh_slot[u];
    const float scale = fmaxf(__fdiv_rn(__uint_as_float(mx), FMT == KV8_INT8 ? 127.f : 448.f), kKv8MinScale);
    const bool finite = mx < 0x7f800000u;
    uint32_t clo[2] = {0u, 0u}, chi[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!finite) lo[i] = hi[i] = 0.f;            // codes stay numbers: what tells of the row is its scale
      clo[i >> 2] |= kv8_code<FMT>(__fdiv_rn(lo[i], scale)) << (8 * (i & 3));
      chi[i >> 2] |= kv8_code<FMT>(__fdiv_rn(hi[i], scale)) << (8 * (i & 3));
    }
    uint8_t* blk = a.pool + ((size_t)page * a.hkv + kvh) * kv8_block_bytes(HD);
    uint8_t* codes = blk + (is_v ? kKv8Page * HD : 0) + slot * HD + l * 8;
    *reinterpret_cast<uint2*>(codes) = make_uint2(clo[0], clo[1]);
    *reinterpret_cast<uint2*>(codes + HALF) = make_uint2(chi[0], chi[1]);
    if (l == 0) reinterpret_cast<float*>(blk + 2 * kKv8Page * HD)[slot * 2 + is_v] = finite ? scale : __uint_as_float(0x7fffffffu);
  }
}

// Pages [n_out] of the pool as bf16 pages [n_out][2][hkv][16][hd], code * scale rounded once; slots from n_tokens on are zeros.  A CTA
// expands a page of a KV head, a thread eight codes of K and eight of V, so that a warp's stores are whole lines.  Bound by memory: 65536
// tokens of 8 heads of 128 68 us (407 MB, 5.95 TB/s, 0.92 of a copy's rate; 72 with blocks of 256 threads over pages and heads at large).
template <int HD, int FMT>
__global__ void __launch_bounds__(2 * HD) kv8_read_kernel(const Kv8ReadArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const int pi = blockIdx.x, h = blockIdx.y, c = threadIdx.x, row = c / (HD / 8);
  const bool live = (long)pi * kKv8Page + row < a.n_tokens;
  const int page = live ? a.pages[pi] : -1;
  const bool there = page >= 0 && page < a.n_pages;
  if (live && !there && c == 0) atomicExch(a.status, (int)B2_ERR_BOUNDS);
  uint2 w[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
  uint2 sc = make_uint2(0u, 0u);
  if (there) {
    const uint8_t* blk = a.pool + ((size_t)page * a.hkv + h) * kv8_block_bytes(HD);
    w[0] = ld_nc_v2(blk + c * 8);
    w[1] = ld_nc_v2(blk + kKv8Page * HD + c * 8);
    sc = ld_nc_v2(blk + 2 * kKv8Page * HD + row * 8);
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const float s = __uint_as_float(kv ? sc.y : sc.x);
    float f[8];
    kv8_values<FMT>(w[kv].x, f);
    kv8_values<FMT>(w[kv].y, f + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = there ? __fmul_rn(f[i], s) : 0.f;
    *reinterpret_cast<uint4*>(a.out + (((size_t)pi * 2 + kv) * a.hkv + h) * kKv8Page * HD + c * 8) = pack8(f);
  }
}

template <class K, class... A>
int launch(K kernel, dim3 blocks, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks; cfg.blockDim = dim3(threads); cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? B2_OK : B2_ERR_LAUNCH;
}

}  // namespace
}  // namespace b2

using namespace b2;

B2_API int b2_kv8_store(const Kv8StoreArgs* args, int hd, int fmt, cudaStream_t st) {
  const Kv8StoreArgs& a = *args;
  if (a.n < 1 || a.hq < 1 || a.hkv < 1 || a.n_seq < 1 || a.bt_cols < 1 || a.n_pages < 1) return B2_ERR_ARG;
  if ((hd != 64 && hd != 128) || (fmt != KV8_INT8 && fmt != KV8_FP8) || a.ld % 8 || a.ldq % 8) return B2_ERR_ARG;
  const int hpw = 32 / (hd / 16), turns = (a.hq + 2 * a.hkv + hpw - 1) / hpw;
  // few tokens: a CTA for eight turns, so that no warp has two; many: a CTA for a token, whose sines and cosines are taken once
  const int most = (turns + 7) / 8, parts = (long)a.n * most <= 148 * 4 ? most : 1;
  // two tokens a CTA where that leaves every SM one: 2048 tokens of 64 + 16 heads (two and a half turns a warp) 17.1 us instead of 19.5,
  // 4000 of 24 + 8 (one turn a warp) 17.8 instead of 21.3; 48 tokens 3.4 instead of 2.5
  const int toks = parts == 1 && a.n >= 2 * 148 ? 2 : 1;
  const long blocks = ((long)a.n + toks - 1) / toks * parts;
  if (blocks > 0x7fffffffl) return B2_ERR_ARG;
  auto k = hd == 128 ? (fmt == KV8_INT8 ? kv8_store_kernel<128, KV8_INT8> : kv8_store_kernel<128, KV8_FP8>)
                     : (fmt == KV8_INT8 ? kv8_store_kernel<64, KV8_INT8> : kv8_store_kernel<64, KV8_FP8>);
  return launch(k, dim3((unsigned)blocks), 256, st, a, parts, toks);
}

B2_API int b2_kv8_read(const Kv8ReadArgs* args, int hd, int fmt, cudaStream_t st) {
  const Kv8ReadArgs& a = *args;
  if (a.n_out < 1 || a.hkv < 1 || a.hkv > 65535 || a.n_pages < 1 || a.n_tokens < 0) return B2_ERR_ARG;
  if ((hd != 64 && hd != 128) || (fmt != KV8_INT8 && fmt != KV8_FP8)) return B2_ERR_ARG;
  auto k = hd == 128 ? (fmt == KV8_INT8 ? kv8_read_kernel<128, KV8_INT8> : kv8_read_kernel<128, KV8_FP8>)
                     : (fmt == KV8_INT8 ? kv8_read_kernel<64, KV8_INT8> : kv8_read_kernel<64, KV8_FP8>);
  return launch(k, dim3(a.n_out, a.hkv), 2 * hd, st, a);
}
