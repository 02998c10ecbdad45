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

namespace {

__device__ __forceinline__ void unpack4(uint2 v, float (&f)[4]) {
  const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&v.x), b = *reinterpret_cast<const __nv_bfloat162*>(&v.y);
  f[0] = __low2float(a); f[1] = __high2float(a); f[2] = __low2float(b); f[3] = __high2float(b);
}
__device__ __forceinline__ uint2 pack4(const float (&f)[4]) {
  uint2 v;
  *reinterpret_cast<__nv_bfloat162*>(&v.x) = __floats2bfloat162_rn(f[0], f[1]);
  *reinterpret_cast<__nv_bfloat162*>(&v.y) = __floats2bfloat162_rn(f[2], f[3]);
  return v;
}

// Rotation (pairs i, i + hd/2) by pos * inv_freq, q rounded once to bf16, k and v quantised from fp32.
// HD / 8 lanes hold a head, four rotary pairs each, so a warp takes 32 / (HD / 8) heads at a time.
template <int HD, int FMT>
__global__ void __launch_bounds__(256) kv8_store_kernel(const Kv8StoreArgs a, int warps_per_tok) {
  constexpr int LPH = HD / 8, HPW = 32 / LPH, HALF = HD / 2;
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, l = lane % LPH;
  const long gw = (long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int tok = (int)(gw / warps_per_tok), w = (int)(gw % warps_per_tok);
  if (tok >= a.n) return;
  const int pos = a.tok_pos[tok], seq = a.tok_seq[tok];
  int page = -1;
  if (pos >= 0 && pos / kKv8Page < a.bt_cols && seq >= 0 && seq < a.n_seq) page = a.block_table[(size_t)seq * a.bt_ld + pos / kKv8Page];
  const bool stored = page >= 0 && page < a.n_pages;
  if (!stored && lane == 0) atomicExch(a.status, (int)B2_ERR_BOUNDS);

  // The angle in turns, in 64 bits: a 32-bit product of a position of 100000 and a frequency near one is off by several
  // thousandths of a radian.  Its fraction goes to sincospi, which needs no argument reduction of its own.
  float c[4], s[4];
  const int rpos = a.rope_pos ? a.rope_pos[tok] : pos;
  const float4 f4 = *reinterpret_cast<const float4*>(a.inv_freq + l * 4);
  const float fr[4] = {f4.x, f4.y, f4.z, f4.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = a.rope_pos3 ? a.rope_pos3[(size_t)min((int)a.pair_axis[l * 4 + i], 2) * a.n + tok] : rpos;
    double t = (double)p * (double)fr[i] * 0.15915494309189535;
    t -= rint(t);
    sincospif((float)(2.0 * t), &s[i], &c[i]);
  }

  const int heads = a.hq + 2 * a.hkv;
  const int turns = (heads + HPW - 1) / HPW;
  for (int turn = w; turn < turns; turn += warps_per_tok) {
    const int head = turn * HPW + lane / LPH;
    const bool live = head < heads;
    float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
      const bf16* src = a.qkv + (size_t)tok * a.ld + (size_t)head * HD + l * 4;
      unpack4(*reinterpret_cast<const uint2*>(src), lo);
      unpack4(*reinterpret_cast<const uint2*>(src + HALF), hi);
    }
    if (head < a.hq + a.hkv) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = lo[i], y = hi[i];
        lo[i] = x * c[i] - y * s[i];
        hi[i] = y * c[i] + x * s[i];
      }
    }
    if (live && head < a.hq) {
      bf16* dst = a.q_out + (size_t)tok * a.ldq + (size_t)head * HD + l * 4;
      *reinterpret_cast<uint2*>(dst) = pack4(lo);
      *reinterpret_cast<uint2*>(dst + HALF) = pack4(hi);
    }
    // the largest magnitude, compared as bits: a NaN's are above an infinity's, so neither is lost
    uint32_t mx = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = max(mx, max(__float_as_uint(lo[i]) & 0x7fffffffu, __float_as_uint(hi[i]) & 0x7fffffffu));
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (!live || head < a.hq || !stored) continue;
    const bool is_v = head >= a.hq + a.hkv;
    const int kvh = head - a.hq - (is_v ? a.hkv : 0), slot = pos % kKv8Page;
    const float scale = fmaxf(__fdiv_rn(__uint_as_float(mx), FMT == KV8_INT8 ? 127.f : 448.f), kKv8MinScale);
    const bool finite = mx < 0x7f800000u;
    uint32_t clo = 0, chi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!finite) lo[i] = hi[i] = 0.f;            // codes stay numbers: what tells of the row is its scale
      clo |= kv8_code<FMT>(__fdiv_rn(lo[i], scale)) << (8 * i);
      chi |= kv8_code<FMT>(__fdiv_rn(hi[i], scale)) << (8 * i);
    }
    uint8_t* blk = a.pool + ((size_t)page * a.hkv + kvh) * kv8_block_bytes(HD);
    uint8_t* row = blk + (is_v ? kKv8Page * HD : 0) + slot * HD + l * 4;
    *reinterpret_cast<uint32_t*>(row) = clo;
    *reinterpret_cast<uint32_t*>(row + HALF) = chi;
    if (l == 0) reinterpret_cast<float*>(blk + 2 * kKv8Page * HD)[slot * 2 + is_v] = finite ? scale : __uint_as_float(0x7fffffffu);
  }
}

// Pages [n_out] of the pool as bf16 pages [n_out][2][hkv][16][hd]; slots from n_tokens on are zeros.  One thread, sixteen codes.
template <int HD, int FMT>
__global__ void __launch_bounds__(256) kv8_read_kernel(const uint8_t* __restrict__ pool, int n_pages, int hkv, const int* __restrict__ pages,
                                                       int n_out, long n_tokens, bf16* __restrict__ out, int* __restrict__ status) {
  constexpr int CPR = HD / 16, CPB = 2 * kKv8Page * CPR;      // 16-code chunks of a row and of a block
  pdl_wait();
  pdl_launch_dependents();
  const long id = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const long b = id / CPB;
  const int c = (int)(id % CPB);
  if (b >= (long)n_out * hkv) return;
  const int pi = (int)(b / hkv), h = (int)(b % hkv);
  const int kv = c / (CPB / 2), row = (c / CPR) % kKv8Page, cc = c % CPR;
  const int page = pages[pi];
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = 0.f;
  if ((long)pi * kKv8Page + row < n_tokens) {
    if (page < 0 || page >= n_pages) {
      if (c == 0) atomicExch(status, (int)B2_ERR_BOUNDS);
    } else {
      const uint8_t* blk = pool + ((size_t)page * hkv + h) * kv8_block_bytes(HD);
      const uint4 w = *reinterpret_cast<const uint4*>(blk + (size_t)c * 16);
      const float s = reinterpret_cast<const float*>(blk + 2 * kKv8Page * HD)[row * 2 + kv];
      const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = kv8_value<FMT>((wd[i >> 2] >> (8 * (i & 3))) & 0xffu) * s;
    }
  }
  __align__(16) __nv_bfloat162 o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  uint4* dst = reinterpret_cast<uint4*>(out + (((size_t)pi * 2 + kv) * hkv + h) * kKv8Page * HD + (size_t)row * HD + cc * 16);
  dst[0] = reinterpret_cast<const uint4*>(o)[0];
  dst[1] = reinterpret_cast<const uint4*>(o)[1];
}

template <class K, class... A>
int launch(K kernel, long blocks, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks); cfg.blockDim = dim3(threads); cfg.stream = st;
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
  if ((hd != 64 && hd != 128) || (fmt != KV8_INT8 && fmt != KV8_FP8) || a.ld % 4 || a.ldq % 4) return B2_ERR_ARG;
  const int hpw = 32 / (hd / 8), turns = (a.hq + 2 * a.hkv + hpw - 1) / hpw;
  const int wpt = std::min(turns, 8);
  const long blocks = ((long)a.n * wpt + 7) / 8;
  if (blocks > 0x7fffffffl) return B2_ERR_ARG;
  auto k = hd == 128 ? (fmt == KV8_INT8 ? kv8_store_kernel<128, KV8_INT8> : kv8_store_kernel<128, KV8_FP8>)
                     : (fmt == KV8_INT8 ? kv8_store_kernel<64, KV8_INT8> : kv8_store_kernel<64, KV8_FP8>);
  return launch(k, blocks, 256, st, a, wpt);
}

B2_API int b2_kv8_read(const uint8_t* pool, int n_pages, int hkv, int hd, int fmt, const int* pages, int n_out, long n_tokens,
                       bf16* out, int* status, cudaStream_t st) {
  if (n_out < 1 || hkv < 1 || n_pages < 1 || n_tokens < 0) return B2_ERR_ARG;
  if ((hd != 64 && hd != 128) || (fmt != KV8_INT8 && fmt != KV8_FP8)) return B2_ERR_ARG;
  const long blocks = ((long)n_out * hkv * 2 * hd + 255) / 256;
  if (blocks > 0x7fffffffl) return B2_ERR_ARG;
  auto k = hd == 128 ? (fmt == KV8_INT8 ? kv8_read_kernel<128, KV8_INT8> : kv8_read_kernel<128, KV8_FP8>)
                     : (fmt == KV8_INT8 ? kv8_read_kernel<64, KV8_INT8> : kv8_read_kernel<64, KV8_FP8>);
  return launch(k, blocks, 256, st, pool, n_pages, hkv, pages, n_out, n_tokens, out, status);
}
