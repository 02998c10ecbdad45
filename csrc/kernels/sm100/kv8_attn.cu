// Attention of new tokens over 8-bit key-value pages (format: kv8.cuh): decode steps, verify blocks (causal or tree mask)
// and short prefill chunks.  Counterpart in the reference: the INT8 KV of its dense layers, which expands tiles to bf16 and
// attends to those (kernels/m1/m1_dense8.cu:65-126); here the codes go straight into the products.
//
//     o = sum_j p_j vs_j vc_j / sum_j p_j,    p_j = 2^(s_j - m),    s_j = log2(e) / sqrt(hd) * ks_j * (q . kc_j)
//
// over the keys j that the row sees.  One pass with a running reference m.  The int8 codes kc go into an integer product with q in
// sixteen bits; e4m3's, and all vc, become fp16 numbers (exactly: both formats fit).  The scales stay in fp32: ks multiplies the
// finished product, vs the weight before it is rounded.
//
// Split.  A sequence's keys are cut every split_keys keys, a constant of the engine; one CTA of four warps takes the keys of one
// (group, KV head, columns, split), page i of them on warp i % 4, and joins its warps in shared memory.  Rows with one split are
// finished there, the others leave (o, m, l) per split to kv8_join_kernel.  What a row adds up and in which order depends on its
// own position alone, so a row has the same bits in a decode step, a verify block or any batch.
//
// Products.  The group's rows times the q heads of a KV head are the columns ("N" of the MMA, eight to a tile), keys are the rows
// of K q^T and head channels the rows of V^T p^T, so a single decode row with eight q heads fills its tiles.  The order of
// channels inside a product and of keys inside a page is free, and chosen so that every lane loads sixteen bytes of a row at a
// time straight from global memory into its fragments; shared memory is not used on the way.  Only the weights need a
// transposition between the products (movmatrix).
//
// Range.  The weights reach the second product as fp16 numbers p_j vs_j.  m follows the largest s_j + log2 of vs_j's power of two,
// so what is rounded is each key's contribution relative to the largest one, whatever the size of V; a key that has weight but no
// V (a row of zeros has the least scale) cannot push the others out of fp16's range.  m is raised only when a column's largest
// value has grown by 2^8 (fp16 has room for that), which leaves the accumulators alone for nearly all pages.
#include <algorithm>
#include <type_traits>

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
  int split_keys, max_splits;
  float* part_o;                            // [n_tok][hq][max_splits][hd]; unused when max_splits is 1
  float* part_ml;                           // [n_tok][hq][max_splits][2]
};

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 2;                  // pairs of pages that a warp has in shared memory or under way
constexpr float kNoRef = -3.4028234e38f;    // m before the first key
constexpr float kGrow = 8.f;                // log2 of what a column may grow before m follows
// l sums 2^(s - m) * 2^30 and the weights carry vs * 2^-30: with V of any size between 2^-64 and 2^121 neither leaves fp32
constexpr float kUp = 30.f, kDown = 9.313225746154785e-10f;

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// four e4m3 numbers -> fp16 pairs (0, 1) and (2, 3)
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t& x, uint32_t& y) {
  asm("{ .reg .b16 lo, hi; mov.b32 {lo, hi}, %2; cvt.rn.f16x2.e4m3x2 %0, lo; cvt.rn.f16x2.e4m3x2 %1, hi; }" : "=r"(x), "=r"(y) : "r"(w));
}
// D(16x8, s32) += A(16x32, u8, row) * B(32x8, s8 or u8, col)
template <bool SIGNED>
__device__ __forceinline__ void mma_u8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (SIGNED)
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Of two rows' words: pairs (row a, row b) of bytes 2 * HI and 2 * HI + 1
template <int FMT, int HI>
__device__ __forceinline__ void cross_pairs(uint32_t wa, uint32_t wb, uint32_t& x, uint32_t& y) {
  if (FMT == KV8_INT8) {
    const uint32_t z = __byte_perm(wa, wb, HI ? 0x7632 : 0x5410);
    x = lop3_and_or(z, 0x00ff00ffu, 0x64006400u);          // 0x64xx is 1024 + xx, 1152 above the code
    y = __byte_perm(z, 0x64646464u, 0x4341);
  } else {
    e4m3_pairs(__byte_perm(wa, wb, HI ? 0x7362 : 0x5140), x, y);
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

struct Group { int tok0, cnt, first, last, seq; bool ok; };

// A group and whether everything it names is there; `last` is the last slot that its rows may see.
__device__ __forceinline__ Group group_at(const Kv8AttnArgs& a, int g) {
  Group r = {0, 0, 0, -1, 0, true};
  if (g >= a.n_groups) return r;
  r.tok0 = a.grp_tok0[g]; r.cnt = a.grp_cnt[g];
  if (r.cnt < 1) { r.cnt = 0; return r; }
  r.ok = r.cnt <= 32 && r.tok0 >= 0 && r.tok0 <= a.n_tok - r.cnt;
  if (!r.ok) return r;
  r.seq = a.tok_seq[r.tok0]; r.first = a.tok_pos[r.tok0];
  r.last = r.cnt == 1 ? r.first : a.tok_pos[r.tok0 + r.cnt - 1];
  r.ok = r.seq >= 0 && r.seq < a.n_seq && r.last < a.bt_cols * kKv8Page && r.last / a.split_keys < a.max_splits;
  return r;
}
__device__ __forceinline__ int splits_of(int last_key, int split_keys) { return last_key < 0 ? 1 : last_key / split_keys + 1; }

// Copies of blocks into the ring and where a lane finds its bytes there.  A block is looked at as 128-byte lines (one row of 128
// channels, two of 64); the 16-byte pieces of a line are permuted so that the eight lanes of a load's phase hit different banks:
// for K these are two rows times four neighbouring pieces, for V four rows times two.
template <int HD>
struct Ring {
  static constexpr int kSlab = kKv8Page * HD;
  uint32_t src, dst_k, dst_v[kSlab / 512];           // a lane's copies: 512 bytes a turn
  uint32_t rd_k, rd_v;
  __device__ __forceinline__ Ring(int lane) {
    const int g = lane >> 2, t = lane & 3, l4 = lane >> 3, c = lane & 7;
    src = lane * 16;
    // lines 4k + l4: K by the line's parity in units of two rows, V by fours of rows
    dst_k = l4 * 128 + ((c ^ ((HD == 128 ? l4 >> 1 : l4) & 1) * 4) << 4);
#pragma unroll
    for (int k = 0; k < kSlab / 512; ++k) dst_v[k] = kSlab + (4 * k + l4) * 128 + ((c ^ ((HD == 128 ? k : 2 * k + (l4 >> 1)) * 2)) << 4);
    rd_k = HD == 128 ? 2 * g * 128 + ((t ^ (g & 1) * 4) << 4) : g * 128 + ((t ^ (g & 1) * 4) << 4);
    rd_v = kSlab + (HD == 128 ? 4 * t * 128 + ((g ^ t * 2) << 4) : 2 * t * 128 + (((g >> 1) ^ t * 2) << 4) + (g & 1) * 8);
  }
  __device__ __forceinline__ void copy(uint32_t stage, const uint8_t* blk, int lane) const {
#pragma unroll
    for (int k = 0; k < kSlab / 512; ++k) {
      cp_async16(stage + dst_k + k * 512, blk + src + k * 512);
      cp_async16(stage + dst_v[k], blk + kSlab + src + k * 512);
    }
    if (lane < 8) cp_async16(stage + 2 * kSlab + src, blk + 2 * kSlab + src);
  }
  __device__ __forceinline__ uint4 k(uint32_t stage, int r, int c) const {      // row 2g + r, piece t + 4c
    if (HD == 128) return lds128(stage + ((rd_k + r * 128) ^ (c * 64)));
    return lds128(stage + (rd_k ^ (r * 64)));
  }
  __device__ __forceinline__ void v(uint32_t stage, int r, uint32_t (&w)[HD / 32]) const {     // row 4t + r, channels g * HD / 8 and on
    if constexpr (HD == 128) {
      const uint4 u = lds128(stage + rd_v + r * 128);
      w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
      const uint2 u = lds64(stage + ((rd_v + (r >> 1) * 128) ^ ((r & 1) * 64)));
      w[0] = u.x; w[1] = u.y;
    }
  }
};

// One CTA's share of a group: keys of one split for eight or sixteen columns.
struct Item {
  int tok0, cnt, first, last, col0, kvh, split;
  int n_my, page;                        // pages of this warp; lane i holds the number of page i
};

template <int HD>
constexpr int attn_smem() { return kWarps * kStages * 2 * kv8_block_bytes(HD); }

template <int HD, int FMT, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) kv8_attn_kernel(const Kv8AttnArgs a) {
  constexpr int KC = HD / 64;            // 16-byte pieces of a K row per lane
  constexpr int KW = HD / 16;            // words of a K row per lane
  constexpr int VW = HD / 32;            // words of a V row per lane
  constexpr int MT = HD / 16;            // channel tiles of V^T p^T
  constexpr int COLS = NT * 8;
  constexpr int LDO = HD + 4;
  constexpr int BLK = kv8_block_bytes(HD);
  constexpr int PAIR = 2 * BLK;
  // a warp's results of an item go over the pair of pages that it used last, which is not refilled before they have been read
  static_assert(COLS * LDO * 4 <= PAIR, "a tile of results fits a pair of pages");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sh_m[kWarps][COLS], sh_l[kWarps][COLS];
  __shared__ int sh_at[kWarps];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int gq = a.hq / a.hkv;
  const Ring<HD> ring(lane);
  const uint32_t mem = smem_u32(smem) + warp * kStages * PAIR;

  // Items are numbered group after group and cut evenly over the CTAs; neighbours differ in the split first, so a CTA keeps its
  // q for most of them.  Every lane holds one group of a run of 32 and the number of items up to it.
  int run = -1, base = 0, total = 0, incl = 0, mine = 0;
  Group grp = {0, 0, 0, -1, 0, true};
  auto load_run = [&](int r) {
    run = r;
    grp = group_at(a, r * 32 + lane);
    mine = grp.ok && grp.cnt > 0 ? splits_of(grp.last, a.split_keys) * a.hkv * ((grp.cnt * gq + COLS - 1) / COLS) : 0;
    incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += v; }
    total = __shfl_sync(0xffffffffu, incl, 31);
  };
  int all = 0;
  for (int r = 0; r * 32 < a.n_groups; ++r) {
    load_run(r);
    if (!grp.ok && blockIdx.x == 0 && warp == 0) atomicExch(a.status, (int)B2_ERR_BOUNDS);
    all += total;
  }
  const int share = all / (int)gridDim.x, rest = all % (int)gridDim.x, id = blockIdx.x;
  int item = id * share + min(id, rest);
  const int item_end = item + share + (id < rest ? 1 : 0);
  if (item >= item_end) return;
  if (run != 0) load_run(0);
  auto fetch = [&](int at, Item& it) {
    while (at - base >= total) { base += total; load_run(run + 1); }
    at -= base;
    const int src = __ffs(__ballot_sync(0xffffffffu, incl > at)) - 1;
    at -= __shfl_sync(0xffffffffu, incl, src) - __shfl_sync(0xffffffffu, mine, src);
    it.tok0 = __shfl_sync(0xffffffffu, grp.tok0, src); it.cnt = __shfl_sync(0xffffffffu, grp.cnt, src);
    it.first = __shfl_sync(0xffffffffu, grp.first, src); it.last = __shfl_sync(0xffffffffu, grp.last, src);
    const int seq = __shfl_sync(0xffffffffu, grp.seq, src), ns = splits_of(it.last, a.split_keys);
    const int ctiles = (it.cnt * gq + COLS - 1) / COLS;
    it.split = at % ns; at /= ns;
    it.col0 = at % ctiles * COLS; it.kvh = at / ctiles;
    const int k_begin = it.split * a.split_keys, k_end = min(it.last + 1, k_begin + a.split_keys);
    const int n_pg = (k_end - k_begin + kKv8Page - 1) / kKv8Page;           // 0 for a group without keys
    it.n_my = (n_pg - warp + kWarps - 1) / kWarps;                          // at most 32: split_keys is at most 2048
    it.page = -1;
    if (lane < it.n_my) it.page = a.block_table[(size_t)seq * a.bt_ld + k_begin / kKv8Page + warp + kWarps * lane];
    __syncwarp();
  };
  Item cur, nxt;
  fetch(item, nxt);
  cur = nxt;
  cur.tok0 = -1;                         // no q yet
  int wr = 0, rd = 0, pending = 0;       // stages to fill and to read next; pairs sent for and not yet used
  // where this warp fetches (nxt once it is ahead of cur): pages left to send for and which come next
  int f_i = 0, f_n = 0, f_page = 0, f_kvh = 0;
  bool ahead = false, more = true;

  // q, every column scaled by a power of two; qs undoes it on the scores and brings the softmax scale.
  // int8: sixteen bits of fixed point, the largest value in [2^14, 2^15), as a signed and an unsigned byte (hi * 256 + lo): K's bytes
  // then feed the product as they are, and the sums are exact.  What is lost is at most 2^-15 of the column's largest value, as much as
  // a weight in fp16 loses.  The 128 in K's bytes comes off again with the accumulators' start, -128 * sum(q).
  // e4m3: fp16 with the largest value in [2^10, 2^11), where a bf16 number stays exact down to 2^-24 of that.
  uint32_t qb[NT][KW][2];
  float qs[NT][2];
  int q0[NT][2];

  for (; item < item_end; ++item) {
    const bool same_q = nxt.tok0 == cur.tok0 && nxt.cnt == cur.cnt && nxt.col0 == cur.col0 && nxt.kvh == cur.kvh;
    cur = nxt;
    if (!ahead) { f_i = 0; f_n = cur.n_my; f_page = cur.page; f_kvh = cur.kvh; }
    ahead = false;
    more = item + 1 < item_end;
    if (more) fetch(item + 1, nxt);
    const int tok0 = cur.tok0, cnt = cur.cnt, first = cur.first, last = cur.last, col0 = cur.col0, kvh = cur.kvh, split = cur.split, n_my = cur.n_my;
    const int k_begin = split * a.split_keys, k_end = min(last + 1, k_begin + a.split_keys);
    const unsigned valid = __ballot_sync(0xffffffffu, lane < n_my && (unsigned)cur.page < (unsigned)a.n_pages);
    auto top_up = [&]() {
      while (pending < kStages) {
        if (f_i >= f_n) {
          if (ahead || !more) return;
          ahead = true;
          f_i = 0; f_n = nxt.n_my; f_page = nxt.page; f_kvh = nxt.kvh;
          continue;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && f_i + 1 >= f_n) break;
          int p = __shfl_sync(0xffffffffu, f_page, f_i + h);
          if ((unsigned)p >= (unsigned)a.n_pages) {       // its keys are masked below; something there is copied in their place
            if (lane == 0) atomicExch(a.status, (int)B2_ERR_BOUNDS);
            p = 0;
          }
          ring.copy(mem + wr + h * BLK, a.pool + ((size_t)p * a.hkv + f_kvh) * BLK, lane);
        }
        cp_async_commit();
        wr ^= PAIR;
        ++pending;
        f_i += 2;
      }
    };
    top_up();

    if (!same_q) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int col = col0 + n * 8 + g;
        const bool live = col < cnt * gq;
        uint4 raw[KC][2];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            raw[c][h] = make_uint4(0u, 0u, 0u, 0u);
            if (live) raw[c][h] = *reinterpret_cast<const uint4*>(a.q + (size_t)(tok0 + col / gq) * a.ldq + (size_t)(kvh * gq + col % gq) * HD + (t + 4 * c) * 16 + h * 8);
            const uint32_t* w = &raw[c][h].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, max((w[i] & 0x7fffu) << 16, w[i] & 0x7fff0000u));
          }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = min((FMT == KV8_INT8 ? 268u : 264u) - (top >> 23), 253u);
        const float up = __uint_as_float(e << 23);
        float down = __uint_as_float((254u - e) << 23) * a.scale_log2;
        if (top >= 0x7f800000u) down = __uint_as_float(0x7fffffffu);           // an infinity or a NaN in q: a column of NaN
        int sum = 0;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int w = 0; w < 4; ++w) {                // four channels of a K word
            const uint32_t a0 = (&raw[c][w >> 1].x)[2 * (w & 1)], a1 = (&raw[c][w >> 1].x)[2 * (w & 1) + 1];
            const float f0 = __uint_as_float(a0 << 16) * up, f1 = __uint_as_float(a0 & 0xffff0000u) * up;
            const float f2 = __uint_as_float(a1 << 16) * up, f3 = __uint_as_float(a1 & 0xffff0000u) * up;
            if constexpr (FMT == KV8_INT8) {
              const int i0 = __float2int_rn(f0), i1 = __float2int_rn(f1), i2 = __float2int_rn(f2), i3 = __float2int_rn(f3);
              sum += i0 + i1 + i2 + i3;
              const uint32_t p01 = __byte_perm(i0, i1, 0x5140), p23 = __byte_perm(i2, i3, 0x5140);      // lo, lo, hi, hi
              qb[n][c * 4 + w][0] = __byte_perm(p01, p23, 0x7632);
              qb[n][c * 4 + w][1] = __byte_perm(p01, p23, 0x5410);
            } else {
              qb[n][c * 4 + w][0] = pack_half(f0, f1);
              qb[n][c * 4 + w][1] = pack_half(f2, f3);
            }
          }
        qs[n][0] = __shfl_sync(0xffffffffu, down, 8 * t);
        qs[n][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
        if constexpr (FMT == KV8_INT8) {
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          q0[n][0] = -128 * __shfl_sync(0xffffffffu, sum, 8 * t);
          q0[n][1] = -128 * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
        }
      }
    }

    // m is the reference less kUp, so that 2^(s - m) carries the 2^30
    float o[NT][MT][4], m[NT][2], l[NT][2];
    // int8: V's fp16 numbers are 1152 above the codes; the same sums of 1152 alone are taken off at the end.  Both lose alike to
    // the accumulators' truncation, 2^-23 of 1152 a step, so that what is left of it is a random part below 2^-10 of a code.
    float bias[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = kNoRef; l[n][0] = l[n][1] = 0.f;
      bias[n][0] = bias[n][1] = bias[n][2] = bias[n][3] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    for (int i = 0; i < n_my; i += 2) {
      // this pair has arrived once no more copies are under way than were sent for after it
      if (pending >= 2) cp_async_wait<1>(); else cp_async_wait<0>();
      __syncwarp();
      const uint32_t stage = mem + rd;
      // s[h]: page i + h, keys 2g (0, 1) and 2g + 1 (2, 3), columns 2t (0, 2) and 2t + 1 (1, 3)
      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (FMT == KV8_INT8) {
          int hi[NT][4], lo[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) { hi[n][j] = 0; lo[n][j] = q0[n][j & 1]; }
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint4 k0 = ring.k(stage + h * BLK, 0, c), k1 = ring.k(stage + h * BLK, 1, c);
#pragma unroll
            for (int w = 0; w < 4; w += 2) {
              const uint32_t f[4] = {(&k0.x)[w], (&k1.x)[w], (&k0.x)[w + 1], (&k1.x)[w + 1]};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma_u8<true>(hi[n], f, qb[n][c * 4 + w][0], qb[n][c * 4 + w + 1][0]);
                mma_u8<false>(lo[n], f, qb[n][c * 4 + w][1], qb[n][c * 4 + w + 1][1]);
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[h][n][j] = __int2float_rn(hi[n][j] * 256 + lo[n][j]);
        } else {
#pragma unroll
          for (int n = 0; n < NT; ++n) s[h][n][0] = s[h][n][1] = s[h][n][2] = s[h][n][3] = 0.f;
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint4 k0 = ring.k(stage + h * BLK, 0, c), k1 = ring.k(stage + h * BLK, 1, c);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t f[4];
              e4m3_pairs((&k0.x)[w], f[0], f[2]);
              e4m3_pairs((&k1.x)[w], f[1], f[3]);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_f16_16816(s[h][n], f, qb[n][c * 4 + w][0], qb[n][c * 4 + w][1]);
            }
          }
        }
      }
      float e[2][2], vs[2][2];                      // of keys 2g, 2g + 1: log2 of V scale's power of two; V scale 2^-30
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 su = lds128(stage + h * BLK + 2 * kKv8Page * HD + g * 16);        // (K, V) scales of keys 2g, 2g + 1
        e[h][0] = __uint_as_float(0x4b000000u | (su.y >> 23)) - 8388735.f;
        e[h][1] = __uint_as_float(0x4b000000u | (su.w >> 23)) - 8388735.f;
        vs[h][0] = __fmul_rn(__uint_as_float(su.y), kDown);
        vs[h][1] = __fmul_rn(__uint_as_float(su.w), kDown);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[h][n][j] = __fmul_rn(__fmul_rn(s[h][n][j], __uint_as_float(j < 2 ? su.x : su.z)), qs[n][j & 1]);
      }
      const int kb = k_begin + (warp + kWarps * i) * kKv8Page;              // the pair's second page begins 64 keys later
      const unsigned have = valid >> i & 3u;
      // from the group's first slot on, at the split's end and where a page is missing, keys are looked at one by one
      const bool partly = kb + (kWarps + 1) * kKv8Page > min(first, k_end) || have != 3u;
      if (partly) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int col = col0 + n * 8 + 2 * t + j, row = min(col / gq, cnt - 1);
            const int pos = cnt == 1 ? last : min(a.tok_pos[tok0 + row], last);
            const unsigned mask = a.tree_mask ? a.tree_mask[tok0 + row] : 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const int key = kb + h * kWarps * kKv8Page + 2 * g + r, in = key - first;
                const bool seen = key <= pos && key < k_end && (have >> h & 1u) && (!a.tree_mask || in < 0 || (in < 32 && ((mask >> (in & 31)) & 1u)));
                if (!seen) s[h][n][2 * r + j] = -INFINITY;
              }
          }
      }
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float top = fmaxf(fmaxf(__fadd_rn(s[0][n][j], e[0][0]), __fadd_rn(s[0][n][2 + j], e[0][1])),
                                  fmaxf(__fadd_rn(s[1][n][j], e[1][0]), __fadd_rn(s[1][n][2 + j], e[1][1])));
          grows |= top > __fadd_rn(m[n][j], kUp + kGrow);
        }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = fmaxf(fmaxf(__fadd_rn(s[0][n][j], e[0][0]), __fadd_rn(s[0][n][2 + j], e[0][1])),
                             fmaxf(__fadd_rn(s[1][n][j], e[1][0]), __fadd_rn(s[1][n][2 + j], e[1][1])));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            if (mx > __fadd_rn(m[n][j], kUp + kGrow)) {
              const float f = ex2(__fadd_rn(m[n][j], kUp - mx));
              m[n][j] = __fadd_rn(mx, -kUp);
              l[n][j] = __fmul_rn(l[n][j], f);
              bias[n][j] = __fmul_rn(bias[n][j], f);
              bias[n][2 + j] = bias[n][j];
#pragma unroll
              for (int k = 0; k < MT; ++k) { o[n][k][j] = __fmul_rn(o[n][k][j], f); o[n][k][2 + j] = __fmul_rn(o[n][k][2 + j], f); }
            }
          }
        __syncwarp();
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = ex2(__fadd_rn(s[h][n][j], -m[n][j & 1]));
            l[n][j & 1] = __fadd_rn(l[n][j & 1], p);
            w[j] = __fmul_rn(p, vs[h][j >> 1]);
          }
          if (partly)                               // a row that is not seen may have the scale NaN
#pragma unroll
            for (int j = 0; j < 4; ++j) if (s[h][n][j] == -INFINITY) w[j] = 0.f;
          pb[h][n][0] = transpose8x8(pack_half(w[0], w[1]));
          pb[h][n][1] = transpose8x8(pack_half(w[2], w[3]));
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t vw[4][VW];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ring.v(stage + h * BLK, r, vw[r]);
          // bytes past the end may be e4m3's NaN, which a weight of zero does not silence
          if (FMT == KV8_FP8 && partly && (kb + h * kWarps * kKv8Page + 4 * t + r >= k_end || !(have >> h & 1u)))
#pragma unroll
            for (int w = 0; w < VW; ++w) vw[r][w] = 0u;
        }
        if (h == 1) {
          __syncwarp();                             // the pair has been read
          rd ^= PAIR;
          --pending;
          if (i + 2 < n_my) top_up();               // the last pair's place holds the results first
        }
        if constexpr (FMT == KV8_INT8) {
          const uint32_t f[4] = {0x64806480u, 0x64806480u, 0x64806480u, 0x64806480u};         // 1152
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(bias[n], f, pb[h][n][0], pb[h][n][1]);
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t f[4];
          cross_pairs<FMT, 0>(vw[0][w], vw[2][w], f[0], f[1]);
          cross_pairs<FMT, 0>(vw[1][w], vw[3][w], f[2], f[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][2 * w], f, pb[h][n][0], pb[h][n][1]);
          cross_pairs<FMT, 1>(vw[0][w], vw[2][w], f[0], f[1]);
          cross_pairs<FMT, 1>(vw[1][w], vw[3][w], f[2], f[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][2 * w + 1], f, pb[h][n][0], pb[h][n][1]);
        }
      }
    }

    const int at = warp * kStages * PAIR + (rd ^ PAIR);
    if (lane == 0) sh_at[warp] = n_my > 0 ? at : -1;
    if (n_my > 0) {
      float (*tile)[LDO] = reinterpret_cast<float (*)[LDO]>(smem + at);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float x = l[n][j];
          x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const int c = n * 8 + 2 * t + j;
          if (g == 0) { sh_m[warp][c] = m[n][j]; sh_l[warp][c] = __fmul_rn(x, kDown); }
          const float b = FMT == KV8_INT8 ? -bias[n][j] : 0.f;
#pragma unroll
          for (int k = 0; k < MT; k += 2)
            *reinterpret_cast<float4*>(&tile[c][g * (HD / 8) + 2 * k]) = make_float4(__fadd_rn(o[n][k][j], b), __fadd_rn(o[n][k][2 + j], b),
                                                                                     __fadd_rn(o[n][k + 1][j], b), __fadd_rn(o[n][k + 1][2 + j], b));
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < COLS * (HD / 4); i += kWarps * 32) {
      const int c = i / (HD / 4), d = i % (HD / 4) * 4, col = col0 + c;
      if (col >= cnt * gq) continue;
      const int tok = tok0 + col / gq, head = kvh * gq + col % gq;
      const int ns = splits_of(cnt == 1 ? last : min(a.tok_pos[tok], last), a.split_keys);
      if (split >= ns) continue;
      float M = kNoRef;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) if (sh_at[w] >= 0) M = fmaxf(M, sh_m[w][c]);
      float L = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (sh_at[w] < 0) continue;
        const float f = ex2(__fadd_rn(sh_m[w][c], -M));
        const float4 y = *reinterpret_cast<const float4*>(smem + sh_at[w] + (c * LDO + d) * 4);
        L = __fmaf_rn(sh_l[w][c], f, L);
        x.x = __fmaf_rn(y.x, f, x.x); x.y = __fmaf_rn(y.y, f, x.y); x.z = __fmaf_rn(y.z, f, x.z); x.w = __fmaf_rn(y.w, f, x.w);
      }
      if (ns == 1) {
        const float inv = L == 0.f ? 0.f : __fdiv_rn(1.f, L);
        uint2 v;
        *reinterpret_cast<__nv_bfloat162*>(&v.x) = __floats2bfloat162_rn(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv));
        *reinterpret_cast<__nv_bfloat162*>(&v.y) = __floats2bfloat162_rn(__fmul_rn(x.z, inv), __fmul_rn(x.w, inv));
        *reinterpret_cast<uint2*>(a.out + (size_t)tok * a.ldo + (size_t)head * HD + d) = v;
      } else {
        const size_t slot = ((size_t)tok * a.hq + head) * a.max_splits + split;
        *reinterpret_cast<float4*>(a.part_o + slot * HD + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(M, L);
      }
    }
    __syncthreads();                                // results have been read: their places take pages again
  }
}

// Joins the splits of rows that have more than one: a CTA per (group, row, q head).  Sixteen sums, sum j of the splits j, j + 16, ...
// in order, are added in order of j.  WARPS warps take 16 / WARPS sums each, side by side; both variants give the same bits.
template <int HD, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) kv8_join_kernel(const Kv8AttnArgs a, int rows_at_once) {
  constexpr int PER = HD / 32, SETS = 16, MY = SETS / WARPS, AHEAD = 8 / MY;
  using Vec = std::conditional_t<PER == 4, float4, float2>;
  __shared__ float sh[SETS][HD + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int head = blockIdx.x % a.hq, r0 = blockIdx.x / a.hq % rows_at_once;
  const Group grp = group_at(a, blockIdx.x / a.hq / rows_at_once);
  if (!grp.ok) return;
  for (int r = r0; r < grp.cnt; r += rows_at_once) {
    const int tok = grp.tok0 + r;
    const int ns = splits_of(grp.cnt == 1 ? grp.last : min(a.tok_pos[tok], grp.last), a.split_keys);
    if (ns == 1) continue;
    const size_t slot = ((size_t)tok * a.hq + head) * a.max_splits;
    const Vec* po = reinterpret_cast<const Vec*>(a.part_o + slot * HD) + lane;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + slot;
    float M = kNoRef;
    for (int s = lane; s < ns; s += 32) M = fmaxf(M, ml[s].x);
    M = warp_max(M);
    float L[MY], x[MY][PER];
#pragma unroll
    for (int k = 0; k < MY; ++k) {
      L[k] = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) x[k][i] = 0.f;
    }
    for (int s0 = warp * MY; s0 < ns; s0 += AHEAD * SETS) {
      float2 w[AHEAD][MY];
      Vec y[AHEAD][MY];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
#pragma unroll
        for (int k = 0; k < MY; ++k) {                 // past the end: the last split again, with the weight zero
          const int s = min(s0 + j * SETS + k, ns - 1);
          w[j][k] = ml[s];
          y[j][k] = po[(size_t)s * 32];
        }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
#pragma unroll
        for (int k = 0; k < MY; ++k) {
          const float f = s0 + j * SETS + k < ns ? ex2(__fadd_rn(w[j][k].x, -M)) : 0.f;
          L[k] = __fmaf_rn(w[j][k].y, f, L[k]);
#pragma unroll
          for (int i = 0; i < PER; ++i) x[k][i] = __fmaf_rn((&y[j][k].x)[i], f, x[k][i]);
        }
    }
#pragma unroll
    for (int k = 0; k < MY; ++k) {
#pragma unroll
      for (int i = 0; i < PER; ++i) sh[warp * MY + k][lane * PER + i] = x[k][i];
      if (lane == 0) sh[warp * MY + k][HD] = L[k];
    }
    __syncthreads();
    for (int d = threadIdx.x; d < HD; d += WARPS * 32) {
      float sum = sh[0][d], Ls = sh[0][HD];
#pragma unroll
      for (int w = 1; w < SETS; ++w) { sum = __fadd_rn(sum, sh[w][d]); Ls = __fadd_rn(Ls, sh[w][HD]); }
      a.out[(size_t)tok * a.ldo + (size_t)head * HD + d] = __float2bfloat16_rn(Ls == 0.f ? 0.f : __fmul_rn(sum, __fdiv_rn(1.f, Ls)));
    }
    __syncthreads();
  }
}

template <class K, class... A>
cudaError_t launch(K kernel, unsigned blocks, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int HD, int FMT>
int run(const Kv8AttnArgs& a, cudaStream_t st) {
  const long rows = ((long)a.n_tok + a.n_groups - 1) / a.n_groups;           // of a group, on average
  const int gq = a.hq / a.hkv;
  // columns of one item: eight where a group fills no more (a decode step of up to eight q heads per KV head), else sixteen,
  // which halves the loads and conversions of K and V
  const bool wide = rows * gq > 8;
  const long items = (long)a.n_groups * a.hkv * a.max_splits * ((rows * gq + (wide ? 15 : 7)) / (wide ? 16 : 8));
  const unsigned grid = (unsigned)std::min<long>(items, 148 * (wide ? 2 : 3));
  auto kernel = wide ? kv8_attn_kernel<HD, FMT, 2> : kv8_attn_kernel<HD, FMT, 1>;
  constexpr int smem = attn_smem<HD>();
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);     // of the current device
  if (e == cudaSuccess) e = launch(kernel, grid, kWarps * 32, smem, st, a);
  if (e == cudaSuccess && a.max_splits > 1) {
    // few rows with many splits: sixteen warps a CTA keep enough loads under way
    const unsigned blocks = (unsigned)(a.n_groups * rows * a.hq);
    e = a.max_splits > 16 && blocks <= 148 * 4 ? launch(kv8_join_kernel<HD, 16>, blocks, 512, 0, st, a, (int)rows)
                                               : launch(kv8_join_kernel<HD, 4>, blocks, 128, 0, st, a, (int)rows);
  }
  return e == cudaSuccess ? B2_OK : B2_ERR_LAUNCH;
}

}  // namespace
}  // namespace b2

using namespace b2;

B2_API int b2_kv8_attn(const Kv8AttnArgs* args, int hd, int fmt, cudaStream_t st) {
  const Kv8AttnArgs& a = *args;
  if (a.n_groups < 1 || a.n_tok < 1 || a.hkv < 1 || a.hq < 1 || a.hq % a.hkv || a.n_seq < 1 || a.bt_cols < 1 || a.n_pages < 1) return B2_ERR_ARG;
  if ((hd != 64 && hd != 128) || (fmt != KV8_INT8 && fmt != KV8_FP8) || a.ldq % 8 || a.ldo % 8) return B2_ERR_ARG;
  if (a.split_keys < kKv8Page || a.split_keys > 2048 || a.split_keys % kKv8Page || a.max_splits < 1) return B2_ERR_ARG;
  if (a.max_splits > 1 && (!a.part_o || !a.part_ml)) return B2_ERR_ARG;
  // item and block numbers are 32-bit
  if (a.bt_cols > (1 << 26) || (long)a.n_groups * a.hq * 32 * a.max_splits > 0x7fff0000l || ((long)a.n_tok + a.n_groups) * a.hq > 0x7fffffffl) return B2_ERR_ARG;
  if (hd == 128) return fmt == KV8_INT8 ? run<128, KV8_INT8>(a, st) : run<128, KV8_FP8>(a, st);
  return fmt == KV8_INT8 ? run<64, KV8_INT8>(a, st) : run<64, KV8_FP8>(a, st);
}
