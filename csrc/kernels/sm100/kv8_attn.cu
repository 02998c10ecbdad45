// Attention of new tokens over 8-bit key-value pages (format: kv8.cuh): decode steps, verify blocks (causal or tree mask)
// and short prefill chunks.  Counterpart in the reference: the INT8 KV of its dense layers, which expands tiles to bf16 and
// attends to those (kernels/m1/m1_dense8.cu:65-126); here the codes become operands in registers.
//
//     o = sum_j p_j vs_j vc_j / sum_j p_j,    p_j = 2^(s_j - m),    s_j = log2(e) / sqrt(hd) * ks_j * (q . kc_j)
//
// over the keys j that the row sees.  One pass with a running reference m.  The codes kc and vc become fp16 numbers (exactly: both
// formats fit), q's too, times a power of two of its column.  The scales stay in fp32: ks multiplies the finished product, vs the
// weight before it is rounded.
//
// Split.  A sequence's keys are cut every split_keys keys, a constant of the engine; one CTA of four warps takes the keys of one
// (group, KV head, columns, split), page i of them on warp i % 4, and joins its warps in shared memory.  Rows with one split are
// finished there, the others leave (o, m, l) per split to kv8_join_kernel.  What a row adds up and in which order depends on its
// own position alone, so a row has the same bits in a decode step, a verify block or any batch.
//
// Products.  The group's rows times the q heads of a KV head are the columns, eight to a tile, so that a single decode row with eight
// q heads wastes nothing.  S = q K^T takes q as A (its rows are the columns, eight of sixteen where there are no more) and K's bytes
// as fp16 as B; its result is, lane for lane, the B operand of O^T = V^T P^T, whose A are V's bytes as fp16.  The order of channels
// inside a product and of keys inside a page is free, and chosen so that every lane reads sixteen bytes of a row at a time and nothing
// has to be moved between lanes or registers.
//
// Loads.  Every warp copies its own pages, two at a time, into one of two places in shared memory (cp.async, no barrier but the
// warp's) and runs ahead into the CTA's next item, whose page numbers were fetched an item earlier.
//
// Range.  The weights reach the second product as fp16 numbers p_j vs_j: what is rounded is each key's contribution relative to the
// largest one, whatever the size of V, and a key that has weight but no V (a row of zeros has the least scale) cannot push the others
// out of fp16's range.  Scores are formed in fp32 from up to 2^27 times ks, and weights of keys are lost below 2^-126 times the power
// of two of V's scale: rows of K and V may be as large as 2^100.  m begins as the largest contribution of a warp's first pair of pages
// and is raised only when a weight passes kGrow = 2^14, a quarter of fp16's range, which leaves the accumulators alone for nearly all
// pages.
//
// What bounds it, and what it measured (B200, 64 q and 8 KV heads of 128, join included).  Decode: the copies.  One sequence of 131072
// keys 57 us in int8, 55.5 in fp8 (277 MB: 4.9 and 5.0 TB/s; the same loop with its copies alone 48 us), 24 sequences of 2000 to 4001
// in fp8 34.7 us (155 MB, 4.5 TB/s; 30 us), one of 700 7.3 us: launch, one page's latency, join.  Verify blocks (4 sequences of 5626
// to 9001, 6 rows each, int8): 51 us for 63 MB, the chain of products, weights and conversions of two warps a scheduler (0.42
// instructions a cycle; 680 of them a pair of pages and 700 an item of six pairs, three or four items a CTA); sixteen columns an item:
// twenty-four were 7 % slower and eight convert all of K and V twice as often. Tried and slower: codes in registers instead of shared
// memory (24 sequences 53 us), pages converted once for 64 columns by all warps together (verify 66 us when this took 54; a barrier
// every pair of pages), bulk copies of four rows (41 and 63 us: they arrive later), tcgen05 products with V converted into shared
// memory (54 and 56 us, 77 for 131072 keys: with eight columns the products are all issue and latency, and rows of verify blocks must
// not differ from decode), joining in the last CTA of a row (45 us).
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
constexpr int kJoin = 16;                   // splits that are joined at once
constexpr float kNoRef = -3.4028234e38f;    // m before the first key
constexpr float kGrow = 16384.f;              // what a weight may reach before m follows

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// The square root of 2^(m - to).  Sums of p are brought from m to another reference in two such steps: beside rows of V near the largest
// numbers, m of rows of zeros lies more than 126 lower, and 2^(m - to) is no number, while their p (as much larger) still count.
__device__ __forceinline__ float ex2_half(float m, float to) { return ex2(__fmul_rn(0.5f, __fadd_rn(m, -to))); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Taken off here and not from the finished sums (64 instructions a pair of pages less, 1 % of the time): the accumulators truncate,
// and 1152 in every term cost a flat row of 131072 keys half of its last bf16 digit.
__device__ __forceinline__ uint32_t minus_1152(uint32_t two) {
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&two), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&v);
}
// The four channels of a K word as fp16 pairs (0, 1) and (2, 3)
template <int FMT>
__device__ __forceinline__ void k_pairs(uint32_t w, uint32_t& x, uint32_t& y) {
  if (FMT == KV8_INT8) {
    x = minus_1152(__byte_perm(w, 0x64646464u, 0x4140));               // 0x64xx is 1024 + xx
    y = minus_1152(__byte_perm(w, 0x64646464u, 0x4342));
  } else {
    e4m3_pairs(w, x, y);
  }
}
// Of two rows' words: pairs (row a, row b) of bytes 2 * HI and 2 * HI + 1
template <int FMT, int HI>
__device__ __forceinline__ void cross_pairs(uint32_t wa, uint32_t wb, uint32_t& x, uint32_t& y) {
  if (FMT == KV8_INT8) {
    const uint32_t z = __byte_perm(wa, wb, HI ? 0x7632 : 0x5410);
    x = minus_1152(lop3_and_or(z, 0x00ff00ffu, 0x64006400u));          // 0x64xx is 1024 + xx
    y = minus_1152(__byte_perm(z, 0x64646464u, 0x4341));
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
// for K these are two neighbouring rows times four pieces, for V every fourth row times two.
template <int HD>
struct Ring {
  static constexpr int kSlab = kKv8Page * HD;
  uint32_t dst_k, dst_v[kSlab / 512];                // a lane's copies: 512 bytes a turn
  uint32_t rd_k, rd_v;
  __device__ __forceinline__ Ring(int lane) {
    const int g = lane >> 2, t = lane & 3, l4 = lane >> 3, c = lane & 7;
    // lines 4k + l4.  K: by the row's parity (rows of 64 channels lie right as they are); V: by the row / 4
    dst_k = l4 * 128 + ((c ^ (HD == 128 ? (l4 & 1) * 4 : 0)) << 4);
#pragma unroll
    for (int k = 0; k < kSlab / 512; ++k) dst_v[k] = kSlab + (4 * k + l4) * 128 + ((c ^ ((HD == 128 ? k : 2 * k + (l4 >> 1)) * 2)) << 4);
    rd_k = HD == 128 ? (4 * (g >> 1) + (g & 1)) * 128 + ((t ^ (g & 1) * 4) << 4) : 2 * (g >> 1) * 128 + ((g & 1) * 4 + t << 4);
    rd_v = kSlab + (HD == 128 ? 4 * t * 128 + ((g ^ t * 2) << 4) : 2 * t * 128 + (((g >> 1) ^ t * 2) << 4) + (g & 1) * 8);
  }
  // `blk` is the block's address plus 16 * lane
  __device__ __forceinline__ void copy(uint32_t stage, const uint8_t* blk, int lane) const {
#pragma unroll
    for (int k = 0; k < kSlab / 512; ++k) {
      cp_async16(stage + dst_k + k * 512, blk + k * 512);
      cp_async16(stage + dst_v[k], blk + kSlab + k * 512);
    }
    if (lane < 8) cp_async16(stage + 2 * kSlab + 16 * lane, blk + 2 * kSlab);
  }
  // row 4 (g / 2) + g % 2 + 2 r, piece t + 4c
  __device__ __forceinline__ uint4 k(uint32_t stage, int r, int c) const {
    if (HD == 128) return lds128(stage + r * 256 + (rd_k ^ (c * 64)));
    return lds128(stage + r * 128 + rd_k);
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
  int tok0, cnt, first, last, seq, ns, col0, kvh, split;
  int pairs, page;                       // pairs of pages of this warp, at least one; lane i holds the number of page i, -1 if none
};

template <int HD>
constexpr int attn_smem() { return kWarps * 2 * 2 * kv8_block_bytes(HD); }

template <int HD, int FMT, int NT>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) kv8_attn_kernel(const Kv8AttnArgs a) {
  constexpr int KC = HD / 64;            // 16-byte pieces of a K row per lane
  constexpr int VW = HD / 32;            // words of a V row per lane
  constexpr int MT = HD / 16;            // channel tiles of V^T P^T
  constexpr int QK = HD / 16;            // k-steps of q K^T
  constexpr int COLS = NT * 8;
  constexpr int LDO = HD + 4;
  constexpr int BLK = kv8_block_bytes(HD), PAIR = 2 * BLK;
  // a warp's results of an item go over the pair of pages that it used last, which is not refilled before they have been read
  static_assert(COLS * LDO * 4 <= PAIR, "a tile of results fits a pair of pages");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float sh_m[COLS][kWarps], sh_l[COLS][kWarps];
  __shared__ __align__(16) int sh_at[kWarps];
  // a column's first part, or its place in the output if it has one split; its splits, 0 behind the last column
  struct __align__(16) Target { long to; int ns; };
  __shared__ Target sh_to[COLS];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int gq = a.hq / a.hkv;
  const Ring<HD> ring(lane);
  const uint32_t mem = smem_u32(smem) + warp * 2 * PAIR, flip = mem ^ (mem + PAIR);

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
  auto fetch = [&](int at, Item& it, bool next) {
    if (next && it.split + 1 < it.ns) {
      ++it.split;
    } else {
      while (at - base >= total) { base += total; load_run(run + 1); }
      at -= base;
      const int src = __ffs(__ballot_sync(0xffffffffu, incl > at)) - 1;
      at -= __shfl_sync(0xffffffffu, incl, src) - __shfl_sync(0xffffffffu, mine, src);
      it.tok0 = __shfl_sync(0xffffffffu, grp.tok0, src); it.cnt = __shfl_sync(0xffffffffu, grp.cnt, src);
      it.first = __shfl_sync(0xffffffffu, grp.first, src); it.last = __shfl_sync(0xffffffffu, grp.last, src);
      it.seq = __shfl_sync(0xffffffffu, grp.seq, src);
      it.ns = splits_of(it.last, a.split_keys);
      const int ctiles = (it.cnt * gq + COLS - 1) / COLS;
      it.split = at % it.ns; at /= it.ns;
      it.col0 = at % ctiles * COLS; it.kvh = at / ctiles;
    }
    const int k_begin = it.split * a.split_keys, k_end = min(it.last + 1, k_begin + a.split_keys);
    const int n_pg = (k_end - k_begin + kKv8Page - 1) / kKv8Page;           // 0 for a group without keys
    const int n_my = (n_pg - warp + kWarps - 1) / kWarps;                   // at most 32: split_keys is at most 2048
    it.pairs = max((n_my + 1) >> 1, 1);
    it.page = -1;
    if (lane < n_my) it.page = a.block_table[(size_t)it.seq * a.bt_ld + k_begin / kKv8Page + warp + kWarps * lane];
    __syncwarp();
  };
  Item cur, nxt;
  fetch(item, nxt, false);
  cur = nxt;
  uint32_t rd = mem;                     // the pair in use; the other one is under way
  const int stride = a.hkv * BLK;
  // Sends for pair x of cur, or the first of nxt once cur has no more; every call is one group of copies, so that all but the last
  // group have arrived when at most one is under way.  A page that is not there is not copied: its keys are masked below.
  auto send = [&](uint32_t stage, int x) {
    const bool mine = x < cur.pairs;
    const uint8_t* base = a.pool + (mine ? cur.kvh : nxt.kvh) * BLK + 16 * lane;
    const int page = mine ? cur.page : nxt.page, at = mine ? 2 * x : 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = __shfl_sync(0xffffffffu, page, at + h);
      if ((unsigned)p < (unsigned)a.n_pages) ring.copy(stage + h * BLK, base + (long)p * stride, lane);
    }
    cp_async_commit();
  };

  // q, every column scaled by a power of two; qs undoes it on the scores and brings the softmax scale.
  // The largest value lies in [2^10, 2^11): a bf16 number keeps its eight digits down to 2^-27 of that (fp16's step there is 2^-24), and
  // sums of 128 products with codes up to 448 stay below 2^28.  int8 keys once went into an integer product as they are, with q as two
  // bytes of fixed point: 4 to 6 % less time (131072 keys 54.2 us instead of 56.1, the verify block 47.6 instead of 50.6), but a channel
  // below 2^-7 of the largest one lost digits, and with a channel of K as much larger the result was off by up to a tenth.  A third byte
  // of q mends that too and takes longer (58.3 and 52.7).
  uint32_t qa[QK][4];
  float qs[NT];

  send(rd, 0);
  for (bool same_q = false; item < item_end; ++item) {
    if (same_q) same_q = nxt.tok0 == cur.tok0 && nxt.cnt == cur.cnt && nxt.col0 == cur.col0 && nxt.kvh == cur.kvh;
    cur = nxt;
    if (item + 1 < item_end) fetch(item + 1, nxt, true); else nxt.page = -1;
    const int tok0 = cur.tok0, cnt = cur.cnt, first = cur.first, last = cur.last, col0 = cur.col0, kvh = cur.kvh, split = cur.split, pairs = cur.pairs;
    const int k_begin = split * a.split_keys, k_end = min(last + 1, k_begin + a.split_keys);
    const unsigned valid = __ballot_sync(0xffffffffu, (unsigned)cur.page < (unsigned)a.n_pages);
    send(rd ^ flip, 1);

    if (!same_q) {
      if (threadIdx.x < COLS) {
        const int col = col0 + threadIdx.x;
        Target x = {0, 0};
        if (col < cnt * gq) {
          const int tok = tok0 + col / gq, head = kvh * gq + col % gq;
          x.ns = cnt == 1 ? cur.ns : splits_of(min(a.tok_pos[tok], last), a.split_keys);
          x.to = x.ns == 1 ? (long)tok * a.ldo + (long)head * HD : ((long)tok * a.hq + head) * a.max_splits;
        }
        sh_to[threadIdx.x] = x;
      }
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
        const uint32_t e = min(264u - (top >> 23), 253u);
        // an infinity or a NaN in q: every score is NaN; those of keys that are not seen become -infinity like any other
        const float up = top >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : __uint_as_float(e << 23);
        qs[n] = __fmul_rn(__uint_as_float((254u - e) << 23), a.scale_log2);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int w = 0; w < 4; ++w) {                // four channels of a K word; rows g and g + 8 of the tile: columns g and g + 8
            const uint32_t a0 = (&raw[c][w >> 1].x)[2 * (w & 1)], a1 = (&raw[c][w >> 1].x)[2 * (w & 1) + 1];
            qa[c * 4 + w][n] = pack_half(__uint_as_float(a0 << 16) * up, __uint_as_float(a0 & 0xffff0000u) * up);
            qa[c * 4 + w][2 + n] = pack_half(__uint_as_float(a1 << 16) * up, __uint_as_float(a1 & 0xffff0000u) * up);
            if (NT == 1) qa[c * 4 + w][1] = qa[c * 4 + w][3] = 0u;
          }
      }
    }
    same_q = true;

    // o: channels g * HD / 8 + 2k (0, 1) and + 1 (2, 3) of columns 2t (0, 2) and 2t + 1 (1, 3); m and l: of column g
    float o[NT][MT][4], m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = kNoRef; l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
    }

    for (int i = 0; i < pairs; ++i) {
      cp_async_wait<1>();
      __syncwarp();
      const uint32_t stage = rd;
      // s[h][n]: page 2i + h of this warp, column n * 8 + g, keys 4t .. 4t + 3
      float s[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint4 k = ring.k(stage + h * BLK, r, c);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t b0, b1;
              k_pairs<FMT>((&k.x)[w], b0, b1);
              mma_f16_16816(x, qa[c * 4 + w], b0, b1);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) { s[h][n][2 * r] = x[2 * n]; s[h][n][2 * r + 1] = x[2 * n + 1]; }
        }
      }
      float vs[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint4 su = lds128(stage + h * BLK + 2 * kKv8Page * HD + t * 32 + r * 16);       // (K, V) scales of two keys
          vs[h][2 * r] = __uint_as_float(su.y); vs[h][2 * r + 1] = __uint_as_float(su.w);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            s[h][n][2 * r] = __fmul_rn(s[h][n][2 * r], __uint_as_float(su.x));
            s[h][n][2 * r + 1] = __fmul_rn(s[h][n][2 * r + 1], __uint_as_float(su.z));
          }
        }
      const int kb = k_begin + (warp + 2 * kWarps * i) * kKv8Page;          // the pair's second page begins 64 keys later
      const unsigned have = valid >> 2 * i & 3u;
      // from the group's first slot on, at the split's end and where a page is missing, keys are looked at one by one
      const bool partly = kb + (kWarps + 1) * kKv8Page > min(first, k_end) || have != 3u;
      if (partly) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int row = min((col0 + n * 8 + g) / gq, cnt - 1);
          const int pos = cnt == 1 ? last : min(a.tok_pos[tok0 + row], last);
          const unsigned mask = a.tree_mask ? a.tree_mask[tok0 + row] : 0u;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = kb + h * kWarps * kKv8Page + 4 * t + j, in = key - first;
              const bool seen = key <= pos && key < k_end && (have >> h & 1u) && (!a.tree_mask || in < 0 || (in < 32 && ((mask >> (in & 31)) & 1u)));
              if (!seen) s[h][n][j] = -INFINITY;
            }
        }
        __syncwarp();
      }
      float w[2][NT][4];
      float sum[NT];
      auto weigh = [&]() {
        float top = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          sum[n] = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float p = ex2(__fmaf_rn(s[h][n][j], qs[n], -m[n]));
              sum[n] = __fadd_rn(sum[n], p);
              w[h][n][j] = __fmul_rn(p, vs[h][j]);
            }
          if (partly)             // a key that is not seen may have the scale NaN
#pragma unroll
            for (int j = 0; j < 8; ++j) if (s[j >> 2][n][j & 3] == -INFINITY) w[j >> 2][n][j & 3] = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) top = fmaxf(top, w[j >> 2][n][j & 3]);
        }
        return top;
      };
      if (i == 0 || __any_sync(0xffffffffu, weigh() > kGrow)) {
        // columns that passed it: m becomes their largest s + log2 of vs's power of two, so that weights begin below 2 again
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float top = i == 0 ? INFINITY : 0.f, mx = kNoRef;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (i != 0) top = fmaxf(top, w[j >> 2][n][j & 3]);
            const float e = __uint_as_float(0x4b000000u | (__float_as_uint(vs[j >> 2][j & 3]) >> 23)) - 8388735.f;
            mx = fmaxf(mx, __fadd_rn(__fmul_rn(s[j >> 2][n][j & 3], qs[n]), e));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          float f = 1.f;
          float half = 1.f;
          if (top > kGrow) { half = ex2_half(m[n], mx); f = __fmul_rn(half, half); m[n] = mx; }
          if (i == 0) continue;                     // nothing has been added up
          l[n] = __fmul_rn(__fmul_rn(l[n], half), half);
          const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            o[n][k][0] = __fmul_rn(o[n][k][0], f0); o[n][k][1] = __fmul_rn(o[n][k][1], f1);
            o[n][k][2] = __fmul_rn(o[n][k][2], f0); o[n][k][3] = __fmul_rn(o[n][k][3], f1);
          }
        }
        weigh();
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) l[n] = __fadd_rn(l[n], sum[n]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) { pb[n][0] = pack_half(w[h][n][0], w[h][n][1]); pb[n][1] = pack_half(w[h][n][2], w[h][n][3]); }
        uint32_t vw[4][VW];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ring.v(stage + h * BLK, r, vw[r]);
          // bytes past the end may be e4m3's NaN, which a weight of zero does not silence
          if (FMT == KV8_FP8 && partly && (kb + h * kWarps * kKv8Page + 4 * t + r >= k_end || !(have >> h & 1u)))
#pragma unroll
            for (int x = 0; x < VW; ++x) vw[r][x] = 0u;
        }
        if (h == 1) {
          __syncwarp();                             // the pair has been read
          if (i + 1 < pairs) {                      // the last pair's place holds the results first
            send(rd, i + 2);
            rd ^= flip;
          }
        }
#pragma unroll
        for (int x = 0; x < VW; ++x) {
          uint32_t f[4];
          cross_pairs<FMT, 0>(vw[0][x], vw[1][x], f[0], f[1]);
          cross_pairs<FMT, 0>(vw[2][x], vw[3][x], f[2], f[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][2 * x], f, pb[n][0], pb[n][1]);
          cross_pairs<FMT, 1>(vw[0][x], vw[1][x], f[0], f[1]);
          cross_pairs<FMT, 1>(vw[2][x], vw[3][x], f[2], f[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16_16816(o[n][2 * x + 1], f, pb[n][0], pb[n][1]);
        }
      }
    }

    float (*tile)[LDO] = reinterpret_cast<float (*)[LDO]>(smem + (rd - smem_u32(smem)));
    if (lane == 0) sh_at[warp] = rd - smem_u32(smem);
    rd ^= flip;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float x = l[n];
      x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = __fadd_rn(x, __shfl_xor_sync(0xffffffffu, x, 2));
      if (t == 0) { sh_m[n * 8 + g][warp] = m[n]; sh_l[n * 8 + g][warp] = x; }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int k = 0; k < MT; k += 2)
          *reinterpret_cast<float4*>(&tile[n * 8 + 2 * t + j][g * (HD / 8) + 2 * k]) =
              make_float4(o[n][k][j], o[n][k][2 + j], o[n][k + 1][j], o[n][k + 1][2 + j]);
      }
    }
    __syncthreads();
    const int4 at = *reinterpret_cast<const int4*>(sh_at);
#pragma unroll
    for (int i = threadIdx.x; i < COLS * (HD / 4); i += kWarps * 32) {
      const int c = i / (HD / 4), d = i % (HD / 4) * 4;
      const Target target = sh_to[c];
      const int ns = target.ns;
      const long to = target.to;
      if (split >= ns) continue;
      const float4 ms = *reinterpret_cast<const float4*>(sh_m[c]), ls = *reinterpret_cast<const float4*>(sh_l[c]);
      const float M = fmaxf(fmaxf(fmaxf(ms.x, ms.y), ms.z), ms.w);
      float L = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float half = ex2_half((&ms.x)[w], M), f = __fmul_rn(half, half);
        const float4 y = *reinterpret_cast<const float4*>(smem + (&at.x)[w] + (c * LDO + d) * 4);
        L = __fmaf_rn(__fmul_rn((&ls.x)[w], half), half, L);
        x.x = __fmaf_rn(y.x, f, x.x); x.y = __fmaf_rn(y.y, f, x.y); x.z = __fmaf_rn(y.z, f, x.z); x.w = __fmaf_rn(y.w, f, x.w);
      }
      if (ns == 1) {
        const float inv = L == 0.f ? 0.f : __fdiv_rn(1.f, L);
        uint2 v;
        *reinterpret_cast<__nv_bfloat162*>(&v.x) = __floats2bfloat162_rn(__fmul_rn(x.x, inv), __fmul_rn(x.y, inv));
        *reinterpret_cast<__nv_bfloat162*>(&v.y) = __floats2bfloat162_rn(__fmul_rn(x.z, inv), __fmul_rn(x.w, inv));
        *reinterpret_cast<uint2*>(a.out + to + d) = v;
      } else {
        const long slot = to + split;
        *reinterpret_cast<float4*>(a.part_o + slot * HD + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + slot * 2) = make_float2(M, L);
      }
    }
    __syncthreads();                                // results have been read: their places take pages again
    // pages that are named and not there: reported once an item, -1 past the split's end is none
    const int n_pg = (k_end - k_begin + kKv8Page - 1) / kKv8Page;
    if (warp + kWarps * lane < n_pg && !(valid >> lane & 1u)) atomicExch(a.status, (int)B2_ERR_BOUNDS);
  }
}

// Joins the splits of rows that have more than one.  A block of kJoin neighbouring splits is one warp's: all its parts are under way
// at once and added in order.  `warps` of them share a (row, q head); block b is warp b % 16's, the warps' sums are added in order.
// With warps == 1 (rows of at most sixteen splits) a CTA has four (row, q head)s.  Neither choice changes a row's bits:
//     o = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M),    M = max_s m_s
// Bound by latency: a warp's loads, the exchange and the launch.  171 splits of 64 heads (131072 keys) add 3 to 6 us to the kernel before,
// two to six splits 1.6 to 2.5; with a head's parts loaded one after the other it was 2 us more at 256 splits.
template <int HD>
__global__ void __launch_bounds__(512) kv8_join_kernel(const Kv8AttnArgs a, int rows_at_once, int warps) {
  constexpr int PER = HD / 32;
  using Vec = std::conditional_t<PER == 4, float4, float2>;
  __shared__ float sh_x[16][HD], sh_m[16], sh_l[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int task = warps == 1 ? blockIdx.x * 4 + warp : blockIdx.x, w = warps == 1 ? 0 : warp;
  const int head = task % a.hq, r0 = task / a.hq % rows_at_once;
  // (groups and positions are from before the kernel that this one follows, which has waited for them)
  const Group grp = group_at(a, task / a.hq / rows_at_once);
  pdl_wait();
  pdl_launch_dependents();
  if (!grp.ok) return;
  for (int r = r0; r < grp.cnt; r += rows_at_once) {
    const int tok = grp.tok0 + r;
    const int ns = splits_of(grp.cnt == 1 ? grp.last : min(a.tok_pos[tok], grp.last), a.split_keys);
    if (ns == 1) continue;
    const size_t slot = ((size_t)tok * a.hq + head) * a.max_splits;
    float M = kNoRef, L = 0.f, x[PER];
#pragma unroll
    for (int d = 0; d < PER; ++d) x[d] = 0.f;
    for (int s0 = w * kJoin; s0 < ns; s0 += warps * kJoin) {
      const int n = min(ns - s0, kJoin);
      const float2 part = lane < n ? reinterpret_cast<const float2*>(a.part_ml)[slot + s0 + lane] : make_float2(kNoRef, 0.f);
      const Vec* po = reinterpret_cast<const Vec*>(a.part_o + (slot + s0) * HD) + lane;
      Vec y[kJoin];
#pragma unroll
      for (int j = 0; j < kJoin; ++j) y[j] = po[min(j, n - 1) * 32];        // past the end: the last part again, with the weight zero
      const float m = warp_max(part.x), M2 = fmaxf(M, m), half = lane < n ? ex2_half(part.x, m) : 0.f, f = __fmul_rn(half, half);
      float z[PER], l = warp_sum(__fmul_rn(__fmul_rn(part.y, half), half));
#pragma unroll
      for (int d = 0; d < PER; ++d) z[d] = 0.f;
#pragma unroll
      for (int j = 0; j < kJoin; ++j) {
        const float fj = __shfl_sync(0xffffffffu, f, j);
#pragma unroll
        for (int d = 0; d < PER; ++d) z[d] = __fmaf_rn((&y[j].x)[d], fj, z[d]);
      }
      const float old_half = ex2_half(M, M2), add_half = ex2_half(m, M2), old = __fmul_rn(old_half, old_half), add = __fmul_rn(add_half, add_half);
      M = M2;
      L = __fmaf_rn(__fmul_rn(l, add_half), add_half, __fmul_rn(__fmul_rn(L, old_half), old_half));
#pragma unroll
      for (int d = 0; d < PER; ++d) x[d] = __fmaf_rn(z[d], add, __fmul_rn(x[d], old));
    }
    if (warps > 1 && ns > kJoin) {
#pragma unroll
      for (int d = 0; d < PER; ++d) sh_x[warp][lane * PER + d] = x[d];
      if (lane == 0) { sh_m[warp] = M; sh_l[warp] = L; }
      __syncthreads();
      if (warp == 0)
        for (int v = 1; v < warps; ++v) M = fmaxf(M, sh_m[v]);
      const float own_half = ex2_half(sh_m[0], M), own = __fmul_rn(own_half, own_half);
      if (warp == 0) {
        L = __fmul_rn(__fmul_rn(L, own_half), own_half);
#pragma unroll
        for (int d = 0; d < PER; ++d) x[d] = __fmul_rn(x[d], own);
        for (int v = 1; v < warps; ++v) {
          const float half = ex2_half(sh_m[v], M), f = __fmul_rn(half, half);
          L = __fmaf_rn(__fmul_rn(sh_l[v], half), half, L);
#pragma unroll
          for (int d = 0; d < PER; ++d) x[d] = __fmaf_rn(sh_x[v][lane * PER + d], f, x[d]);
        }
      }
      __syncthreads();
    }
    if (w == 0) {
      const float inv = L == 0.f ? 0.f : __fdiv_rn(1.f, L);
      bf16* out = a.out + (size_t)tok * a.ldo + (size_t)head * HD + lane * PER;
#pragma unroll
      for (int d = 0; d < PER; d += 2) *reinterpret_cast<__nv_bfloat162*>(out + d) = __floats2bfloat162_rn(__fmul_rn(x[d], inv), __fmul_rn(x[d + 1], inv));
    }
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
    const int warps = std::min((a.max_splits + kJoin - 1) / kJoin, 16);
    const long tasks = (long)a.n_groups * rows * a.hq;
    e = launch(kv8_join_kernel<HD>, (unsigned)(warps == 1 ? (tasks + 3) / 4 : tasks), warps == 1 ? 128 : 32 * warps, 0, st, a, (int)rows, warps);
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
