// Attention of a few query tokens over the paged FP8 cache (kv_pages.cuh):
// softmax(q K^T * scale) V per query row, K = code * page scale, and the weight that every cached
// token receives added to its mass.
//
// The cache is read once and that bounds it: 2 D bytes per token and KV head against
// 4 D * rows operations, far below the tensor cores' rate for the few rows (query heads of one KV
// head x query tokens) of a decode step. So the products run on mma.sync.m16n8k16 (f16 in, fp32
// accumulators): e4m3 -> f16 is one exact conversion per two codes, and the instruction's fragments
// let the codes go from shared memory to the tensor core without leaving the warp. The cache is its
// 16-row operand in both products, S^T = K Q^T and O^T = V^T P^T, and the query rows its 8 columns
// (one group of 8, or two; four rows twice): no operand is padding where a KV head has 4 or 8 rows. (With the queries as the
// 16-row operand the same kernel had twice the products and outputs: 66 us against 60 at 4 sequences
// of 131072 tokens.) What has to be fast is the stream: every warp keeps its own ring of slabs of K
// and V in flight with cp.async (32 tokens each, 16 where a page has no more: 54 us against 60) and
// never waits for another warp inside an item.
//
//  * Work is cut into equal parts whatever the lengths: the slabs of all (sequence, KV head, row
//    tile) items stand in one line, and each block takes a contiguous part of it. A block's first
//    and last item may be shared with its neighbours: their partial results (maximum, sum,
//    output) go to two slots of the block's own, and a second small launch merges them in an
//    order of their own, so the same inputs give the same bits.
//  * Queries enter as f16, each row in units of a power of two that puts its largest value in
//    [2^14, 2^15): bf16 and f16 values keep all their bits down to 2^-29 of the row's largest;
//    fp32 ones are split into two f16 terms (22 bits) and the product is taken twice.
//  * The weights enter the product with V in two f16 terms too (22 bits; with one, outputs were off by up
//    to 2^-12 of sum p |v|, a tenth more than f16's own rounding in all). Up to four rows, as with four
//    query heads per KV head, leave half of the MMA's columns: these hold the rows once more, take the second
//    terms and are added at an item's end, at no product more (64 x 2048: 31.9 -> 32.2 us, 4 x 65536 of
//    D = 64: 52.0 -> 52.4). More rows take the product twice (4 x 131072, 8 rows: 52.8 both ways; 16 x 4096
//    of 16 rows: 20.8 -> 22.4).
//  * An MMA cuts the sum that it carries to 24 bits instead of rounding it. For fp32 queries the products of 16
//    tokens start from zero and are added to the output by themselves (16 x 60000 tokens, 32 / 8 heads,
//    positive values: off by 3e-7, carried 1.1e-5; 4 x 131072 52.4 -> 53.0 us, 16 x 4096 of 16 rows 24.2 ->
//    27.1). 16-bit outputs, whose last bit is 2^-11 and 2^-8, take the carried sums (f16 with 16 rows: 22.3 us,
//    25.7 otherwise).
//  * The running maximum is that of t = s + log2(V scale), s the score in log2 units: the weight
//    that multiplies the V codes is w = 2^(s - m) * V scale, with m = t - 10 at a slab's largest t,
//    so w fits f16, its two terms keep it to 2^-35 of the largest at least, and the page's scale costs
//    one multiplication. Sums use 2^(s - m) itself, in fp32. (Adding every slab's product to the
//    output with its own scale instead would cost 32 more multiply-adds per lane and slab.)
//    log2(V scale) is cut at -80, which keeps the sums finite; pages whose scale is below about
//    2^-105 lose bits of their values, which are below 2^-96 then.
//
// 4 sequences of 131072 tokens, 16 / 2 heads, D = 128: 52 us = 5.2 TB/s = 0.79 of the measured copy,
// of which about 8 us are fixed (two launches, the line's cut, the pipelines' fill, the merge): one
// sequence of 4096 tokens, whose stream is 1.3 us, takes 10.8 us.
#pragma once

#include "kv_pages.cuh"

namespace kab {

// An item that several blocks share: which one, the first and the last of the blocks and the slot of
// the first (the others' is 0); last -1: no such item.
struct PagesCut {
  int b, h, tile, first, last, slot;
};

struct PagesAttnArgs {
  PagePool pool;
  const void* q;
  int64_t qb, qh, qt;
  void* out;
  float scale_log2;  // sm_scale * log2(e)
  int heads_q, q_len, causal;  // q_len: query tokens of this launch, of those of the call
  int tail;                    // causal: newest tokens of every sequence that belong to later launches' queries
  int q_skip, out_rows;        // the call's query tokens less this launch's; rows of one KV head in `out`
  int rows, row_tiles;   // rows of one KV head (query heads x query tokens), tiles of 4, 8 or 16 of them
  float* partial;        // [grid, 2 slots, a tile's rows, D + 2]: output, maximum, sum
  PagesCut* cuts;        // [items or grid]: the shared items, by item or by the block that begins them
  int cuts_by_item;
  float* scores;         // [batch, heads, rows, capacity] in log2 units, or NULL
  float* ml;             // [batch, heads, rows, 2]: reference and reciprocal sum, with scores
  int64_t capacity;      // max_pages * page_tokens
};

template <int T>
__device__ __forceinline__ void store_elem(void* base, int64_t i, float v) {
  if constexpr (T == kF32) static_cast<float*>(base)[i] = v;
  else if constexpr (T == kBF16) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(base)[i] = __float2half_rn(v);
}

// ------------------------------------------------------------------ instructions

// Two e4m3 codes (low half of `pair`, low byte first) as f16.
__device__ __forceinline__ uint32_t e4m3x2_f16(uint32_t pair) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(r) : "r"(pair));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_f16_high(uint32_t pair) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}" : "=r"(r) : "r"(pair));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 f16x2_values(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a *= c, b *= d in one instruction.
__device__ __forceinline__ void scale_pair(float& a, float& b, float c, float d) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n mul.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
// a += c, b += d in one instruction.
__device__ __forceinline__ void add_pair(float& a, float& b, float c, float d) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n add.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
// An 8 x 8 matrix of f16 over the warp (lane (g, t) holds row g, columns 2 t and 2 t + 1), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// 16 bytes to shared memory without waiting; `bytes` 0 writes zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ------------------------------------------------------------------ layout

// ROWS: query rows that share one pass over the cache: 8 or 16, the MMA's columns, or 4, whose columns 4 .. 7
// hold the same rows again and take the second terms of their weights. SL: tokens of a slab.
template <int D, int ROWS, int SL, bool SPLIT>
struct PagesLayout {
  static constexpr int kWarps = 4, kThreads = kWarps * 32, kRows = ROWS, NR = ROWS == 16 ? 2 : 1, kCols = 8 * NR;
  static constexpr bool kLight = NR == 1 && !SPLIT;
  static constexpr int kSlabBytes = SL * D;  // K or V of one slab
  static constexpr int kStageBytes = 2 * kSlabBytes;
  // blocks per SM by registers and shared memory, and as many stages as fit beside them
  static constexpr int kBlocks = SL == 16 ? (kLight ? 5 : 4) : 3;
  static constexpr int kStages = SL * D == 4096 || (SL == 16 && kLight) ? 2 : 3;
  static constexpr int kQBytes = D / 16 * 32 * 8 * NR * (SPLIT ? 2 : 1);
  // a row of the warps' outputs in the merge: its pitch keeps the fragments' float4 stores two to a bank
  static constexpr int kPitch = D + 4;
  static constexpr int kMergeBytes = kWarps * kRows * (kPitch + 2) * 4;
  static constexpr int kRing = kWarps * kStages * kStageBytes > kMergeBytes ? kWarps * kStages * kStageBytes : kMergeBytes;
  static constexpr int kScales = kWarps * kStages * 2 * 4;
  static constexpr int kSmem = kQBytes + kRing + kScales + kCols * 4 + 32;
};

// Byte offset of 16-byte chunk `chunk` of token `row` in a slab: the chunks are permuted so that
// both readers touch all 32 banks: K (8 consecutive tokens x 4 lanes' chunks) and V (every second
// token x neighbouring chunks).
template <int D>
__device__ __forceinline__ uint32_t slab_offset(int row, int chunk) {
  if constexpr (D == 128) return row * 128 + ((chunk ^ (row & 7)) << 4);
  else return (row >> 1) * 128 + (((((row & 1) << 2) | chunk) ^ (((row >> 1) & 3) << 1)) << 4);
}

// An item's queries, pipeline fill, merge and output cost a block about as much as 20 slabs of 16 tokens
// (64 sequences of up to 2048 tokens: 45.8 us with 2, 35.2 with 6, 31.9 with 20, 33.4 with 40).
constexpr int kItemCost = 20;
constexpr float kNoScore = -3.3e38f;  // below every finite score
// A row's weights are at most 2^10 when its reference is set; the reference moves again only when
// one would pass 2^15.9, the end of f16: rarely after the first slab, while every row's running
// maximum would move often enough to rescale a lane's outputs in most slabs.
constexpr float kWeightBits = 10.0f, kWeightRoom = 5.9f;
constexpr float kLeastLogScale = -80.0f;

// ------------------------------------------------------------------ the kernel

// Where a position of the line of slabs lies: sequence, head, row tile, and the item's first unit.
struct PagesItem {
  int b, h, tile, length, slabs;
  unsigned first;
};

// Tokens of sequence b that any query of this launch sees, cut to what the page table can hold.
__device__ __forceinline__ int pages_tokens(const PagesAttnArgs& a, int b) {
  const int cap = a.pool.max_pages << a.pool.page_shift;
  return max(min(max(__ldg(a.pool.lengths + b), 0), cap) - a.tail, 0);
}

// Four output elements of row r (of a KV head's rows) from their weighted sum and the row's sum.
template <int T, int D>
__device__ __forceinline__ void pages_finish(const PagesAttnArgs& a, int b, int h, int r, int d, int n, float4 acc,
                                             float ref, float sum) {
  const int seen = a.causal ? max(0, n - a.q_len + 1 + r % a.q_len) : n;
  const float inv = seen > 0 ? 1.0f / sum : 0.0f;  // a row that sees nothing gives zeros
  const int64_t head = static_cast<int64_t>(b) * a.pool.heads + h, row = head * a.rows + r;
  const int64_t at = (head * a.out_rows + r + (a.q_skip != 0 ? r / a.q_len * a.q_skip : 0)) * D + d;
  if constexpr (T == kF32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
        make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  } else {
    store_elem<T>(a.out, at, acc.x * inv);
    store_elem<T>(a.out, at + 1, acc.y * inv);
    store_elem<T>(a.out, at + 2, acc.z * inv);
    store_elem<T>(a.out, at + 3, acc.w * inv);
  }
  if (d == 0 && a.ml != nullptr) {
    a.ml[2 * row] = ref;
    a.ml[2 * row + 1] = inv;
  }
}

template <int T, int D, int ROWS, int SL>
__global__ void __launch_bounds__(PagesLayout<D, ROWS, SL, T == kF32>::kThreads, PagesLayout<D, ROWS, SL, T == kF32>::kBlocks)
pages_attention_kernel(PagesAttnArgs a, unsigned* status) {
  using L = PagesLayout<D, ROWS, SL, T == kF32>;
  constexpr int NR = L::NR, COLS = L::kCols;
  constexpr bool SPLIT = T == kF32, Q_HELD = NR == 1 && !SPLIT, TWICE = ROWS == 4;
  constexpr int U = SL / 16, SHIFT = SL == 16 ? 4 : 5;  // 16-token parts of a slab
  constexpr int COST = kItemCost * 16 / SL;
  constexpr int ST = L::kStages, NW = L::kWarps, NT = L::kThreads, PITCH = L::kPitch;
  constexpr int STEPS = D / 16, MT = D / 16, CHUNKS = D / 16, COPIES = SL * D / 512;
  extern __shared__ __align__(128) uint8_t smem[];
  uint2* q_frag = reinterpret_cast<uint2*>(smem);                  // [hi, lo][NR][STEPS][32]
  uint8_t* ring = smem + L::kQBytes;
  float* sc_all = reinterpret_cast<float*>(ring + L::kRing);
  float* q_unit = sc_all + NW * ST * 2;                            // [COLS] units of the query rows
  int* shared_i = reinterpret_cast<int*>(q_unit + COLS);
  float* merge_o = reinterpret_cast<float*>(ring);                 // [NW][ROWS][PITCH]
  float* merge_ml = merge_o + NW * ROWS * PITCH;                   // [NW][ROWS][2]

  const PagePool& p = a.pool;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int P = 1 << p.page_shift, group = a.heads_q / p.heads, per_seq = p.heads * a.row_tiles;

  // the merge may be set up while this kernel runs: it waits for its end by itself
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // ---- this block's part of the line
  auto units_of = [&](int b) -> unsigned {
    const int n = pages_tokens(a, b);
    return max((n + SL - 1) >> SHIFT, 1) + COST;  // an empty sequence is one empty slab: its output is written too
  };
  const int chunk = (p.batch + NT - 1) / NT;
  unsigned mine = 0;
  for (int i = 0; i < chunk; ++i) {
    const int b = tid * chunk + i;
    if (b < p.batch) mine += units_of(b) * per_seq;
  }
  unsigned upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  unsigned* warp_sum = reinterpret_cast<unsigned*>(ring);
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
  unsigned total = 0, before = upto - mine;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  // at least four units per block: with fewer, more parts to merge cost more than the idle blocks save
  // (1 x 4096 tokens: 12.1 us with one, 10.5 with four, 11.2 with eight)
  const unsigned grid = min(gridDim.x, max(total / 4u, 1u)), share = total / grid, longer = total % grid;
  if (blockIdx.x >= grid) {
    if (tid == 0 && !a.cuts_by_item) a.cuts[blockIdx.x].last = -1;
    return;
  }
  // the first `longer` blocks take one unit more
  const unsigned lo = share * blockIdx.x + min(blockIdx.x, longer), hi = lo + share + (blockIdx.x < longer);
  auto block_of = [&](unsigned unit) -> unsigned {
    const unsigned split = longer * (share + 1);
    return unit < split ? unit / (share + 1) : longer + (unit - split) / share;
  };
  if (lo >= before && lo < before + mine) {  // one thread: the sequence that `lo` lies in
    unsigned at = before;
    int b = tid * chunk;
    while (lo >= at + units_of(b) * per_seq) at += units_of(b++) * per_seq;
    shared_i[0] = b;
    shared_i[1] = static_cast<int>(at);
  }
  __syncthreads();
  PagesItem it;
  it.b = shared_i[0];
  {
    const unsigned at = shared_i[1], n = units_of(it.b), i = (lo - at) / n;
    it.h = i / a.row_tiles;
    it.tile = i % a.row_tiles;
    it.first = at + i * n;
  }

  uint8_t* my_ring = ring + warp * ST * L::kStageBytes;
  const uint32_t my_ring_s = static_cast<uint32_t>(__cvta_generic_to_shared(my_ring));
  float* my_sc = sc_all + warp * ST * 2;
  const uint32_t my_sc_s = static_cast<uint32_t>(__cvta_generic_to_shared(my_sc));

  // this lane's share of a slab's copies: chunk lane % CHUNKS of every STEP-th token
  constexpr int STEP = 32 / CHUNKS;
  const int k_tok = static_cast<int>(p.st[0]), v_tok = static_cast<int>(p.st[1]);
  const int k_page = static_cast<int>(p.sp[0]), v_page = static_cast<int>(p.sp[1]);
  const int k_lane = lane / CHUNKS * k_tok + lane % CHUNKS * 16, v_lane = lane / CHUNKS * v_tok + lane % CHUNKS * 16;
  const int sc_page = static_cast<int>(lane & 1 ? p.ssp[1] : p.ssp[0]);
  const uint32_t lane_off = slab_offset<D>(lane / CHUNKS, lane % CHUNKS);
  // slab_offset of the share's i-th token: for D = 128 the tokens are 4 apart, which flips bit 2 of the chunk
  auto share_off = [&](int i) -> uint32_t { return (D == 128 && (i & 1) ? lane_off ^ 64u : lane_off) + i * 512; };

  PagesCut cut{0, 0, 0, 0, -1, 0};
  for (unsigned pos = lo; pos < hi;) {
    it.length = max(page_length(p, it.b, status) - a.tail, 0);
    const unsigned end = it.first + units_of(it.b);
    it.slabs = static_cast<int>(end - it.first) - COST;
    // the item's first COST units stand for what an item costs beside its slabs
    const int s0 = max(0, static_cast<int>(pos - it.first) - COST);
    const int s1 = static_cast<int>(min(end, hi) - it.first) - COST;
    pos = end;
    const int n = it.length;
    const int rows = min(ROWS, a.rows - it.tile * ROWS);
    const int seen_by_all = a.causal ? max(0, n - a.q_len + 1) : n;
    if (s1 > 0) {
      // tokens that the row of column c sees
      auto seen_of = [&](int c) -> int {
        return a.causal ? max(0, n - a.q_len + 1 + (it.tile * ROWS + c % ROWS) % a.q_len) : n;
      };

      const uint8_t* kbase = p.codes[0] + it.h * p.sh[0];
      const uint8_t* vbase = p.codes[1] + it.h * p.sh[1];
      const int32_t* table = p.table + it.b * p.table_stride;
      // lane 0 fetches K's scales, lane 1 V's
      const float* sc_base = lane & 1 ? p.scale[1] + it.h * p.ssh[1] : p.scale[0] + it.h * p.ssh[0];
      uint32_t valid = 0;  // bit s: stage s holds a page of the pool

      auto page_at = [&](int slab) -> int {
        if (slab >= s1 || slab * SL >= n) return -1;
        const int page = __ldg(table + (slab >> (p.page_shift - SHIFT)));
        if (static_cast<unsigned>(page) < static_cast<unsigned>(p.num_pages)) return page;
        if (lane == 0) atomicOr(status, kDevBounds);
        return -1;
      };
      auto issue = [&](int slab, int page, int stage) {
        if (page >= 0) {
          const int slot = (slab << SHIFT) & (P - 1);
          const uint8_t* ks = kbase + static_cast<int64_t>(page) * k_page + (slot * k_tok + k_lane);
          const uint8_t* vs = vbase + static_cast<int64_t>(page) * v_page + (slot * v_tok + v_lane);
          const uint32_t dst = my_ring_s + stage * L::kStageBytes;
          if (slab * SL + SL <= seen_by_all) {
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
              copy16(dst + share_off(i), ks + i * STEP * k_tok, 16);
              copy16(dst + share_off(i) + L::kSlabBytes, vs + i * STEP * v_tok, 16);
            }
          } else {
            // zeros past the sequence's end; V of tokens that not every row sees is added apart, so
            // that a NaN there stays with the rows that see it
#pragma unroll
            for (int i = 0; i < COPIES; ++i) {
              const int tok = slab * SL + lane / CHUNKS + i * STEP;
              copy16(dst + share_off(i), ks + i * STEP * k_tok, tok < n ? 16 : 0);
              copy16(dst + share_off(i) + L::kSlabBytes, vs + i * STEP * v_tok, tok < seen_by_all ? 16 : 0);
            }
          }
          if (lane < 2) copy4(my_sc_s + (stage * 2 + lane) * 4, sc_base + static_cast<int64_t>(page) * sc_page);
          valid |= 1u << stage;
        } else {
          valid &= ~(1u << stage);
        }
        copies_commit();
      };

      __syncthreads();  // the previous item's readers of the ring, q_frag and q_unit are done
      const int first = s0 + warp;
#pragma unroll
      for (int i = 0; i < ST - 1; ++i) issue(first + NW * i, page_at(first + NW * i), i);
      int next_page = page_at(first + NW * (ST - 1));

      // ---- the queries, as B fragments: b0 / b1 of step j are dims chunk * 16 + 4 i + {0, 1} / {2, 3}
      // of row g, where lane t reads K's chunks 2 t and 2 t + 1 (D = 128) or t (D = 64)
      {
        constexpr int PARTS = NT / COLS, E = D / PARTS;
        const int r = tid / PARTS, part = tid % PARTS, rr = it.tile * ROWS + r % ROWS;
        float v[E];
        uint32_t top = 0;
        if (r % ROWS < rows) {
          const int hq = it.h * group + rr / a.q_len, qi = rr % a.q_len;
          const int64_t base = it.b * a.qb + hq * a.qh + qi * a.qt + part * E;
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = load_elem<T>(a.q, base + e);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = PARTS / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // 2^(14 - e): the largest value lands in [2^14, 2^15); rows of zeros, infinities or NaN as they are
        const int e = static_cast<int>(top >> 23) - 127;
        const bool plain = top == 0 || top >= 0x7F800000u;
        const float up = plain ? 1.0f : __uint_as_float((127u + 14u - max(e, -100)) << 23);
        if (part == 0) q_unit[r] = 1.0f / up;
#pragma unroll
        for (int e2 = 0; e2 < E; e2 += 2) {
          const int d = part * E + e2, c = d >> 4, i = (d & 15) >> 2, pair = (d >> 1) & 1;
          const int tt = D == 128 ? c >> 1 : c, j = (D == 128 ? (c & 1) * 4 : 0) + i;
          const float x0 = v[e2] * up, x1 = v[e2 + 1] * up;
          uint32_t* slot = reinterpret_cast<uint32_t*>(&q_frag[((r >> 3) * STEPS + j) * 32 + (r & 7) * 4 + tt]) + pair;
          const uint32_t hi2 = f16x2_of(x0, x1);
          *slot = hi2;
          if constexpr (SPLIT) {
            const float2 h = f16x2_values(hi2);
            slot[NR * STEPS * 32 * 2] = plain ? 0u : f16x2_of(x0 - h.x, x1 - h.y);
          }
        }
        __syncthreads();
      }
      uint2 q_held[Q_HELD ? STEPS : 1];
      if constexpr (Q_HELD) {
#pragma unroll
        for (int j = 0; j < STEPS; ++j) q_held[j] = q_frag[j * 32 + lane];
      }
      // rows 2 t and 2 t + 1 of group r: units, reference, sum; O^T fragments of 16 dims x 8 rows
      float unit[NR][2], m[NR][2], l[NR][2], o[NR][MT][4];
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          unit[r][e] = q_unit[r * 8 + 2 * t + e] * a.scale_log2;
          m[r][e] = kNoScore;
          l[r][e] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < MT; ++j) o[r][j][0] = o[r][j][1] = o[r][j][2] = o[r][j][3] = 0.0f;
      }

      int stage = 0;
      for (int slab = first; slab < s1; slab += NW) {
        copies_wait<ST - 2>();
        __syncwarp();
        const int ahead = slab + NW * (ST - 1);
        issue(ahead, next_page, stage == 0 ? ST - 1 : stage - 1);
        next_page = page_at(ahead + NW);
        if ((valid >> stage) & 1u) {
          const uint8_t* kb = my_ring + stage * L::kStageBytes;
          const uint8_t* vb = kb + L::kSlabBytes;
          const float ksc = my_sc[stage * 2], vsc = my_sc[stage * 2 + 1];
          // ---- S^T: tokens g and g + 8 of each 16-token part, rows 2 t and 2 t + 1. Where a slab is
          // one part, two accumulators halve the chain of dependent products.
          constexpr int ACC = U == 1 ? 2 : 1;
          float s[NR][U][4], s2[NR][4];
#pragma unroll
          for (int r = 0; r < NR; ++r) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s2[r][e] = 0.0f;
#pragma unroll
              for (int u = 0; u < U; ++u) s[r][u][e] = 0.0f;
            }
          }
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            const int ch = D == 128 ? 2 * t + h : t;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const uint4 k0 = *reinterpret_cast<const uint4*>(kb + u * 16 * D + slab_offset<D>(g, ch));
              const uint4 k1 = *reinterpret_cast<const uint4*>(kb + u * 16 * D + slab_offset<D>(g + 8, ch));
              const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int j = h * 4 + i;
                const uint32_t ka[4] = {e4m3x2_f16(w0[i]), e4m3x2_f16(w1[i]), e4m3x2_f16_high(w0[i]),
                                        e4m3x2_f16_high(w1[i])};
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                  const uint2 q = Q_HELD ? q_held[Q_HELD ? j : 0] : q_frag[(r * STEPS + j) * 32 + lane];
                  mma_f16(ACC == 2 && (i & 1) ? s2[r] : s[r][u], ka, q.x, q.y);
                  if constexpr (SPLIT) {
                    const uint2 ql = q_frag[((NR + r) * STEPS + j) * 32 + lane];
                    mma_f16(ACC == 2 && (i & 1) ? s2[r] : s[r][u], ka, ql.x, ql.y);
                  }
                }
              }
            }
          }
          const float size = fabsf(vsc), lv = size > 0.0f ? fmaxf(__log2f(size), kLeastLogScale) : kLeastLogScale;
          const int tok = slab * SL + g;
          uint32_t pb[NR][U][2], pl[NR][U][2];
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float c0 = unit[r][0] * ksc, c1 = unit[r][1] * ksc;
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) {
              if constexpr (ACC == 2) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[r][u][e] += s2[r][e];
              }
              scale_pair(s[r][u][0], s[r][u][1], c0, c1);
              scale_pair(s[r][u][2], s[r][u][3], c0, c1);
            }
            if (slab * SL + SL > seen_by_all) {
              const int seen0 = seen_of(r * 8 + 2 * t), seen1 = seen_of(r * 8 + 2 * t + 1);
#pragma unroll
              for (int u = 0; u < U; ++u) {
                if (tok + 16 * u >= seen0) s[r][u][0] = -INFINITY;
                if (tok + 16 * u >= seen1) s[r][u][1] = -INFINITY;
                if (tok + 16 * u + 8 >= seen0) s[r][u][2] = -INFINITY;
                if (tok + 16 * u + 8 >= seen1) s[r][u][3] = -INFINITY;
              }
            }
            if (a.scores != nullptr) {
              float* at = a.scores +
                          ((static_cast<int64_t>(it.b) * p.heads + it.h) * a.rows + it.tile * ROWS + r * 8 + 2 * t) * a.capacity + tok;
#pragma unroll
              for (int u = 0; u < U; ++u) {
                if (r * 8 + 2 * t < rows) at[16 * u] = s[r][u][0], at[16 * u + 8] = s[r][u][2];
                if (r * 8 + 2 * t + 1 < rows)
                  at[a.capacity + 16 * u] = s[r][u][1], at[a.capacity + 16 * u + 8] = s[r][u][3];
              }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              t0 = fmaxf(t0, fmaxf(s[r][u][0], s[r][u][2]));
              t1 = fmaxf(t1, fmaxf(s[r][u][1], s[r][u][3]));
            }
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) {
              t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, x));
              t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, x));
            }
            t0 += lv - kWeightBits;
            t1 += lv - kWeightBits;
            if (__any_sync(0xffffffffu, t0 > m[r][0] + kWeightRoom || t1 > m[r][1] + kWeightRoom)) {
              const float n0 = t0 > m[r][0] + kWeightRoom ? t0 : m[r][0];
              const float n1 = t1 > m[r][1] + kWeightRoom ? t1 : m[r][1];
              const float f0 = exp2_approx(m[r][0] - n0), f1 = exp2_approx(m[r][1] - n1);
              m[r][0] = n0;
              m[r][1] = n1;
              l[r][0] *= f0;
              l[r][1] *= f1;
#pragma unroll
              for (int j = 0; j < MT; ++j) {
                scale_pair(o[r][j][0], o[r][j][1], f0, f1);
                scale_pair(o[r][j][2], o[r][j][3], f0, f1);
              }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              float(&x)[4] = s[r][u];
              x[0] = exp2_approx(x[0] - m[r][0]);
              x[1] = exp2_approx(x[1] - m[r][1]);
              x[2] = exp2_approx(x[2] - m[r][0]);
              x[3] = exp2_approx(x[3] - m[r][1]);
              l[r][0] += x[0] + x[2];
              l[r][1] += x[1] + x[3];
              scale_pair(x[0], x[1], vsc, vsc);
              scale_pair(x[2], x[3], vsc, vsc);
              // the weights of 8 tokens x 8 rows, transposed into the B fragment of O^T = V^T P^T
              const uint32_t w0 = f16x2_of(x[0], x[1]), w1 = f16x2_of(x[2], x[3]);
              const float2 h0 = f16x2_values(w0), h1 = f16x2_values(w1);
              const uint32_t l0 = f16x2_of(x[0] - h0.x, x[1] - h0.y), l1 = f16x2_of(x[2] - h1.x, x[3] - h1.y);
              if constexpr (!TWICE) {
                pb[r][u][0] = transpose8(w0);
                pb[r][u][1] = transpose8(w1);
                pl[r][u][0] = transpose8(l0);
                pl[r][u][1] = transpose8(l1);
              } else {
                pb[r][u][0] = transpose8(t < 2 ? w0 : l0);
                pb[r][u][1] = transpose8(t < 2 ? w1 : l1);
              }
            }
          }
          // the tokens that only some rows see (fewer than q_len of them). With 16 rows before the
          // product, so that the weights' registers are free in it (92 to 144 bytes spill otherwise)
          auto some_see = [&] {
            for (int x = max(seen_by_all, slab * SL); x < min(n, slab * SL + SL); ++x) {
              const int k = x - slab * SL, from = ((k & 7) << 2) | t;
              const int page = __ldg(table + (x >> p.page_shift));
              const uint8_t* v = vbase + page * p.sp[1] + (x & (P - 1)) * p.st[1] + g * (D / 8);
  #pragma unroll
              for (int r = 0; r < NR; ++r) {
                float w0 = 0.0f, w1 = 0.0f;
  #pragma unroll
                for (int i = 0; i < 2 * U; ++i) {
                  const float e0 = __shfl_sync(0xffffffffu, s[r][i >> 1][(i & 1) * 2], from);
                  const float e1 = __shfl_sync(0xffffffffu, s[r][i >> 1][(i & 1) * 2 + 1], from);
                  if (k >> 3 == i) w0 = e0, w1 = e1;
                }
                bool sees0 = x < seen_of(r * 8 + 2 * t), sees1 = x < seen_of(r * 8 + 2 * t + 1);
                if constexpr (TWICE) sees0 = sees0 && t < 2, sees1 = sees1 && t < 2;
  #pragma unroll
                for (int j = 0; j < MT; ++j) {
  #pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    const float value = e4m3_value_hw(__ldg(v + 2 * j + e));
                    if (sees0) o[r][j][2 * e] = fmaf(w0, value, o[r][j][2 * e]);
                    if (sees1) o[r][j][2 * e + 1] = fmaf(w1, value, o[r][j][2 * e + 1]);
                  }
                }
              }
            }
          };
          if constexpr (ROWS == 16) some_see();
          // ---- O^T: row g of MMA tile j is dim g * D / 8 + 2 j, row g + 8 the next one, so a lane's
          // bytes of a token are consecutive; tokens 2 t, 2 t + 1 and 2 t + 8, 2 t + 9 of each part
          constexpr int W = D / 32;  // 4-byte words per lane and token
#pragma unroll
          for (int u = 0; u < U; ++u) {
            uint32_t r0[W], r1[W], r2[W], r3[W];
            auto take = [&](int row, uint32_t(&r)[W]) {
              if constexpr (D == 128) {
                const uint4 x = *reinterpret_cast<const uint4*>(vb + u * 16 * D + slab_offset<D>(row, g));
                r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
              } else {
                const uint2 x = *reinterpret_cast<const uint2*>(vb + u * 16 * D + slab_offset<D>(row, g >> 1) + (g & 1) * 8);
                r[0] = x.x, r[1] = x.y;
              }
            };
            take(2 * t, r0);
            take(2 * t + 1, r1);
            take(2 * t + 8, r2);
            take(2 * t + 9, r3);
#pragma unroll
            for (int w = 0; w < W; ++w) {
              const uint32_t x0 = __byte_perm(r0[w], r1[w], 0x5140), x1 = __byte_perm(r0[w], r1[w], 0x7362);
              const uint32_t y0 = __byte_perm(r2[w], r3[w], 0x5140), y1 = __byte_perm(r2[w], r3[w], 0x7362);
              const uint32_t va[4] = {e4m3x2_f16(x0), e4m3x2_f16_high(x0), e4m3x2_f16(y0), e4m3x2_f16_high(y0)};
              const uint32_t vc[4] = {e4m3x2_f16(x1), e4m3x2_f16_high(x1), e4m3x2_f16(y1), e4m3x2_f16_high(y1)};
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                float none[2][4] = {};
                float(&to0)[4] = SPLIT ? none[0] : o[r][2 * w];
                float(&to1)[4] = SPLIT ? none[1] : o[r][2 * w + 1];
                mma_f16(to0, va, pb[r][u][0], pb[r][u][1]);
                mma_f16(to1, vc, pb[r][u][0], pb[r][u][1]);
                if constexpr (!TWICE) {
                  mma_f16(to0, va, pl[r][u][0], pl[r][u][1]);
                  mma_f16(to1, vc, pl[r][u][0], pl[r][u][1]);
                }
                if constexpr (SPLIT) {  // a rounded addition for every 16 tokens
#pragma unroll
                  for (int e = 0; e < 4; e += 2) {
                    add_pair(o[r][2 * w][e], o[r][2 * w][e + 1], to0[e], to0[e + 1]);
                    add_pair(o[r][2 * w + 1][e], o[r][2 * w + 1][e + 1], to1[e], to1[e + 1]);
                  }
                }
              }
            }
          }
          if constexpr (ROWS != 16) some_see();
        }
        stage = stage == ST - 1 ? 0 : stage + 1;
      }
      copies_wait<0>();
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
          l[r][0] += __shfl_xor_sync(0xffffffffu, l[r][0], x);
          l[r][1] += __shfl_xor_sync(0xffffffffu, l[r][1], x);
        }
      }

      if constexpr (TWICE) {  // columns 4 .. 7 to 0 .. 3
#pragma unroll
        for (int j = 0; j < MT; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[0][j][e] += __shfl_xor_sync(0xffffffffu, o[0][j][e], 2);
        }
      }

      // ---- the warps' parts of this block's share of the item
      __syncthreads();  // the ring is free
#pragma unroll
      for (int r = 0; r < NR; ++r) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = r * 8 + 2 * t + e;
          if (row < rows) {
            float* at = merge_o + (warp * ROWS + row) * PITCH + g * (D / 8);
#pragma unroll
            for (int j = 0; j < MT; j += 2)
              *reinterpret_cast<float4*>(at + 2 * j) =
                  make_float4(o[r][j][e], o[r][j][2 + e], o[r][j + 1][e], o[r][j + 1][2 + e]);
            if (g == 0) {
              merge_ml[(warp * ROWS + row) * 2] = m[r][e];
              merge_ml[(warp * ROWS + row) * 2 + 1] = l[r][e];
            }
          }
        }
      }
      __syncthreads();
      const bool whole = s0 == 0 && s1 == it.slabs;
      float* my_part = a.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (it.first <= lo ? 0 : 1)) * ROWS * (D + 2);
      for (int i = tid; i < rows * (D / 4); i += NT) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float ref = kNoScore, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) ref = fmaxf(ref, merge_ml[(w * ROWS + r) * 2]);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float f = exp2_approx(merge_ml[(w * ROWS + r) * 2] - ref);
          sum = fmaf(f, merge_ml[(w * ROWS + r) * 2 + 1], sum);
          const float4 x = *reinterpret_cast<const float4*>(merge_o + (w * ROWS + r) * PITCH + d);
          acc.x = fmaf(f, x.x, acc.x);
          acc.y = fmaf(f, x.y, acc.y);
          acc.z = fmaf(f, x.z, acc.z);
          acc.w = fmaf(f, x.w, acc.w);
        }
        if (whole) {
          pages_finish<T, D>(a, it.b, it.h, it.tile * ROWS + r, d, n, acc, ref, sum);
        } else {
          __stcg(reinterpret_cast<float4*>(my_part + r * D + d), acc);
          if (d == 0) __stcg(reinterpret_cast<float2*>(my_part + ROWS * D + 2 * r), make_float2(ref, sum));
        }
      }
      if (s0 == 0) {
        // the merge goes from this block to the one that holds the item's last unit
        const PagesCut c{it.b, it.h, it.tile, static_cast<int>(blockIdx.x),
                         whole ? -1 : static_cast<int>(block_of(end - 1)), it.first <= lo ? 0 : 1};
        if (!whole) cut = c;
        if (a.cuts_by_item && tid == 0) a.cuts[(it.b * p.heads + it.h) * a.row_tiles + it.tile] = c;
      }
    }
    // ---- the next item
    it.first = end;
    if (++it.tile == a.row_tiles) {
      it.tile = 0;
      if (++it.h == p.heads) {
        it.h = 0;
        ++it.b;
      }
    }
  }
  if (tid == 0 && !a.cuts_by_item) a.cuts[blockIdx.x] = cut;
}

// The items that several blocks share: WARPS warps per row add the blocks' outputs, each with its
// weight, in an order that depends on nothing but their number. A block per item (16 warps per row:
// few items, shared by many blocks) or per block of the attention (4: many items, few shared by more
// than two) and 16 / WARPS rows.
template <int T, int D, int ROWS, int WARPS>
__global__ void __launch_bounds__(512) pages_merge_kernel(PagesAttnArgs a) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PagesCut cut = a.cuts[blockIdx.x];
  if (cut.last < 0) return;
  constexpr int LANES = D / 4, SIDES = 32 / LANES, SHARES = WARPS * SIDES;  // lanes per part, parts side by side
  constexpr int GROUPS = 16 / WARPS;
  __shared__ float4 sums[GROUPS][SHARES][LANES];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / WARPS;
  const int share = warp % WARPS * SIDES + lane / LANES;
  const int row = blockIdx.y * GROUPS + group, r = cut.tile * ROWS + row, parts = cut.last - cut.first + 1;
  const bool live = row < ROWS && r < a.rows;
  auto part_of = [&](int i) -> const float* {
    return a.partial + static_cast<int64_t>(2 * (cut.first + i) + (i == 0 ? cut.slot : 0)) * (ROWS * (D + 2));
  };
  float ref = kNoScore, sum = 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (live) {
#pragma unroll 4
    for (int i = lane; i < parts; i += 32) ref = fmaxf(ref, __ldg(part_of(i) + ROWS * D + 2 * row));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    const int d = lane % LANES * 4;
#pragma unroll 8
    for (int i = share; i < parts; i += SHARES) {
      const float* part = part_of(i);
      const float f = exp2_approx(__ldg(part + ROWS * D + 2 * row) - ref);
      const float4 x = __ldg(reinterpret_cast<const float4*>(part + row * D + d));
      acc.x = fmaf(f, x.x, acc.x);
      acc.y = fmaf(f, x.y, acc.y);
      acc.z = fmaf(f, x.z, acc.z);
      acc.w = fmaf(f, x.w, acc.w);
    }
    sums[group][share][lane % LANES] = acc;
    if (warp % WARPS == 0) {
#pragma unroll 4
      for (int i = lane; i < parts; i += 32) {
        const float2 ml = __ldg(reinterpret_cast<const float2*>(part_of(i) + ROWS * D + 2 * row));
        sum = fmaf(exp2_approx(ml.x - ref), ml.y, sum);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
  }
  __syncthreads();
  if (!live || share != 0) return;
#pragma unroll
  for (int s = 1; s < SHARES; ++s) {
    const float4 x = sums[group][s][lane];
    acc.x += x.x;
    acc.y += x.y;
    acc.z += x.z;
    acc.w += x.w;
  }
  const int n = pages_tokens(a, cut.b);
  pages_finish<T, D>(a, cut.b, cut.h, r, lane * 4, n, acc, ref, sum);
}

// The mass of every cached token: its weights, from the stored scores and the rows' final
// reference and sum, added in the order of the rows. One thread per four tokens and KV head (they
// stand in one page), one 16-byte load per row. Sequences with a common prefix may name the same page, so
// what each of them gives is added atomically: one addition per token where a page is a sequence's own.
// (Against a plain load and store: 9 x 4 x 1500 17.8 -> 19.1 us, 32 x 8192 64.8 us either way; four tokens in
// one atomic addition the same.)
__global__ void __launch_bounds__(256) pages_mass_kernel(PagesAttnArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PagePool& p = a.pool;
  const int h = blockIdx.y, b = blockIdx.z;
  const int n = pages_tokens(a, b);
  const int x = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (x >= n) return;
  const int page = __ldg(p.table + b * p.table_stride + (x >> p.page_shift));
  if (page < 0 || page >= p.num_pages) return;  // reported by the attention
  float* mass = p.mass + page * p.msp + h * p.msh + (x & ((1 << p.page_shift) - 1));
  const int64_t row0 = (static_cast<int64_t>(b) * p.heads + h) * a.rows;
  const float* s = a.scores + row0 * a.capacity + x;
  const float2* ml = reinterpret_cast<const float2*>(a.ml) + row0;
  float received[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  // of the four tokens, those that row r sees: all (past n nothing is added) but near the end of several queries
  const int first_sees = n - a.q_len + 1 - x;
  const bool some = a.causal && first_sees < 4 && a.q_len > 1;
#pragma unroll 4
  for (int r = 0; r < a.rows; ++r) {
    const float2 f = __ldg(ml + r);
    const float4 v = __ldg(reinterpret_cast<const float4*>(s + r * a.capacity));
    float w[4] = {exp2_approx(v.x - f.x) * f.y, exp2_approx(v.y - f.x) * f.y, exp2_approx(v.z - f.x) * f.y,
                  exp2_approx(v.w - f.x) * f.y};
    if (some) {  // a row gives nothing to the others, also where its sum is NaN
      const int left = first_sees + r % a.q_len;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = e < left ? w[e] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) received[e] += w[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (x + e < n) atomicAdd(mass + e, received[e]);
  }
}

}  // namespace kab
