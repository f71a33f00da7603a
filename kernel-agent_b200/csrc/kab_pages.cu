// extern "C" entry points of the paged FP8 KV cache (kv_pages.cuh, attention_pages.cuh): the
// append, the attention over the pages and the eviction, and this translation unit's device
// status word.
#include <algorithm>
#include <type_traits>

#include "kab_host.h"

namespace kab {
__device__ unsigned g_pages_status = 0;
}  // namespace kab

#include "attention_pages.cuh"
#include "kv_pages.cuh"

namespace kab {

unsigned pages_device_status(bool clear, cudaStream_t stream) {
  unsigned v = 0;
  cudaMemcpyFromSymbolAsync(&v, g_pages_status, sizeof v, 0, cudaMemcpyDeviceToHost, stream);
  cudaStreamSynchronize(stream);
  if (clear) {
    const unsigned zero = 0;
    cudaMemcpyToSymbolAsync(g_pages_status, &zero, sizeof zero, 0, cudaMemcpyHostToDevice, stream);
  }
  return v;
}

namespace {

// The device address of the status word of the current device (looked up once per device).
unsigned* status_word() {
  static unsigned* at[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (at[dev] == nullptr) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_pages_status) != cudaSuccess) return nullptr;
    at[dev] = static_cast<unsigned*>(p);
  }
  return at[dev];
}

int pool_check(const KabKvPages* c, PagePool* p) {
  KAB_REQUIRE(c != nullptr, "null parameters");
  KAB_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "head_dim %lld: the paged cache takes 64 or 128",
              (long long)c->head_dim);
  KAB_REQUIRE(c->page_tokens == 16 || c->page_tokens == 32 || c->page_tokens == 64 || c->page_tokens == 128,
              "page_tokens %lld: 16, 32, 64 or 128", (long long)c->page_tokens);
  KAB_REQUIRE(c->batch >= 0 && c->heads_kv > 0 && c->num_pages >= 0 && c->max_pages >= 0, "bad shape");
  KAB_REQUIRE(c->batch < 65536 && c->heads_kv < 65536, "at most 65535 sequences and KV heads");
  KAB_REQUIRE(c->num_pages < (int64_t(1) << 31) && c->max_pages * c->page_tokens < (int64_t(1) << 30),
              "the page table or the pool is too large");
  if (c->batch == 0) return KAB_OK;
  KAB_REQUIRE(c->lengths != nullptr, "null lengths");
  KAB_REQUIRE(c->num_pages == 0 || (c->k_pages && c->v_pages && c->k_scale && c->v_scale), "null pages");
  KAB_REQUIRE(c->max_pages == 0 || (c->page_table != nullptr && c->num_pages > 0), "null page table or empty pool");
  KAB_REQUIRE(aligned(c->k_pages, 16) && aligned(c->v_pages, 16), "the pages must be 16-byte aligned");
  KAB_REQUIRE(c->k_stride_page % 16 == 0 && c->k_stride_head % 16 == 0 && c->k_stride_token % 16 == 0 &&
                  c->v_stride_page % 16 == 0 && c->v_stride_head % 16 == 0 && c->v_stride_token % 16 == 0,
              "page strides must be multiples of 16 bytes");
  const int64_t wide = int64_t(1) << 31;
  KAB_REQUIRE(c->k_stride_page < wide && c->v_stride_page < wide && c->ks_stride_page < wide &&
                  c->vs_stride_page < wide && c->k_stride_token * c->page_tokens < wide &&
                  c->v_stride_token * c->page_tokens < wide && c->k_stride_page >= 0 && c->v_stride_page >= 0 &&
                  c->k_stride_token >= 0 && c->v_stride_token >= 0 && c->ks_stride_page >= 0 && c->vs_stride_page >= 0,
              "page strides and a page's tokens must span less than 2^31 bytes");
  *p = PagePool{};
  p->codes[0] = c->k_pages;
  p->codes[1] = c->v_pages;
  p->scale[0] = c->k_scale;
  p->scale[1] = c->v_scale;
  p->mass = c->mass;
  p->sp[0] = c->k_stride_page, p->sh[0] = c->k_stride_head, p->st[0] = c->k_stride_token;
  p->sp[1] = c->v_stride_page, p->sh[1] = c->v_stride_head, p->st[1] = c->v_stride_token;
  p->ssp[0] = c->ks_stride_page, p->ssh[0] = c->ks_stride_head;
  p->ssp[1] = c->vs_stride_page, p->ssh[1] = c->vs_stride_head;
  p->msp = c->mass_stride_page, p->msh = c->mass_stride_head;
  p->table = c->page_table;
  p->table_stride = c->table_stride;
  p->lengths = c->lengths;
  p->num_pages = static_cast<int>(c->num_pages);
  p->heads = static_cast<int>(c->heads_kv);
  p->page_shift = c->page_tokens == 16 ? 4 : c->page_tokens == 32 ? 5 : c->page_tokens == 64 ? 6 : 7;
  p->max_pages = static_cast<int>(c->max_pages);
  p->batch = static_cast<int>(c->batch);
  return KAB_OK;
}

template <int T>
void launch_append(const AppendArgs& a, dim3 grid, int ch, unsigned* status, cudaStream_t s) {
  if (ch <= 1) append_pages_kernel<T, 1><<<grid, 256, 0, s>>>(a, status);
  else if (ch <= 2) append_pages_kernel<T, 2><<<grid, 256, 0, s>>>(a, status);
  else if (ch <= 4) append_pages_kernel<T, 4><<<grid, 256, 0, s>>>(a, status);
  else append_pages_kernel<T, 8><<<grid, 256, 0, s>>>(a, status);
}

// Query rows that share one pass over the cache.
int tile_rows(int rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : 16; }

int attention_check(const KabKvPagesAttention* p, PagesAttnArgs* g) {
  KAB_REQUIRE(p != nullptr, "null parameters");
  if (int e = pool_check(&p->cache, &g->pool)) return e;
  KAB_REQUIRE(valid_dtype(p->q_dtype), "unknown dtype %d", p->q_dtype);
  KAB_REQUIRE(p->heads_q >= 0 && p->q_len >= 0, "negative shape");
  KAB_REQUIRE(p->heads_q % p->cache.heads_kv == 0, "heads_q %lld is not a multiple of heads_kv %lld",
              (long long)p->heads_q, (long long)p->cache.heads_kv);
  KAB_REQUIRE(p->heads_q * p->q_len < (int64_t(1) << 20), "too many query rows per sequence");
  KAB_REQUIRE(!p->use_mass || p->cache.mass != nullptr || p->cache.num_pages == 0, "use_mass without a mass");
  g->qb = p->q_stride_b;
  g->qh = p->q_stride_h;
  g->qt = p->q_stride_t;
  g->scale_log2 = p->sm_scale * 1.4426950408889634f;
  g->heads_q = static_cast<int>(p->heads_q);
  g->causal = p->causal != 0;
  g->capacity = p->cache.max_pages * p->cache.page_tokens;
  return KAB_OK;
}

// What one set of launches takes of a call: sequences and query tokens.
struct AttentionPart {
  int64_t batch, queries;
};
// All of them without mass. With it the scores of every (row, token of the page table) are kept until the
// rows' sums are known: as many query tokens, or sequences with all of theirs, as keep those in 256 MB (a
// prompt of 4 x 2048 tokens and 32 heads would take 2.1 GB).
constexpr int64_t kScoresMost = int64_t(256) << 20;
AttentionPart attention_part(const KabKvPagesAttention* p) {
  const int64_t pair = p->heads_q * p->cache.max_pages * p->cache.page_tokens * 4;  // a sequence's query token
  if (!p->use_mass || pair == 0) return {p->cache.batch, p->q_len};
  const int64_t fit = std::max<int64_t>(1, kScoresMost / pair);
  if (fit >= p->q_len) return {std::min(p->cache.batch, fit / p->q_len), p->q_len};
  return {1, fit >= 16 ? fit / 16 * 16 : fit};
}
// The arguments of the part at sequence b0 and query token q0.
void attention_args(const KabKvPagesAttention* p, int64_t b0, int64_t batch, int64_t q0, int64_t queries,
                    PagesAttnArgs* g) {
  const int64_t size = p->q_dtype == KAB_F32 ? 4 : 2, group = p->heads_q / p->cache.heads_kv;
  g->pool.batch = static_cast<int>(batch);
  g->pool.table = p->cache.page_table + b0 * p->cache.table_stride;
  g->pool.lengths = p->cache.lengths + b0;
  g->q = static_cast<const uint8_t*>(p->q) + (b0 * p->q_stride_b + q0 * p->q_stride_t) * size;
  g->out = static_cast<uint8_t*>(p->out) + (b0 * p->heads_q * p->q_len + q0) * p->cache.head_dim * size;
  g->q_len = static_cast<int>(queries);
  g->tail = p->causal ? static_cast<int>(p->q_len - q0 - queries) : 0;
  g->q_skip = static_cast<int>(p->q_len - queries);
  g->out_rows = static_cast<int>(group * p->q_len);
  g->rows = static_cast<int>(group * queries);
  const int tile = tile_rows(g->rows);
  g->row_tiles = (g->rows + tile - 1) / tile;
}

// The launch's workspace: the blocks' partial results and cuts and, with mass, the scores and the
// rows' references. Nothing in it has to be zero.
struct AttentionPlan {
  int grid = 0, merges = 0;  // blocks of the attention; items, or blocks where those are fewer
  size_t cuts = 0, partial = 0, ml = 0, scores = 0;
  size_t bytes() const { return cuts + partial + ml + scores; }
};
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Opts the kernel instance into its shared memory and returns the blocks of it that fit on the
// GPU at once (asked once per device), or -1.
template <int T, int D, int ROWS, int SL>
int attention_blocks() {
  using L = PagesLayout<D, ROWS, SL, T == kF32>;
  static int blocks[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if (blocks[dev] == 0) {
    auto kern = pages_attention_kernel<T, D, ROWS, SL>;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, L::kThreads, L::kSmem) != cudaSuccess || n < 1)
      return -1;
    blocks[dev] = std::min(n, L::kBlocks) * sm_count();
  }
  return blocks[dev];
}

// The kernel instance of a call: f(type, head_dim, rows of a tile, tokens of a slab).
template <int V>
using Int = std::integral_constant<int, V>;
template <int T, int D, int SL, typename F>
auto with_rows(int rows, F&& f) {
  const int tile = tile_rows(rows);
  return tile == 4   ? f(Int<T>(), Int<D>(), Int<4>(), Int<SL>())
         : tile == 8 ? f(Int<T>(), Int<D>(), Int<8>(), Int<SL>())
                     : f(Int<T>(), Int<D>(), Int<16>(), Int<SL>());
}
template <int T, int D, typename F>
auto with_slabs(int rows, int64_t page, F&& f) {
  return page == 16 ? with_rows<T, D, 16>(rows, f) : with_rows<T, D, 32>(rows, f);
}
template <typename F>
auto with_instance(const KabKvPagesAttention* p, int rows, F&& f) {
  const int64_t d = p->cache.head_dim, page = p->cache.page_tokens;
  if (p->q_dtype == KAB_BF16) return d == 128 ? with_slabs<kBF16, 128>(rows, page, f) : with_slabs<kBF16, 64>(rows, page, f);
  if (p->q_dtype == KAB_F16) return d == 128 ? with_slabs<kF16, 128>(rows, page, f) : with_slabs<kF16, 64>(rows, page, f);
  return d == 128 ? with_slabs<kF32, 128>(rows, page, f) : with_slabs<kF32, 64>(rows, page, f);
}

int attention_plan(const KabKvPagesAttention* p, const PagesAttnArgs& g, AttentionPlan* plan) {
  plan->grid = with_instance(p, g.rows, [](auto T, auto D, auto ROWS, auto SL) {
    return attention_blocks<decltype(T)::value, decltype(D)::value, decltype(ROWS)::value, decltype(SL)::value>();
  });
  if (plan->grid < 0) return fail(KAB_ECUDA, "cannot configure the paged attention kernel");
  const size_t items = static_cast<size_t>(g.pool.batch) * g.pool.heads;
  KAB_REQUIRE(items * g.row_tiles * (static_cast<size_t>(g.capacity) / 16 + 1 + kItemCost) < (size_t(1) << 31),
              "sequences x KV heads x row tiles x tokens of the page table is too large");
  plan->merges = static_cast<int>(std::min(items * g.row_tiles, static_cast<size_t>(plan->grid)));
  plan->cuts = round256(static_cast<size_t>(plan->merges) * sizeof(PagesCut));
  plan->partial = round256(static_cast<size_t>(plan->grid) * 2 * tile_rows(g.rows) * (p->cache.head_dim + 2) * 4);
  if (p->use_mass) {
    plan->ml = round256(items * g.rows * 8);
    plan->scores = round256(items * g.rows * static_cast<size_t>(g.capacity) * 4);
  }
  return KAB_OK;
}

// A launch that may be set up while the one before it runs (it waits by itself).
template <typename... Args>
cudaError_t launch_after(void (*kern)(Args...), dim3 grid, int threads, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int T, int D, int ROWS, int SL>
int launch_attention(const PagesAttnArgs& g, const AttentionPlan& plan, unsigned* status, cudaStream_t s) {
  using L = PagesLayout<D, ROWS, SL, T == kF32>;
  pages_attention_kernel<T, D, ROWS, SL><<<plan.grid, L::kThreads, L::kSmem, s>>>(g, status);
  if (int e = check_launch("kab_kv_pages_attention")) return e;
  const int rows = std::min(g.rows, L::kRows);
  if (g.cuts_by_item)
    launch_after(pages_merge_kernel<T, D, L::kRows, 16>, dim3(plan.merges, rows), 512, s, g);
  else
    launch_after(pages_merge_kernel<T, D, L::kRows, 4>, dim3(plan.merges, (rows + 3) / 4), 512, s, g);
  if (int e = check_launch("kab_kv_pages_attention merge")) return e;
  if (g.scores == nullptr || g.capacity == 0) return KAB_OK;
  const dim3 blocks(static_cast<unsigned>((g.capacity + 1023) / 1024), g.pool.heads, g.pool.batch);
  launch_after(pages_mass_kernel, blocks, 256, s, g);
  return check_launch("kab_kv_pages_attention mass");
}

}  // namespace
}  // namespace kab

using namespace kab;

extern "C" {

int kab_kv_pages_append(const KabKvPages* cache, const void* k, const void* v, int dtype, int64_t k_stride_b,
                        int64_t k_stride_h, int64_t k_stride_t, int64_t v_stride_b, int64_t v_stride_h,
                        int64_t v_stride_t, int64_t new_tokens, const int32_t* counts, int32_t* lengths_out,
                        void* stream) {
  AppendArgs a{};
  if (int e = pool_check(cache, &a.pool)) return e;
  KAB_REQUIRE(valid_dtype(dtype), "unknown dtype %d", dtype);
  KAB_REQUIRE(new_tokens >= 0 && new_tokens < (int64_t(1) << 30), "bad number of new tokens");
  if (cache->batch == 0) return KAB_OK;
  KAB_REQUIRE(lengths_out != nullptr, "null lengths_out");
  KAB_REQUIRE(new_tokens == 0 || (k != nullptr && v != nullptr), "null pointer");
  KAB_REQUIRE(aligned(k, 16) && aligned(v, 16) && k_stride_b % 8 == 0 && k_stride_h % 8 == 0 && k_stride_t % 8 == 0 &&
                  v_stride_b % 8 == 0 && v_stride_h % 8 == 0 && v_stride_t % 8 == 0,
              "k and v must be 16-byte aligned and their strides multiples of 8 elements");
  unsigned* status = status_word();
  KAB_REQUIRE(status != nullptr, "no device status word");
  const cudaStream_t s = as_stream(stream);
  const int P = static_cast<int>(cache->page_tokens);
  a.x[0] = k, a.x[1] = v;
  a.xb[0] = k_stride_b, a.xh[0] = k_stride_h, a.xt[0] = k_stride_t;
  a.xb[1] = v_stride_b, a.xh[1] = v_stride_h, a.xt[1] = v_stride_t;
  a.counts = counts;
  const bool in_place = lengths_out == cache->lengths;
  a.lengths_out = in_place ? nullptr : lengths_out;
  a.new_tokens = static_cast<int>(new_tokens);
  // a first page with one free slot, then whole pages
  a.touched = new_tokens == 0 ? 1 : static_cast<int>((new_tokens + P - 2) / P + 1);
  a.d_shift = cache->head_dim == 64 ? 3 : 4;
  KAB_REQUIRE(cache->batch * a.touched < (int64_t(1) << 31), "too many pages");
  if (new_tokens > 0 || !in_place) {
    const int rows = static_cast<int>(std::min<int64_t>(new_tokens, P));
    const int ch = (rows * (1 << a.d_shift) + 255) / 256;
    const dim3 grid(static_cast<unsigned>(cache->batch * a.touched), static_cast<unsigned>(cache->heads_kv), 2);
    if (dtype == KAB_BF16) launch_append<kBF16>(a, grid, ch, status, s);
    else if (dtype == KAB_F16) launch_append<kF16>(a, grid, ch, status, s);
    else launch_append<kF32>(a, grid, ch, status, s);
    if (int e = check_launch("kab_kv_pages_append")) return e;
  }
  if (in_place && new_tokens > 0) {
    advance_lengths_kernel<<<(a.pool.batch + 255) / 256, 256, 0, s>>>(
        cache->lengths, counts, a.new_tokens, a.pool.max_pages << a.pool.page_shift, a.pool.batch, lengths_out);
    return check_launch("kab_kv_pages_append lengths");
  }
  return KAB_OK;
}

int kab_kv_pages_attention_workspace(const KabKvPagesAttention* params, size_t* bytes) {
  PagesAttnArgs g{};
  if (int e = attention_check(params, &g)) return e;
  KAB_REQUIRE(bytes != nullptr, "null pointer");
  *bytes = 0;
  if (params->cache.batch == 0 || params->heads_q == 0 || params->q_len == 0) return KAB_OK;
  const AttentionPart part = attention_part(params);
  for (int64_t queries : {part.queries, params->q_len % part.queries}) {  // the last query tokens may be fewer
    if (queries == 0) continue;
    AttentionPlan plan;
    attention_args(params, 0, part.batch, 0, queries, &g);
    if (int e = attention_plan(params, g, &plan)) return e;
    *bytes = std::max(*bytes, plan.bytes());
  }
  return KAB_OK;
}

int kab_kv_pages_attention(const KabKvPagesAttention* params, void* workspace, size_t workspace_bytes, void* stream) {
  PagesAttnArgs g{};
  if (int e = attention_check(params, &g)) return e;
  if (params->cache.batch == 0 || params->heads_q == 0 || params->q_len == 0) return KAB_OK;
  KAB_REQUIRE(params->q != nullptr && params->out != nullptr, "null pointer");
  KAB_REQUIRE(aligned(params->out, 16), "out must be 16-byte aligned");
  size_t need = 0;
  if (int e = kab_kv_pages_attention_workspace(params, &need)) return e;
  KAB_REQUIRE(workspace != nullptr && workspace_bytes >= need && aligned(workspace, 256),
              "the workspace needs %zu bytes, 256-byte aligned (kab_kv_pages_attention_workspace)", need);
  unsigned* status = status_word();
  KAB_REQUIRE(status != nullptr, "no device status word");
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const cudaStream_t s = as_stream(stream);
  const AttentionPart part = attention_part(params);
  for (int64_t b0 = 0; b0 < params->cache.batch; b0 += part.batch) {
    for (int64_t q0 = 0; q0 < params->q_len; q0 += part.queries) {
      attention_args(params, b0, std::min(part.batch, params->cache.batch - b0), q0,
                     std::min(part.queries, params->q_len - q0), &g);
      AttentionPlan plan;
      if (int e = attention_plan(params, g, &plan)) return e;
      g.cuts = reinterpret_cast<PagesCut*>(w);
      g.cuts_by_item = static_cast<int64_t>(g.pool.batch) * g.pool.heads * g.row_tiles <= plan.grid;
      g.partial = reinterpret_cast<float*>(w + plan.cuts);
      if (params->use_mass) {
        g.ml = reinterpret_cast<float*>(w + plan.cuts + plan.partial);
        g.scores = reinterpret_cast<float*>(w + plan.cuts + plan.partial + plan.ml);
      }
      const int e = with_instance(params, g.rows, [&](auto T, auto D, auto ROWS, auto SL) {
        return launch_attention<decltype(T)::value, decltype(D)::value, decltype(ROWS)::value, decltype(SL)::value>(
            g, plan, status, s);
      });
      if (e != KAB_OK) return e;
    }
  }
  return KAB_OK;
}

int kab_kv_pages_evict(const KabKvPages* cache, const int32_t* out_table, int64_t out_stride, int64_t budget,
                       int64_t recent, int64_t sinks, int32_t* kept, int32_t* lengths_out, void* stream) {
  EvictArgs a{};
  if (int e = pool_check(cache, &a.pool)) return e;
  KAB_REQUIRE(budget >= 1 && recent >= 0 && sinks >= 0 && sinks + recent <= budget,
              "budget %lld must be at least 1 and hold the %lld first and %lld last tokens", (long long)budget,
              (long long)sinks, (long long)recent);
  KAB_REQUIRE(budget < (int64_t(1) << 30), "the budget is too large");
  if (cache->batch == 0) return KAB_OK;
  KAB_REQUIRE(out_table && kept && lengths_out, "null pointer");
  KAB_REQUIRE(cache->mass != nullptr || cache->num_pages == 0, "an eviction needs the tokens' mass");
  KAB_REQUIRE(lengths_out != cache->lengths, "lengths_out must not be the lengths that the eviction reads");
  unsigned* status = status_word();
  KAB_REQUIRE(status != nullptr, "no device status word");
  a.out_table = out_table;
  a.out_stride = out_stride;
  a.kept = kept;
  a.lengths_out = lengths_out;
  a.budget = static_cast<int>(budget);
  a.recent = static_cast<int>(recent);
  a.sinks = static_cast<int>(sinks);
  const cudaStream_t s = as_stream(stream);
  const unsigned heads = static_cast<unsigned>(cache->heads_kv), batch = static_cast<unsigned>(cache->batch);
  // blocks of a head's cluster: 4096 tokens each (8 keys per thread) where 8 of them suffice, else 8 of
  // 16384 (32 keys)
  const int64_t capacity = cache->max_pages * cache->page_tokens;
  const int blocks = capacity <= 4096 ? 1 : capacity <= 8192 ? 2 : capacity <= 16384 ? 4 : 8;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks), heads, batch);
  cfg.blockDim = dim3(kSelectThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(blocks);
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, capacity <= 32768 ? evict_select_kernel<8> : evict_select_kernel<32>, a, blocks, status);
  if (int e = check_launch("kab_kv_pages_evict select")) return e;
  const int64_t P = cache->page_tokens;
  const int64_t pages = std::min((budget + P - 1) / P, std::max<int64_t>(cache->max_pages, 1));
  const dim3 grid(static_cast<unsigned>(pages), heads, batch);
  const int half = cache->head_dim == 64 ? 2 : 3;
  const int ch = static_cast<int>((P << half) / 128);
  if (ch <= 1) launch_after(evict_move_kernel<1>, grid, 128, s, a, half, status);
  else if (ch <= 2) launch_after(evict_move_kernel<2>, grid, 128, s, a, half, status);
  else if (ch <= 4) launch_after(evict_move_kernel<4>, grid, 128, s, a, half, status);
  else launch_after(evict_move_kernel<8>, grid, 128, s, a, half, status);
  return check_launch("kab_kv_pages_evict move");
}

}  // extern "C"
