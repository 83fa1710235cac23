// Shared by the attention kernels over a paged KV cache: the pass's index tables, the line of work that CTAs share out, and what they leave for the join.
//
// A unit of work is (request, KV head, row tile): the rows of a KV head are its request's tokens times the query heads of the group (token-major), cut
// into tiles; its keys are walked in blocks. All units' blocks in a row are one line of work that the CTAs share out evenly, whatever the lengths: a CTA
// that gets the middle of a unit leaves (maximum, sum, unnormalised output) per row in the workspace, and a second small kernel joins the pieces of a
// unit in order. Every CTA finds its own stretch from the lengths, so nothing is planned on the host and nothing read back; the shares depend on lengths
// and shapes alone, and so do the bits.
#pragma once
#include "paged.cuh"

constexpr int MAX_HEAD_COLUMNS = 8;  // head_dim <= 256: each lane owns columns lane + 32 i

struct PassIndex {       // the pass's index tables (all U32)
  const uint32_t *tables, *cached, *starts, *masks, *positions;
  int batch, words;
  int64_t tokens, width, pages;
  uint32_t page;
  int page_shift;        // log2 of the page, or -1
  int64_t window;        // 0: none
};

// What a unit that several CTAs share leaves for the joining kernel: its pieces are slot 2c + 1 of its first CTA c and slots 2(c + 1), 2(c + 2), ...
// `first` is the token of the request's row 0, `row` the tile's first row, `rows` how many it has.
struct SplitUnit { int pieces, kv_head, row, rows; uint32_t first; };
struct TileWork { float* o; float2* ml; SplitUnit* split; };   // o [2 CTAs][tile rows][D]; ml [2 CTAs][tile rows]: maximum in log2 units, sum; split [CTAs]

// Both kernels' limits: one wave of CTAs (up to three to an SM of the tiles kernel with 64 rows at most, one of the tcgen05 kernel with 256)
constexpr int MAX_SHARES = 3 * REDUCE_SMS, MAX_SHARE_ROWS = REDUCE_SMS * 256;

struct AttnDims { int64_t tokens, heads, kv_heads, dim, pages, page; };
struct AttnCall {
  ojc_backend* be; const char* op;
  const ojc_tensor *q, *k, *v; ojc_tensor* out; float* lse;
  PassIndex ix; AttnDims a; float scale; TileWork work;
};
// CTAs to launch: one wave, or fewer where the longest requests that the tables allow have no block for each
inline unsigned attn_ctas(const AttnCall& c, int wave, int tile_rows, int keys) {
  const int64_t rows = c.a.tokens * (c.a.heads / c.a.kv_heads), tiles = (rows + tile_rows - 1) / tile_rows + c.ix.batch;
  const double most = (double)tiles * (double)c.a.kv_heads * (double)(c.ix.width * c.ix.page / keys + 1);
  return most < wave ? (unsigned)most : (unsigned)wave;
}
// The joining kernel behind one that ran `shares` CTAs with tiles of `tile_rows` rows
ojc_status paged_attention_join(const AttnCall& c, unsigned shares, int tile_rows);
// tcgen05 / TMEM form with one or two tiles of 128 rows (BF16, head dims up to 128 of the tiles kernel, pages that tile 128 keys)
bool paged_attention_tcgen05_takes(const AttnCall& c);
ojc_status paged_attention_tcgen05(const AttnCall& c, int tiles);

#ifdef __CUDACC__
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) { uint32_t r; asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo)); return r; }
// A row's softmax so far is (maximum, sum). A row, or a piece of one, that saw scores of -inf alone has maximum -inf and this sum: among others it weighs
// nothing, alone it is 0 / 0. Sum 0 under -inf is a row that saw nothing, NaN one that saw NaN.
constexpr float ONLY_MINUS_INF = -1.0f;
__device__ __forceinline__ float only_minus_inf(bool any, float m, float l) { return any && m == -INFINITY && l == 0.0f ? ONLY_MINUS_INF : l; }
__device__ __forceinline__ float joined_sum(float top, float l, float c, float l2, float c2) { return top == -INFINITY ? l + l2 : l * c + l2 * c2; }
__device__ __forceinline__ float inverse_sum(float m, float l) { return m != -INFINITY ? 1.0f / l : l == 0.0f ? 0.0f : NAN; }
constexpr float LOG2_E = 1.4426950408889634f, LN_2 = 0.6931471805599453f;

// The first place that a row of the request can see (positions of new tokens are at least `cached`). Pages that lie wholly before it are never looked up:
// their entries may name no page any more.
__device__ __forceinline__ uint32_t first_place(const PassIndex& ix, uint32_t cached) { return ix.window > 0 && cached >= ix.window ? cached - (uint32_t)ix.window + 1 : 0; }

struct Request { uint32_t cached, first; int fresh, first_block, blocks, row_tiles; };
template <int KEYS>
__device__ __forceinline__ Request load_request(const PassIndex& ix, int b, int group, int tile_rows, bool* bad) {
  Request r;
  const uint32_t first = ix.starts[b], end = ix.starts[b + 1], cached = ix.cached[b];
  const bool wrong = end < first || end > ix.tokens || (int64_t)cached + (int64_t)(end - first) > ix.width * ix.page;
  *bad |= wrong;
  r.cached = wrong ? 0 : cached;
  r.first = first;
  r.fresh = wrong ? 0 : (int)(end - first);
  r.first_block = (int)(first_place(ix, r.cached) / KEYS);
  r.blocks = r.fresh == 0 ? 0 : (int)((r.cached + (uint32_t)r.fresh + KEYS - 1) / KEYS) - r.first_block;
  r.row_tiles = (int)((uint32_t)(r.fresh * group + tile_rows - 1) / (uint32_t)tile_rows);
  return r;
}

// A place on the line of work; all threads of a CTA hold the same one.
template <int KEYS>
struct Cursor {
  Request r;
  int b, hk, row_tile, block;     // block counts from 0
  __device__ __forceinline__ void step(const PassIndex& ix, int group, int tile_rows, int kv_heads, bool* bad) {
    if (++block < r.blocks) return;
    block = 0;
    if (++row_tile < r.row_tiles) return;
    row_tile = 0;
    if (++hk < kv_heads) return;
    hk = 0;
    do { if (++b >= ix.batch) return; r = load_request<KEYS>(ix, b, group, tile_rows, bad); } while (r.blocks == 0);
  }
};

// One CTA's stretch of the line: `todo` blocks from number `begin` on, the first of them at `at`. The first `longer` of the `ctas` shares have
// `share` + 1 blocks, the others `share`.
template <int KEYS>
struct Share {
  uint32_t begin, ctas, share, longer;
  int todo;
  Cursor<KEYS> at;
  __device__ __forceinline__ uint32_t begin_of(uint32_t c) const { return c * share + min(c, longer); }
  __device__ __forceinline__ uint32_t of_block(uint32_t block) const { return block < longer * (share + 1) ? block / (share + 1) : longer + (block - longer * (share + 1)) / share; }
};
struct ShareScratch { uint32_t sum[32], at; int b; Request r; };

// Called by all THREADS threads of the CTA; false: nothing for it to do. Lengths are read once for up to THREADS requests, twice beyond.
// All sums stop at MAX_LINE, where two of them still add up in 32 bits; a line that long is reported and nobody works on it: the cursor walks every
// request, so no part of a line may be left out of its numbering (units would be taken for ones with pieces beyond the last CTA's).
constexpr uint32_t MAX_LINE = 0x7fffffffu;
template <int KEYS, int THREADS>
__device__ __forceinline__ bool find_share(const PassIndex& ix, int group, int tile_rows, int kv_heads, ShareScratch* sh, Share<KEYS>* out, bool* bad) {
  constexpr int WARPS = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto blocks_of = [&](const Request& r) {
    return (uint32_t)min((unsigned long long)r.blocks * (unsigned)(r.row_tiles * kv_heads), (unsigned long long)MAX_LINE);
  };
  auto scan = [&](uint32_t n, uint32_t* upto) {                  // of a chunk of requests; the chunk's sum comes back
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const uint32_t a = __shfl_up_sync(0xffffffffu, n, o); if (lane >= o) n = min(n + a, MAX_LINE); }
    __syncthreads();
    if (lane == 31) sh->sum[warp] = n;
    __syncthreads();
    *upto = n;
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { if (w < warp) *upto = min(*upto + sh->sum[w], MAX_LINE); sum = min(sum + sh->sum[w], MAX_LINE); }
    return sum;
  };
  Request mine = {};
  uint32_t n = 0, upto = 0, total = 0;
  for (int b0 = 0; b0 < ix.batch; b0 += THREADS) {
    mine = {};
    n = 0;
    if (b0 + tid < ix.batch) { mine = load_request<KEYS>(ix, b0 + tid, group, tile_rows, bad); n = blocks_of(mine); }
    const uint32_t sum = scan(n, &upto);
    total = min(total + sum, MAX_LINE);
  }
  if (total == MAX_LINE) { *bad = true; return false; }
  out->ctas = min(gridDim.x, total);
  if (blockIdx.x >= out->ctas) return false;
  out->share = total / out->ctas;
  out->longer = total - out->share * out->ctas;
  const uint32_t begin = out->begin = out->begin_of(blockIdx.x);
  out->todo = (int)(out->begin_of(blockIdx.x + 1) - begin);
  if (ix.batch <= THREADS) {
    upto -= n;
    if (n && upto <= begin && begin - upto < n) { sh->b = tid; sh->at = upto; sh->r = mine; }
    __syncthreads();
  } else {
    uint32_t carry = 0;
    for (int b0 = 0; b0 < ix.batch; b0 += THREADS) {
      mine = {};
      n = 0;
      if (b0 + tid < ix.batch) { mine = load_request<KEYS>(ix, b0 + tid, group, tile_rows, bad); n = blocks_of(mine); }
      const uint32_t sum = scan(n, &upto);
      upto += carry - n;
      if (n && upto <= begin && begin - upto < n) { sh->b = b0 + tid; sh->at = upto; sh->r = mine; }
      __syncthreads();
      carry += sum;
      if (carry > begin) break;
    }
  }
  Cursor<KEYS>& c = out->at;
  c.b = sh->b;
  c.r = sh->r;
  const uint32_t unit = (begin - sh->at) / (uint32_t)c.r.blocks;
  c.block = (int)(begin - sh->at - unit * (uint32_t)c.r.blocks);
  c.hk = (int)(unit / (uint32_t)c.r.row_tiles);
  c.row_tile = (int)(unit - (uint32_t)c.hk * (uint32_t)c.r.row_tiles);
  return true;
}
#endif
