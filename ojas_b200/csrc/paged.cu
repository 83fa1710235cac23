// Decode over a paged KV cache: the plan of a pass (block tables, slots, positions, ancestor masks), rotary positions and the cache write.
// The attention that reads the pages is paged_attn.cu.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "dispatch.cuh"
#include "paged.cuh"

namespace {

constexpr int PLAN_THREADS = 256, PLAN_MAX_BATCH = 24000;
constexpr uint32_t NO_PAGES = 0xffffffffu;   // a number of the free pages that no call has

// ======================================================================== paged_plan
// Every CTA scans the lengths for itself (the running sums stay in its shared memory: one launch, no order between CTAs) and then looks up the
// request of each of its tokens by bisection. A token's page is either entered already (places below the cached length's last page end) or
// number `first + page - held` of the free pages, so no CTA reads a table entry that another one writes; the token at a page's first place enters it.
// `held` is what the cached length needs, or (HELD) what the request has already been given: pages that drafts took and left again.
// The kernel's time is a few round trips and the first fetch of its code: the four tokens of a thread are unrolled, and checks that stood in each of
// them apart (of entries, of places that pass 32 bits) took 256 prompts from 8.5 to 10.3 us.
template <int PLAN_TOKENS, bool HELD>
__global__ void __launch_bounds__(PLAN_THREADS)
paged_plan_kernel(const uint32_t* __restrict__ cached, const uint32_t* __restrict__ fresh, const uint32_t* __restrict__ held_in, const uint32_t* __restrict__ parents,
                  const uint32_t* __restrict__ free_pages, int64_t n_free, const uint32_t* __restrict__ free_head, uint32_t page, int page_shift, int batch, int64_t width, int64_t tokens,
                  int64_t words, uint32_t* __restrict__ tables, uint32_t* __restrict__ held_out, uint32_t* __restrict__ starts, uint32_t* __restrict__ slots,
                  uint32_t* __restrict__ positions, uint32_t* __restrict__ masks, uint32_t* __restrict__ head_out, uint32_t* fault) {
  extern __shared__ uint32_t sm[];
  uint32_t* s_start = sm;                  // [batch + 1] first token of each request, clipped to the tokens there is room for
  uint32_t* s_first = sm + batch + 1;      // [batch] free pages taken by the requests before; NO_PAGES: none is for this request
  __shared__ unsigned long long w_tok[PLAN_THREADS / 32], w_pg[PLAN_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long tok_carry = 0, pg_carry = 0;
  const uint32_t head32 = *free_head;       // asked for before the lengths' scan
  bool bad = false;
  auto pages = [&](uint32_t x) { const uint32_t q = page_shift >= 0 ? x >> page_shift : x / page; return q + (x != q * page); };
  for (int b0 = 0; b0 < batch; b0 += PLAN_THREADS) {
    const int b = b0 + tid;
    unsigned long long n = 0, g = 0;
    bool passes = false;                     // its places pass 32 bits: no token of it gets a slot, and it takes no page
    if (b < batch) {
      const uint32_t c = cached[b], k = fresh[b], total = c + k;
      n = k;
      passes = total < c;
      bad |= passes;
      uint32_t held = pages(c);
      if (HELD) {
        const uint32_t h = held_in[b];
        bad |= h < held || h > width;
        held = max(held, h);
      }
      g = passes || pages(total) < held ? 0 : pages(total) - held;
    }
    unsigned long long tn = n, tg = g;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long a = __shfl_up_sync(0xffffffffu, tn, o), e = __shfl_up_sync(0xffffffffu, tg, o);
      if (lane >= o) { tn += a; tg += e; }
    }
    __syncthreads();
    if (lane == 31) { w_tok[warp] = tn; w_pg[warp] = tg; }
    __syncthreads();
    unsigned long long before_t = tok_carry, before_g = pg_carry;
    for (int w = 0; w < PLAN_THREADS / 32; ++w) {
      if (w < warp) { before_t += w_tok[w]; before_g += w_pg[w]; }
      tok_carry += w_tok[w]; pg_carry += w_pg[w];
    }
    if (b < batch) {
      s_start[b] = (uint32_t)min(before_t + tn - n, (unsigned long long)tokens);
      s_first[b] = passes ? NO_PAGES : (uint32_t)min(before_g + tg - g, (unsigned long long)NO_PAGES);
    }
  }
  if (tid == 0) s_start[batch] = (uint32_t)min(tok_carry, (unsigned long long)tokens);
  __syncthreads();
  const unsigned long long head = head32;
  if (blockIdx.x == 0) {
    for (int b = tid; b <= batch; b += PLAN_THREADS) starts[b] = s_start[b];
    if (HELD) for (int b = tid; b < batch; b += PLAN_THREADS) {       // what is entered: no further than tokens, free pages and the table reach
      const uint32_t c = cached[b], total = c + (s_start[b + 1] - s_start[b]), held = max(pages(c), held_in[b]);
      const unsigned long long gone = head + s_first[b], left = gone < (unsigned long long)n_free ? n_free - gone : 0;
      held_out[b] = max(held, (uint32_t)min((unsigned long long)(total < c ? 0u : pages(total)), min((unsigned long long)held + left, (unsigned long long)width)));
    }
    if (tid == 0) {
      *head_out = (uint32_t)min(head + pg_carry, max(head, (unsigned long long)n_free));
      if (tok_carry > (unsigned long long)tokens) raise_fault(fault, OP_PAGED_RANGE);
      if (head + pg_carry > (unsigned long long)n_free) raise_fault(fault, OP_PAGED_FULL);
    }
  }
  const uint32_t last = s_start[batch];
  for (int64_t t0 = ((int64_t)blockIdx.x * PLAN_THREADS + tid) * PLAN_TOKENS; t0 < tokens; t0 += (int64_t)gridDim.x * PLAN_THREADS * PLAN_TOKENS) {
    uint32_t slot4[PLAN_TOKENS], pos4[PLAN_TOKENS];
    int lo = 0, hi = batch - 1;            // the last request that starts at or before t0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_start[mid] <= t0) lo = mid; else hi = mid - 1;
    }
    int known = -1;                        // the request and the page that the last token looked up: its neighbours mostly share them
    uint32_t first = 0, c = 0, held = 0, known_page = 0;
    unsigned long long id = 0;
#pragma unroll
    for (int u = 0; u < PLAN_TOKENS; ++u) {
      const int64_t t = t0 + u;
      slot4[u] = OJC_NONE;
      pos4[u] = 0;
      if (t >= tokens) continue;
      if (t >= last) {
        if (masks) for (int64_t w = 0; w < words; ++w) masks[t * words + w] = 0;
        continue;
      }
      while (s_start[lo + 1] <= t) ++lo;   // stops at the latest at the request that holds `last - 1`
      const bool moved = lo != known;
      if (moved) {
        known = lo;
        first = s_start[lo];
        c = cached[lo];
        held = pages(c);
        if (HELD) held = max(held, held_in[lo]);
        if (s_first[lo] == NO_PAGES) held = 0;
      }
      const uint32_t local = (uint32_t)t - first, at = c + local;
      const uint32_t pi = page_shift >= 0 ? at >> page_shift : at / page, off = at - pi * page;
      if (moved || pi != known_page) {
        known_page = pi;
        id = 1ull << 32;                   // no page to be had
        if (pi >= width) bad = true;
        else if (pi < held) id = tables[(int64_t)lo * width + pi];
        else {
          const unsigned long long e = head + s_first[lo] + (pi - held);
          if (e < (unsigned long long)n_free) id = free_pages[e];
        }
      }
      const unsigned long long slot = id * page + off;
      if (slot < 0xffffffffull) {
        slot4[u] = (uint32_t)slot;
        if (off == 0 && pi >= held) tables[(int64_t)lo * width + pi] = (uint32_t)id;
      } else bad |= id < 1ull << 32;       // an entry that names no page, or one whose slots pass 32 bits
      // depth and ancestors: indices fall along the chain, so the mask words fill from the token's own downwards
      uint32_t depth = local;
      if (parents) {
        depth = 0;
        uint32_t cur = local, word = 0;
        int64_t at_word = local >> 5;
        if (masks) {
          for (int64_t w = words - 1; w > at_word; --w) masks[t * words + w] = 0;
          bad |= at_word >= words;
        }
        while (true) {
          if (masks) {
            while ((cur >> 5) < at_word) { if (at_word < words) masks[t * words + at_word] = word; word = 0; --at_word; }
            word |= 1u << (cur & 31);
          }
          const uint32_t up = parents[first + cur];
          if (up == OJC_NONE) break;
          if (up >= cur) { bad = true; break; }
          cur = up;
          ++depth;
        }
        if (masks) for (; at_word >= 0; --at_word) { if (at_word < words) masks[t * words + at_word] = word; word = 0; }
      } else if (masks) {
        bad |= (int64_t)(local >> 5) >= words;
        for (int64_t w = 0; w < words; ++w) masks[t * words + w] = w < (local >> 5) ? 0xffffffffu : w == (local >> 5) ? 0xffffffffu >> (31 - (local & 31)) : 0u;
      }
      pos4[u] = c + depth;
    }
    bool stored = false;
    if constexpr (PLAN_TOKENS == 4) {
      if (t0 + 4 <= tokens && ((uintptr_t)slots & 15) == 0 && ((uintptr_t)positions & 15) == 0) {
        *reinterpret_cast<uint4*>(slots + t0) = make_uint4(slot4[0], slot4[1], slot4[2], slot4[3]);
        *reinterpret_cast<uint4*>(positions + t0) = make_uint4(pos4[0], pos4[1], pos4[2], pos4[3]);
        stored = true;
      }
    }
    if (!stored) {
      for (int u = 0; u < PLAN_TOKENS && t0 + u < tokens; ++u) { slots[t0 + u] = slot4[u]; positions[t0 + u] = pos4[u]; }
    }
  }
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
}

// ======================================================================== vectors of a head
// V elements as floats, in loads and stores of at most 16 bytes
template <int V> __device__ __forceinline__ void load_v(const float* p, float (&v)[V]) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) { const float4 x = *reinterpret_cast<const float4*>(p + i); v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w; }
  } else { const float2 x = *reinterpret_cast<const float2*>(p); v[0] = x.x; v[1] = x.y; }
}
template <int V> __device__ __forceinline__ void store_v(float* p, const float (&v)[V]) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
}
template <int V> struct Words;
template <> struct Words<2> { typedef uint32_t type; };
template <> struct Words<4> { typedef uint2 type; };
template <> struct Words<8> { typedef uint4 type; };
template <int V> __device__ __forceinline__ void load_v(const bf16* p, float (&v)[V]) {
  union { typename Words<V>::type w; uint32_t u[V / 2]; } x;
  x.w = *reinterpret_cast<const typename Words<V>::type*>(p);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) { v[2 * i] = __uint_as_float(x.u[i] << 16); v[2 * i + 1] = __uint_as_float(x.u[i] & 0xffff0000u); }
}
template <int V> __device__ __forceinline__ void store_v(bf16* p, const float (&v)[V]) {
  union { typename Words<V>::type w; bf16 b[V]; } x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.b[i] = __float2bfloat16_rn(v[i]);
  *reinterpret_cast<typename Words<V>::type*>(p) = x.w;
}

// The rotation of one vector's worth of pairs: V pairs (i, i + half) in the half layout, V / 2 neighbours in the interleaved one. What passes
// through is an item of its own, moved as it is.
template <int V, bool INTER, bool F32_RESULT> struct Turn {
  static constexpr int PAIRS = INTER ? V / 2 : V;
  float c[PAIRS], s[PAIRS];
  __device__ __forceinline__ void set(const ojc_rope& rope, int first_pair, uint32_t position, float sign) {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) { rope_turn<F32_RESULT>(rope.turns[first_pair + i], position, rope.amplitude, &c[i], &s[i]); s[i] *= sign; }
  }
  __device__ __forceinline__ void apply(float (&a)[V], float (&b)[V]) const {   // a alone in the interleaved layout
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      float& u = INTER ? a[2 * i] : a[i];
      float& v = INTER ? a[2 * i + 1] : b[i];
      const float x = turned_first(u, v, c[i], s[i]);
      v = turned_second(u, v, c[i], s[i]);
      u = x;
    }
  }
};

// Rotary positions by vectors: a thread forms its pairs' sines and cosines once and goes through `step` heads with them, HEADS at a time so that their
// loads are in flight together (two: 113 us for 32768 x 40 x 128 BF16, 5.9 TB/s; one 129 us, four 146 us with half the warps to an SM).
// Bound by HBM: every element once in and once out.
template <class T, int V, bool INTER>
__global__ void __launch_bounds__(256)
rope_vector_kernel(const __grid_constant__ ojc_rope rope, const T* x, T* y, const uint32_t* __restrict__ positions, uint32_t rows, uint32_t time, uint32_t pos_rows, int heads, int step,
                   int dim, int64_t xb, int64_t xt, int64_t xh, int64_t yb, int64_t yt, int64_t yh, float sign) {
  constexpr int HEADS = 2;
  const uint32_t half = rope.rotary_dim / 2, turned = (INTER ? rope.rotary_dim : half) / V, items = turned + (dim - rope.rotary_dim) / V;
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, row = at / items, item = at % items;
  if (row >= rows) return;
  const int h0 = blockIdx.y * step, h1 = min(heads, h0 + step);
  const uint32_t b = row / time, t = row - b * time;
  const bool turns = item < turned;
  const int e = turns ? (int)(item * V) : (int)(rope.rotary_dim + (item - turned) * V);
  x += b * xb + t * xt + e;
  y += b * yb + t * yt + e;
  Turn<V, INTER, std::is_same<T, float>::value> turn;
  if (turns) turn.set(rope, INTER ? e / 2 : e, positions[pos_rows == rows ? row : t], sign);
  for (int h = h0; h < h1; h += HEADS) {
    float u[HEADS][V], v[HEADS][V];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) if (h + i < h1) {
      load_v<V>(x + (h + i) * xh, u[i]);
      if (turns && !INTER) load_v<V>(x + (h + i) * xh + half, v[i]);
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) if (h + i < h1) {
      if (turns) turn.apply(u[i], v[i]);
      store_v<V>(y + (h + i) * yh, u[i]);
      if (turns && !INTER) store_v<V>(y + (h + i) * yh + half, v[i]);
    }
  }
}

// The cache write by vectors: the same items, a rotated key vector (or pair of vectors) with the value's at the same place. Bound by HBM: 16384 tokens x
// 16 x 128 from F32 into BF16 pages 68 us, 5.9 TB/s.
template <class S, class D, int V, bool INTER>
__global__ void __launch_bounds__(256)
paged_kv_write_vector_kernel(const __grid_constant__ ojc_rope rope, PagesView<D> kp, PagesView<D> vp, RowsView<const S> k, RowsView<const S> v, const uint32_t* __restrict__ slots,
                             const uint32_t* __restrict__ positions, uint32_t tokens, int heads, int step, int dim, uint32_t page, uint32_t n_slots, uint32_t* fault) {
  constexpr int HEADS = 2;
  const uint32_t half = rope.rotary_dim / 2, turned = (INTER ? rope.rotary_dim : half) / V, items = turned + (dim - rope.rotary_dim) / V;
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, t = at / items, item = at % items;
  if (t >= tokens) return;
  const uint32_t slot = slots[t];
  if (slot == OJC_NONE) return;
  if (slot >= n_slots) { if (item == 0) raise_fault(fault, OP_PAGED_RANGE); return; }
  const uint32_t pg = slot / page, off = slot - pg * page;
  const int h0 = blockIdx.y * step, h1 = min(heads, h0 + step);
  const bool turns = item < turned;
  const int e = turns ? (int)(item * V) : (int)(rope.rotary_dim + (item - turned) * V);
  const S *sk = k.ptr + t * k.sn + e, *sv = v.ptr + t * v.sn + e;
  D *dk = kp.ptr + pg * kp.sp + off * kp.st + e, *dv = vp.ptr + pg * vp.sp + off * vp.st + e;
  Turn<V, INTER, std::is_same<D, float>::value> turn;
  if (turns) turn.set(rope, INTER ? e / 2 : e, positions[t], 1.0f);
  for (int h = h0; h < h1; h += HEADS) {
    float a[HEADS][V], b[HEADS][V], c[HEADS][V], d[HEADS][V];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) if (h + i < h1) {
      load_v<V>(sk + (h + i) * k.sh, a[i]);
      load_v<V>(sv + (h + i) * v.sh, c[i]);
      if (turns && !INTER) { load_v<V>(sk + (h + i) * k.sh + half, b[i]); load_v<V>(sv + (h + i) * v.sh + half, d[i]); }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) if (h + i < h1) {
      if (turns) turn.apply(a[i], b[i]);
      store_v<V>(dk + (h + i) * kp.sh, a[i]);
      store_v<V>(dv + (h + i) * vp.sh, c[i]);
      if (turns && !INTER) { store_v<V>(dk + (h + i) * kp.sh + half, b[i]); store_v<V>(dv + (h + i) * vp.sh + half, d[i]); }
    }
  }
}

// The widest vector (8, 4 or 2 elements, at most 16 bytes of the narrower type's) that the rotated part's pieces, the rest and every row start allow; 0: none
int vector_of(int layout, int rotary, int64_t dim, std::initializer_list<std::pair<const ojc_tensor*, int>> tensors) {
  for (int v = 8; v >= 2; v /= 2) {
    bool fits = dim % v == 0 && (layout ? rotary : rotary / 2) % v == 0;
    for (auto& [t, axes] : tensors) {
      const int64_t size = (int64_t)dtype_size(t->dtype), bytes = std::min<int64_t>(16, v * size);
      fits = fits && (uintptr_t)t->data % bytes == 0;
      for (int i = 0; i < axes; ++i) fits = fits && t->stride[i] * size % bytes == 0;
    }
    if (fits) return v;
  }
  return 0;
}

// How many heads a thread goes through: with as many threads as the GPU holds at once each has its share of the work, sines and cosines formed once for
// it. (Twice or four times as many threads: rope 115 against 113 us, write 70 and 78 against 68.)
int heads_per_thread(const ojc_backend* be, int64_t items, int64_t heads) {
  const int64_t most = std::max<int64_t>(1, std::min(heads, items * heads / ((int64_t)be->sm_count * 2048))), groups = (heads + most - 1) / most;
  return (int)((heads + groups - 1) / groups);
}

template <class F> ojc_status by_vector(int v, int layout, F&& f) {
  auto with = [&](auto n) { return layout ? f(n, std::true_type()) : f(n, std::false_type()); };
  if (v == 8) return with(std::integral_constant<int, 8>());
  if (v == 4) return with(std::integral_constant<int, 4>());
  return with(std::integral_constant<int, 2>());
}

// ======================================================================== rotary positions
// Any alignment: one thread per pair of a (token, head), and one per element behind the rotated part.
template <class T>
__global__ void rope_kernel(const __grid_constant__ ojc_rope rope, const T* x, T* y, const uint32_t* __restrict__ positions, int64_t rows, int64_t time,
                            int64_t pos_rows, int heads, int dim, int64_t xb, int64_t xt, int64_t xh, int64_t yb, int64_t yt, int64_t yh, float sign) {
  const int half = rope.rotary_dim / 2, items = half + dim - rope.rotary_dim;
  const int64_t total = rows * heads * items;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int e = (int)(i % items), h = (int)(i / items % heads);
    const int64_t row = i / items / heads, b = row / time, t = row % time;
    const T* px = x + b * xb + t * xt + h * xh;
    T* py = y + b * yb + t * yt + h * yh;
    if (e >= half) { py[rope.rotary_dim + e - half] = px[rope.rotary_dim + e - half]; continue; }
    float c, s;
    rope_turn<std::is_same<T, float>::value>(rope.turns[e], positions[row % pos_rows], rope.amplitude, &c, &s);
    s *= sign;
    const int i0 = rope.layout ? 2 * e : e, i1 = rope.layout ? 2 * e + 1 : e + half;
    const float u = ldf(px, i0), v = ldf(px, i1);
    stf(py, i0, turned_first(u, v, c, s));
    stf(py, i1, turned_second(u, v, c, s));
  }
}

// ======================================================================== paged_kv_write
template <class S, class D>
__global__ void paged_kv_write_kernel(const __grid_constant__ ojc_rope rope, bool rotate, PagesView<D> kp, PagesView<D> vp, RowsView<const S> k, RowsView<const S> v,
                                      const uint32_t* __restrict__ slots, const uint32_t* __restrict__ positions, int64_t tokens, int heads, int dim, uint32_t page,
                                      int64_t n_slots, uint32_t* fault) {
  const int64_t total = tokens * heads * dim;
  bool bad = false;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int e = (int)(i % dim), h = (int)(i / dim % heads);
    const int64_t t = i / dim / heads;
    const uint32_t slot = slots[t];
    if (slot == OJC_NONE) continue;
    if (slot >= n_slots) { bad = true; continue; }
    const uint32_t pg = slot / page, off = slot - pg * page;
    const S* pk = k.ptr + t * k.sn + h * k.sh;
    float a = ldf(pk, e);
    if (rotate && e < rope.rotary_dim) {
      const int half = rope.rotary_dim / 2;
      const int pair = rope.layout ? e / 2 : e % half;
      const bool second = rope.layout ? (e & 1) : e >= half;
      const float other = ldf(pk, rope.layout ? e ^ 1 : second ? e - half : e + half);
      float c, s;
      rope_turn<std::is_same<D, float>::value>(rope.turns[pair], positions[t], rope.amplitude, &c, &s);
      a = second ? turned_second(other, a, c, s) : turned_first(a, other, c, s);
    }
    stf(kp.ptr + pg * kp.sp + off * kp.st + h * kp.sh, e, a);
    stf(vp.ptr + pg * vp.sp + off * vp.st + h * vp.sh, e, ldf(v.ptr + t * v.sn + h * v.sh, e));
  }
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
}

ojc_status u32_vector(const char* op, const char* what, const ojc_tensor* t, int64_t n) {
  OJC_TRY(check_tensor(op, what, t));
  if (t->dtype != OJC_U32) return ojc_fail(OJC_ERR_DTYPE, op, std::string(what) + " is U32");
  if (t->rank != 1 || (n >= 0 && t->shape[0] != n)) return ojc_fail(OJC_ERR_SHAPE, op, std::string(what) + " has the wrong shape");
  return OJC_OK;
}

ojc_status rope_run(ojc_backend* be, const char* op, const ojc_rope* rope, const ojc_tensor* x, const ojc_tensor* positions, ojc_tensor* y, float sign) {
  OJC_ALIVE(be, op);
  OJC_TRY(check_tensor(op, "x", x, false)); OJC_TRY(check_tensor(op, "y", y, false)); OJC_TRY(check_tensor(op, "positions", positions));
  if ((x->rank != 3 && x->rank != 4) || !same_shape(x, y)) return ojc_fail(OJC_ERR_SHAPE, op, "x, y [N, H, D] or [B, T, H, D]");
  if (x->dtype != y->dtype || !is_float(x)) return ojc_fail(OJC_ERR_DTYPE, op, "x, y share F32 or BF16");
  OJC_TRY(own_places(op, "y", y));
  if (positions->dtype != OJC_U32) return ojc_fail(OJC_ERR_DTYPE, op, "positions are U32");
  if (numel(x) == 0) return ojc_fail(OJC_ERR_SHAPE, op, "empty tensor");
  const int r = x->rank;
  const int64_t batch = r == 4 ? x->shape[0] : 1, time = x->shape[r - 3], heads = x->shape[r - 2], dim = x->shape[r - 1], rows = batch * time;
  if (x->stride[r - 1] != 1 || y->stride[r - 1] != 1) return ojc_fail(OJC_ERR_SHAPE, op, "the head_dim axis must be contiguous");
  if (heads > INT32_MAX || dim > INT32_MAX) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "extent out of range");
  OJC_TRY(rope_check(op, rope, dim));
  const int64_t np = numel(positions);
  if (np != rows && !(r == 4 && np == time)) return ojc_fail(OJC_ERR_SHAPE, op, "positions hold one entry per token, or per time step of a rank-4 tensor");
  OJC_CUDA(be, cudaSetDevice(be->device), op);   // the caller's current device may be another backend's
  const int64_t xb = r == 4 ? x->stride[0] : 0, yb = r == 4 ? y->stride[0] : 0;
  return dispatch_float(op, x->dtype, [&](auto t) {
    using T = decltype(t);
    const int v = vector_of(rope->layout, rope->rotary_dim, dim, {{x, r - 1}, {y, r - 1}});
    if (v && rows * dim < INT32_MAX) {
      const int64_t per_row = ((rope->layout ? rope->rotary_dim : rope->rotary_dim / 2) + dim - rope->rotary_dim) / v, step = heads_per_thread(be, rows * per_row, heads);
      const dim3 grid((unsigned)((rows * per_row + 255) / 256), (unsigned)((heads + step - 1) / step));
      if (grid.y <= 65535) return by_vector(v, rope->layout, [&](auto n, auto inter) {
        rope_vector_kernel<T, decltype(n)::value, decltype(inter)::value><<<grid, 256, 0, be->stream>>>(
            *rope, (const T*)x->data, (T*)y->data, (const uint32_t*)positions->data, (uint32_t)rows, (uint32_t)time, (uint32_t)np, (int)heads, (int)step, (int)dim, xb,
            x->stride[r - 3], x->stride[r - 2], yb, y->stride[r - 3], y->stride[r - 2], sign);
        OJC_LAUNCHED(be, op);
        return OJC_OK;
      });
    }
    const int64_t items = rows * heads * (dim - rope->rotary_dim / 2);
    rope_kernel<T><<<elementwise_grid(be, items, 256), 256, 0, be->stream>>>(*rope, (const T*)x->data, (T*)y->data, (const uint32_t*)positions->data, rows, time, np, (int)heads,
                                                                             (int)dim, xb, x->stride[r - 3], x->stride[r - 2], yb, y->stride[r - 3], y->stride[r - 2], sign);
    OJC_LAUNCHED(be, op);
    return OJC_OK;
  });
}

ojc_status plan_run(ojc_backend* be, const char* op, const ojc_tensor* cached_lens, const ojc_tensor* new_lens, const ojc_tensor* held_pages, const ojc_tensor* parents,
                    const ojc_tensor* free_pages, const ojc_tensor* free_head, int64_t page_size, ojc_tensor* block_tables, ojc_tensor* held_pages_out, ojc_tensor* starts, ojc_tensor* slots,
                    ojc_tensor* positions, ojc_tensor* masks, ojc_tensor* free_head_out) {
  OJC_ALIVE(be, op);
  OJC_TRY(u32_vector(op, "cached_lens", cached_lens, -1));
  const int64_t batch = cached_lens->shape[0];
  OJC_TRY(u32_vector(op, "new_lens", new_lens, batch));
  if (held_pages) OJC_TRY(u32_vector(op, "held_pages", held_pages, batch));
  OJC_TRY(u32_vector(op, "free_pages", free_pages, -1)); OJC_TRY(u32_vector(op, "free_head", free_head, 1));
  OJC_TRY(u32_vector(op, "starts", starts, batch + 1)); OJC_TRY(u32_vector(op, "slots", slots, -1));
  const int64_t tokens = slots->shape[0];
  OJC_TRY(u32_vector(op, "positions", positions, tokens)); OJC_TRY(u32_vector(op, "free_head_out", free_head_out, 1));
  OJC_TRY(check_tensor(op, "block_tables", block_tables));
  if (block_tables->dtype != OJC_U32) return ojc_fail(OJC_ERR_DTYPE, op, "block_tables is U32");
  if (block_tables->rank != 2 || block_tables->shape[0] != batch) return ojc_fail(OJC_ERR_SHAPE, op, "block_tables is [B, W]");
  if (parents) OJC_TRY(u32_vector(op, "parents", parents, tokens));
  int64_t words = 0;
  if (masks) {
    OJC_TRY(check_tensor(op, "masks", masks));
    if (masks->dtype != OJC_U32) return ojc_fail(OJC_ERR_DTYPE, op, "masks is U32");
    if (masks->rank != 2 || masks->shape[0] != tokens || masks->shape[1] == 0) return ojc_fail(OJC_ERR_SHAPE, op, "masks is [N, words]");
    words = masks->shape[1];
  }
  const int64_t width = block_tables->shape[1];
  if (batch == 0 || tokens == 0 || width == 0) return ojc_fail(OJC_ERR_SHAPE, op, "every dimension must be non-zero");
  if (batch > PLAN_MAX_BATCH) return ojc_fail(OJC_ERR_UNSUPPORTED, op, "more than 24,000 requests are not supported");
  if (tokens > INT32_MAX || width > INT32_MAX) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "extent out of range");
  if (page_size < 1 || page_size > (1 << 24)) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "page_size must be in 1..=2^24");
  if (free_head_out->data == free_head->data) return ojc_fail(OJC_ERR_SHAPE, op, "free_head_out must be another tensor than free_head");
  OJC_CUDA(be, cudaSetDevice(be->device), op);
  const size_t smem = (size_t)(2 * batch + 1) * 4;
  // a token to a thread while that gives every SM a few CTAs at most (trees' chains of parents then run side by side), else four and 16-byte stores
  const int per_thread = tokens <= (int64_t)be->sm_count * PLAN_THREADS * 4 ? 1 : 4;
  const int64_t per_cta = PLAN_THREADS * per_thread;
  const unsigned grid = (unsigned)std::min<int64_t>((tokens + per_cta - 1) / per_cta, (int64_t)be->sm_count * 4);
  auto* const kernel = held_pages ? (per_thread == 1 ? paged_plan_kernel<1, true> : paged_plan_kernel<4, true>) : per_thread == 1 ? paged_plan_kernel<1, false> : paged_plan_kernel<4, false>;
  static PerDeviceFlag attr;
  if (smem > 48 * 1024 - 256 && !attr[be->device]) {
    for (auto* k : {paged_plan_kernel<1, false>, paged_plan_kernel<4, false>, paged_plan_kernel<1, true>, paged_plan_kernel<4, true>})
      OJC_CUDA(be, cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 * PLAN_MAX_BATCH + 1) * 4), op);
    attr[be->device] = true;
  }
  kernel<<<grid, PLAN_THREADS, smem, be->stream>>>(
      (const uint32_t*)cached_lens->data, (const uint32_t*)new_lens->data, held_pages ? (const uint32_t*)held_pages->data : nullptr, parents ? (const uint32_t*)parents->data : nullptr,
      (const uint32_t*)free_pages->data, free_pages->shape[0], (const uint32_t*)free_head->data, (uint32_t)page_size,
      (page_size & (page_size - 1)) ? -1 : __builtin_ctzll((unsigned long long)page_size), (int)batch, width, tokens, words, (uint32_t*)block_tables->data,
      held_pages_out ? (uint32_t*)held_pages_out->data : nullptr, (uint32_t*)starts->data, (uint32_t*)slots->data, (uint32_t*)positions->data, masks ? (uint32_t*)masks->data : nullptr,
      (uint32_t*)free_head_out->data, be->fault_dev);
  OJC_LAUNCHED(be, op);
  return OJC_OK;
}

}  // namespace

ojc_status rope_check(const char* op, const ojc_rope* rope, int64_t head_dim) {
  if (!rope) return ojc_fail(OJC_ERR_BACKEND, op, "null rope plan");
  if (rope->rotary_dim < 2 || rope->rotary_dim % 2 || rope->rotary_dim > 2 * OJC_ROPE_MAX_PAIRS || (rope->layout != 0 && rope->layout != 1))
    return ojc_fail(OJC_ERR_BACKEND, op, "the rope plan was not made by ojc_rope_plan");
  if (rope->rotary_dim > head_dim) return ojc_fail(OJC_ERR_SHAPE, op, "the rotary dimension exceeds the head dimension");
  return OJC_OK;
}

extern "C" {

ojc_status ojc_rope_plan(const ojc_rope_spec* spec, ojc_rope* rope) {
  const char* op = "rope_plan";
  if (!spec || !rope) return ojc_fail(OJC_ERR_BACKEND, op, "null pointer");
  const ojc_rope_spec& s = *spec;
  if (s.rotary_dim < 2 || s.rotary_dim % 2) return ojc_fail(OJC_ERR_SHAPE, op, "rotary_dim must be even and at least 2");
  if (s.rotary_dim > 2 * OJC_ROPE_MAX_PAIRS) return ojc_fail(OJC_ERR_UNSUPPORTED, op, "rotary_dim above 256");
  if (s.layout != 0 && s.layout != 1) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "layout is 0 (half) or 1 (interleaved)");
  if (s.scaling < 0 || s.scaling > 3) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "scaling is 0 (none), 1 (linear), 2 (base) or 3 (by turns)");
  if (!(s.base >= 1.0) || !std::isfinite(s.base)) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "base must be finite and at least 1");
  if (!std::isfinite((float)s.amplitude)) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "amplitude must be finite in F32");   // as the plan holds it
  if (s.scaling && (!(s.factor >= 1.0) || !std::isfinite(s.factor))) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "factor must be finite and at least 1");
  if (s.scaling == 2 && s.rotary_dim == 2) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "base scaling needs more than one pair");
  if (s.scaling == 3 && (!(s.original_length > 0.0) || !std::isfinite(s.original_length) || !std::isfinite(s.low_turns) || !std::isfinite(s.high_turns) || !(s.high_turns > s.low_turns)))
    return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "by-turns scaling needs original_length > 0 and low_turns < high_turns");
  const long double two_pi = 6.283185307179586476925286766559005768L, R = s.rotary_dim;
  long double base = s.base;
  if (s.scaling == 2) base *= powl((long double)s.factor, R / (R - 2.0L));
  *rope = ojc_rope{};
  rope->rotary_dim = s.rotary_dim;
  rope->layout = s.layout;
  rope->amplitude = (float)s.amplitude;
  for (int i = 0; i < s.rotary_dim / 2; ++i) {
    long double f = powl(base, -2.0L * i / R);
    if (s.scaling == 1) f /= s.factor;
    if (s.scaling == 3) {
      long double w = (s.original_length * f / two_pi - s.low_turns) / ((long double)s.high_turns - s.low_turns);
      w = w < 0.0L ? 0.0L : w > 1.0L ? 1.0L : w;
      f *= w + (1.0L - w) / s.factor;
    }
    rope->turns[i] = (uint64_t)(f / two_pi * 18446744073709551616.0L + 0.5L);   // f <= 1 radian: below 2^62
  }
  return OJC_OK;
}

ojc_status ojc_rope_forward(ojc_backend* be, const ojc_rope* rope, const ojc_tensor* x, const ojc_tensor* positions, ojc_tensor* y) {
  return rope_run(be, "rope_forward", rope, x, positions, y, 1.0f);
}
ojc_status ojc_rope_backward(ojc_backend* be, const ojc_rope* rope, const ojc_tensor* grad_y, const ojc_tensor* positions, ojc_tensor* grad_x) {
  return rope_run(be, "rope_backward", rope, grad_y, positions, grad_x, -1.0f);
}

ojc_status ojc_paged_plan(ojc_backend* be, const ojc_tensor* cached_lens, const ojc_tensor* new_lens, const ojc_tensor* parents, const ojc_tensor* free_pages, const ojc_tensor* free_head,
                          int64_t page_size, ojc_tensor* block_tables, ojc_tensor* starts, ojc_tensor* slots, ojc_tensor* positions, ojc_tensor* masks, ojc_tensor* free_head_out) {
  return plan_run(be, "paged_plan", cached_lens, new_lens, nullptr, parents, free_pages, free_head, page_size, block_tables, nullptr, starts, slots, positions, masks, free_head_out);
}
ojc_status ojc_paged_plan_held(ojc_backend* be, const ojc_tensor* cached_lens, const ojc_tensor* new_lens, const ojc_tensor* held_pages, const ojc_tensor* parents,
                               const ojc_tensor* free_pages, const ojc_tensor* free_head, int64_t page_size, ojc_tensor* block_tables, ojc_tensor* held_pages_out, ojc_tensor* starts,
                               ojc_tensor* slots, ojc_tensor* positions, ojc_tensor* masks, ojc_tensor* free_head_out) {
  const char* op = "paged_plan_held";
  OJC_ALIVE(be, op);
  OJC_TRY(u32_vector(op, "held_pages", held_pages, -1)); OJC_TRY(u32_vector(op, "held_pages_out", held_pages_out, held_pages->shape[0]));
  if (held_pages_out->data == held_pages->data) return ojc_fail(OJC_ERR_SHAPE, op, "held_pages_out must be another tensor than held_pages");
  return plan_run(be, op, cached_lens, new_lens, held_pages, parents, free_pages, free_head, page_size, block_tables, held_pages_out, starts, slots, positions, masks, free_head_out);
}

ojc_status ojc_paged_kv_write(ojc_backend* be, ojc_tensor* k_pages, ojc_tensor* v_pages, const ojc_tensor* k, const ojc_tensor* v, const ojc_tensor* slots, const ojc_rope* rope,
                              const ojc_tensor* positions) {
  const char* op = "paged_kv_write";
  OJC_ALIVE(be, op);
  OJC_TRY(check_tensor(op, "k_pages", k_pages, false)); OJC_TRY(check_tensor(op, "v_pages", v_pages, false));
  OJC_TRY(check_tensor(op, "k", k, false)); OJC_TRY(check_tensor(op, "v", v, false));
  if (k_pages->rank != 4 || !same_shape(k_pages, v_pages)) return ojc_fail(OJC_ERR_SHAPE, op, "k_pages, v_pages [P, page, Hkv, D]");
  if (k->rank != 3 || !same_shape(k, v) || k->shape[1] != k_pages->shape[2] || k->shape[2] != k_pages->shape[3]) return ojc_fail(OJC_ERR_SHAPE, op, "k, v [N, Hkv, D]");
  if (k_pages->dtype != v_pages->dtype || k->dtype != v->dtype || !is_float(k_pages) || !is_float(k)) return ojc_fail(OJC_ERR_DTYPE, op, "k and v, and the pages, share F32 or BF16");
  if (numel(k) == 0 || numel(k_pages) == 0) return ojc_fail(OJC_ERR_SHAPE, op, "empty tensor");
  OJC_TRY(own_places(op, "k_pages", k_pages)); OJC_TRY(own_places(op, "v_pages", v_pages));
  if (k->stride[2] != 1 || v->stride[2] != 1 || k_pages->stride[3] != 1 || v_pages->stride[3] != 1) return ojc_fail(OJC_ERR_SHAPE, op, "the head_dim axis must be contiguous");
  const int64_t tokens = k->shape[0], heads = k->shape[1], dim = k->shape[2], page = k_pages->shape[1], pages = k_pages->shape[0];
  if (page > (1 << 24) || heads > INT32_MAX || dim > INT32_MAX || pages > (int64_t)OJC_NONE / page) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "slot numbers do not fit U32");
  OJC_TRY(u32_vector(op, "slots", slots, tokens));
  if (rope) { OJC_TRY(rope_check(op, rope, dim)); OJC_TRY(u32_vector(op, "positions", positions, tokens)); }
  OJC_CUDA(be, cudaSetDevice(be->device), op);
  return dispatch_float(op, k->dtype, [&](auto s) {
    using S = decltype(s);
    return dispatch_float(op, k_pages->dtype, [&](auto d) {
      using D = decltype(d);
      ojc_rope turn = rope ? *rope : ojc_rope{};
      const int vec = vector_of(turn.layout, turn.rotary_dim, dim, {{k_pages, 3}, {v_pages, 3}, {k, 2}, {v, 2}});
      if (vec && tokens * dim < INT32_MAX) {
        const int64_t per_row = ((turn.layout ? turn.rotary_dim : turn.rotary_dim / 2) + dim - turn.rotary_dim) / vec, step = heads_per_thread(be, tokens * per_row, heads);
        const dim3 grid((unsigned)((tokens * per_row + 255) / 256), (unsigned)((heads + step - 1) / step));
        if (grid.y <= 65535) return by_vector(vec, turn.layout, [&](auto n, auto inter) {
          paged_kv_write_vector_kernel<S, D, decltype(n)::value, decltype(inter)::value><<<grid, 256, 0, be->stream>>>(
              turn, pages_view<D>(k_pages), pages_view<D>(v_pages), rows_view<const S>(k), rows_view<const S>(v), (const uint32_t*)slots->data,
              rope ? (const uint32_t*)positions->data : nullptr, (uint32_t)tokens, (int)heads, (int)step, (int)dim, (uint32_t)page, (uint32_t)(pages * page), be->fault_dev);
          OJC_LAUNCHED(be, op);
          return OJC_OK;
        });
      }
      paged_kv_write_kernel<S, D><<<elementwise_grid(be, numel(k), 256), 256, 0, be->stream>>>(
          turn, rope != nullptr, pages_view<D>(k_pages), pages_view<D>(v_pages), rows_view<const S>(k), rows_view<const S>(v), (const uint32_t*)slots->data,
          rope ? (const uint32_t*)positions->data : nullptr, tokens, (int)heads, (int)dim, (uint32_t)page, pages * page, be->fault_dev);
      OJC_LAUNCHED(be, op);
      return OJC_OK;
    });
  });
}

}  // extern "C"
