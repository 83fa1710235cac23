// Attention of new tokens (one decoded token, a tree of drafts, a piece of a prompt) over a paged KV cache.
//
// out_i = sum_j p_ij v_j, p_ij = exp(s_ij - max_j s_ij) / sum, s_ij = q_i . k_j / sqrt(D) over the places j that row i sees: the cached ones inside
// its window, and of its request's new tokens those in its ancestor mask (or up to itself). One pass over the keys with a running maximum and sum.
#include <algorithm>
#include <type_traits>

#include "dispatch.cuh"
#include "paged_attn.cuh"

namespace {

// the last request that starts at or before token t (requests without tokens share their start with the next one)
__device__ __forceinline__ int request_of(const uint32_t* starts, int batch, uint32_t t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// One warp per (token, head), lanes across keys, f32 sums: any head_dim up to 256, any page size, strides and alignment.
template <class T>
__global__ void __launch_bounds__(128)
paged_attention_rows_kernel(RowsView<const T> q, PagesView<const T> kp, PagesView<const T> vp, PassIndex ix, RowsView<T> out, float* __restrict__ lse, int heads, int group,
                            int dim, float scale, uint32_t* fault) {
  extern __shared__ float sm[];  // [warps][dim] query rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * nwarps + warp, t = row / heads;
  const int h = (int)(row % heads), hk = h / group;
  if (t >= ix.tokens || t >= ix.starts[ix.batch] || t < ix.starts[0]) return;
  const int b = request_of(ix.starts, ix.batch, (uint32_t)t);
  const uint32_t first = ix.starts[b], end = ix.starts[b + 1], local = (uint32_t)t - first;
  const int64_t cached = ix.cached[b], room = ix.width * ix.page;
  bool bad = first > t || end <= t || end > ix.tokens || cached + (end - first) > room;
  const int64_t fresh = bad ? 0 : end - first, total = bad ? 0 : cached + fresh;
  const int64_t place = ix.positions ? ix.positions[t] : cached + local;
  const int64_t low = ix.window > 0 ? place - ix.window : -1;   // keys at positions above `low` are in the window
  bad |= ix.window > 0 && place < cached;
  float* qs = sm + warp * dim;
  const T* qp = q.ptr + t * q.sn + h * q.sh;
  for (int d = lane; d < dim; d += 32) qs[d] = ldf(qp, d);
  __syncwarp();
  float m = -INFINITY, l = 0.0f, o[MAX_HEAD_COLUMNS];
  bool any = false;
#pragma unroll
  for (int i = 0; i < MAX_HEAD_COLUMNS; ++i) o[i] = 0.0f;
  for (int64_t j0 = min(low < 0 ? 0 : low + 1, cached); j0 < total; j0 += 32) {
    const int64_t j = j0 + lane;
    bool sees = j < total;
    if (sees) {
      if (j < cached) sees = j > low;
      else {
        const uint32_t n = (uint32_t)(j - cached);
        sees = ix.masks ? (n >> 5) < (uint32_t)ix.words && (ix.masks[t * ix.words + (n >> 5)] >> (n & 31) & 1u) : n <= local;
        if (sees && ix.window > 0) sees = (ix.positions ? (int64_t)ix.positions[first + n] : cached + n) > low;
      }
    }
    int64_t at = 0;        // the key's offset without the head's
    uint32_t id = 0, off = 0;
    if (sees) {
      const uint32_t pi = (uint32_t)(j / ix.page);
      off = (uint32_t)(j - (int64_t)pi * ix.page);
      id = ix.tables[(int64_t)b * ix.width + pi];
      if (id >= ix.pages) { bad = true; sees = false; id = 0; }
    }
    float s = -INFINITY;
    if (sees) {
      const T* pk = kp.ptr + id * kp.sp + off * kp.st + hk * kp.sh;
      float acc = 0.0f;
      for (int d = 0; d < dim; ++d) acc = fmaf(qs[d], ldf(pk, d), acc);
      s = acc * scale;
    }
    at = id * vp.sp + off * vp.st;
    const uint32_t seen = __ballot_sync(0xffffffffu, sees);
    if (seen == 0) continue;
    any = true;
    const float m_new = fmaxf(m, warp_max(s));
    const float base = m_new == -INFINITY ? 0.0f : m_new;      // every score -inf so far
    const float corr = expf(m - base), p = sees ? expf(s - base) : 0.0f;
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int i = 0; i < MAX_HEAD_COLUMNS; ++i) o[i] *= corr;
    for (uint32_t left = seen; left; left &= left - 1) {
      const int jj = __ffs(left) - 1;
      const float pj = __shfl_sync(0xffffffffu, p, jj);
      const T* pv = vp.ptr + __shfl_sync(0xffffffffu, at, jj) + hk * vp.sh;
#pragma unroll
      for (int i = 0; i < MAX_HEAD_COLUMNS; ++i) { const int d = lane + 32 * i; if (d < dim) o[i] = fmaf(pj, ldf(pv, d), o[i]); }
    }
    m = m_new;
  }
  bool wrong = any && !(isfinite(l) && l > 0.0f && isfinite(m));
  l = only_minus_inf(any, m, l);
  const float inv = inverse_sum(m, l);
  T* po = out.ptr + t * out.sn + h * out.sh;
#pragma unroll
  for (int i = 0; i < MAX_HEAD_COLUMNS; ++i) {
    const int d = lane + 32 * i;
    if (d < dim) { const float v = any ? o[i] * inv : 0.0f; wrong |= !isfinite(v); stf(po, d, v); }
  }
  if (lane == 0 && lse) lse[t * heads + h] = any ? m + logf(l) : -INFINITY;
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
  else if (wrong) raise_fault(fault, OP_PAGED_ATTN);
}

// ======================================================================== tiles on the tensor cores
// Row tiles of 16 * MW rows, key blocks of 64 or 128 (paged_attn.cuh has the line of work).
//
// What bounds it: the cache's bytes for few rows. Four warps to a CTA, one to three CTAs to an SM, two or three stages of 64 or 128 keys each, rows fetched by 16-byte asynchronous
// copies through the block table (a warp's lanes look up their keys' pages one block ahead of the copies). With one row tile (MW 1) the four warps share
// out the keys of a block and each waits for its own rows only; with MW 2 and 4 they share out rows, so that a key is used by 16 * MW rows once loaded.
// Products: mma.sync m16n8k16 (BF16), or m16n8k8 TF32 with each F32 operand split in two (hi*hi + hi*lo + lo*hi: what is
// dropped is 2^-22 of a product, 2^-21 of a weight times a value). Weights are rounded to BF16 for the BF16 product, as the operand has to be; the running
// sum takes them unrounded. Against 64 bits: rms error 1.7e-4 of outputs of rms 0.096 for 64 single tokens over up to 8191 places, 3.0e-4 of 0.13 for trees
// of 63, where F32 weights have 1.6e-4 and 2.1e-4 (the output's own rounding).
constexpr int TILE_WARPS = 4;

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo up to 2^-22 |x|, both TF32
__device__ __forceinline__ void split_tf32(float x, uint32_t* hi, uint32_t* lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(*hi) : "f"(x));
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(*lo) : "f"(x - __uint_as_float(*hi)));
}
// The same for a value, its upper half cut off and not rounded: a finite one stays finite (the last binade would round up to infinity). x = hi + lo up to
// 2^-21 |x|; errors of the outputs are the same, and the cut is cheaper than the conversion (which saturated takes 7 % of the kernel).
__device__ __forceinline__ void split_tf32_value(float x, uint32_t* hi, uint32_t* lo) {
  *hi = __float_as_uint(x) & 0xffffe000u;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(*lo) : "f"(x - __uint_as_float(*hi)));
}
__device__ __forceinline__ float quad_max(float v) { v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1)); return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2)); }
__device__ __forceinline__ float quad_sum(float v) { v += __shfl_xor_sync(0xffffffffu, v, 1); return v + __shfl_xor_sync(0xffffffffu, v, 2); }

template <class T, int D, int MW> struct TileShape {
  // keys to a block: 64, or 128 where rows are short and a warp would have little to do with 16 of them (one row tile, BF16, 64 columns)
  static constexpr int KEYS = std::is_same<T, bf16>::value && D == 64 && MW < 4 ? 128 : 64, WARP_KEYS = KEYS / TILE_WARPS;
  static constexpr int K_PITCH = std::is_same<T, float>::value ? D + 4 : D + 8, V_PITCH = D + 8;   // elements: odd multiples of 16 bytes (ldmatrix), or 4 and 8 banks a row (F32 fragments)
  static constexpr int STAGE = KEYS * (K_PITCH + V_PITCH) * (int)sizeof(T);
  static constexpr bool Q_IN_REGS = std::is_same<T, bf16>::value && D <= 128;
  static constexpr int JOINT = MW < TILE_WARPS ? 16 * (D + 2) * 4 : 0, OFFSETS = 2 * KEYS * 8, Q_TILE = Q_IN_REGS ? 0 : 16 * MW * K_PITCH * (int)sizeof(T);
  // What else an SM holds: two CTAs of three stages, or of two, or one CTA.
  static constexpr int REST = JOINT + OFFSETS + Q_TILE, HALF_SM = 112 * 1024 + 512;
  // With four row tiles a CTA computes more than it waits: three CTAs where a warp does with 168 registers (16 x 128 drafts x 8 heads of 64: 460 -> 385 us;
  // of 128 columns, spilling, 671 -> 893)
  static constexpr bool THIRD = MW == 4 && std::is_same<T, bf16>::value && D <= 80;
  static constexpr int STAGES = THIRD ? 2 : 3 * STAGE + REST <= HALF_SM ? 3 : 2 * STAGE + REST <= HALF_SM ? 2 : 3 * STAGE + REST <= 226 * 1024 ? 3 : 2;
  static constexpr int SMEM = STAGES * STAGE + REST;
  static constexpr int CTAS_PER_SM = THIRD ? 3 : SMEM <= HALF_SM ? 2 : 1;
};

template <class T, int D, int MW>
__global__ void __launch_bounds__(TILE_WARPS * 32, TileShape<T, D, MW>::CTAS_PER_SM)
paged_attention_tiles_kernel(RowsView<const T> q, PagesView<const T> kp, PagesView<const T> vp, PassIndex ix, RowsView<T> out, float* __restrict__ lse, TileWork work, int heads,
                             int group, int kv_heads, float scale, uint32_t* fault) {
  using S = TileShape<T, D, MW>;
  constexpr bool F32 = std::is_same<T, float>::value;
  constexpr int STAGES = S::STAGES;
  constexpr int BLOCK_KEYS = S::KEYS, WARP_KEYS = S::WARP_KEYS;                                           // WARP_KEYS: those that a warp fetches
  constexpr int KW = TILE_WARPS / MW, KEYS = BLOCK_KEYS / KW, NT = KEYS / 8, OT = D / 8, TILE_ROWS = 16 * MW;
  constexpr int CHUNKS = D * (int)sizeof(T) / 16, PER = 16 / (int)sizeof(T);
  constexpr int KSTEP = F32 ? 8 : 16, KSTEPS = D / KSTEP;
  extern __shared__ __align__(128) uint8_t raw[];
  float* joint = reinterpret_cast<float*>(raw + STAGES * S::STAGE);                                   // [16][D] and [16] (m, l): the warps' outputs meet here
  uint64_t* rows_at = reinterpret_cast<uint64_t*>(raw + STAGES * S::STAGE + S::JOINT);
  T* q_tile = reinterpret_cast<T*>(rows_at + 2 * BLOCK_KEYS);                                          // only without Q_IN_REGS
  __shared__ ShareScratch s_share;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, mw = warp % MW, kw = warp / MW, quad = lane >> 2, pair = lane & 3;
  bool bad = false, wrong = false;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tid == 0) work.split[blockIdx.x].pieces = 0;
  Share<BLOCK_KEYS> share;
  const bool any_work = find_share<BLOCK_KEYS, TILE_WARPS * 32>(ix, group, TILE_ROWS, kv_heads, &s_share, &share, &bad);
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
  if (!any_work) return;
  const uint32_t begin = share.begin;
  const int todo = share.todo;
  Cursor<BLOCK_KEYS> use = share.at;
  Cursor<BLOCK_KEYS> ahead = use;                                                                                   // the block whose pages are looked up next

  // ---- copies: warp w fetches WARP_KEYS keys of a block from number w * WARP_KEYS on; with 16, lane l looks up key l's row of K and lane 16 + l its row of V,
  // with 32 a lane does both. Places behind the last one repeat it, those before the first that a row can see repeat that one: what lies there is masked
  // like any place that is not seen.
  const PagesView<const T>& mine = lane < 16 ? kp : vp;
  const char* const mine_ptr = (const char*)mine.ptr;
  const int64_t mine_sp = mine.sp * (int)sizeof(T), mine_st = mine.st * (int)sizeof(T), mine_sh = mine.sh * (int)sizeof(T);
  struct Place { uint32_t id, off; int hk; };
  auto look_up = [&]() {
    Place p;
    const uint32_t last = ahead.r.cached + (uint32_t)ahead.r.fresh - 1;
    const uint32_t j = max(min((uint32_t)((ahead.r.first_block + ahead.block) * BLOCK_KEYS + WARP_KEYS * warp + lane % WARP_KEYS), last), first_place(ix, ahead.r.cached));
    const uint32_t pi = ix.page_shift >= 0 ? j >> ix.page_shift : j / ix.page;
    p.off = j - pi * ix.page;
    p.id = ix.tables[(int64_t)ahead.b * ix.width + pi];
    p.hk = ahead.hk;
    ahead.step(ix, group, TILE_ROWS, kv_heads, &bad);
    return p;
  };
  uint64_t* my_rows = rows_at + warp * 2 * WARP_KEYS;                                                   // K's, then V's
  const uint32_t k_base = smem_addr(raw) + (WARP_KEYS * warp + lane / CHUNKS) * S::K_PITCH * (int)sizeof(T) + (lane % CHUNKS) * 16;
  const uint32_t v_base = smem_addr(raw) + (BLOCK_KEYS * S::K_PITCH + (WARP_KEYS * warp + lane / CHUNKS) * S::V_PITCH) * (int)sizeof(T) + (lane % CHUNKS) * 16;
  auto copy_block = [&](int stage, Place p) {
    if (p.id >= ix.pages) { bad = true; p.id = 0; }
    if (WARP_KEYS == 16) my_rows[lane] = (uint64_t)(mine_ptr + (int64_t)p.id * mine_sp + (int64_t)p.off * mine_st + (int64_t)p.hk * mine_sh);
    else {
      my_rows[lane] = (uint64_t)(kp.ptr + p.id * kp.sp + p.off * kp.st + p.hk * kp.sh);
      my_rows[32 + lane] = (uint64_t)(vp.ptr + p.id * vp.sp + p.off * vp.st + p.hk * vp.sh);
    }
    __syncwarp();
    const uint32_t ka = k_base + stage * S::STAGE, va = v_base + stage * S::STAGE;
    if constexpr (32 % CHUNKS == 0) {                                                                   // a lane keeps its column of 16 bytes
      constexpr int ROWS = 32 / CHUNKS;
      const uint64_t* at = my_rows + lane / CHUNKS;
      const int c = (lane % CHUNKS) * 16;
#pragma unroll
      for (int i = 0; i < WARP_KEYS / ROWS; ++i) copy16(ka + i * ROWS * S::K_PITCH * (int)sizeof(T), (const char*)at[i * ROWS] + c);
#pragma unroll
      for (int i = 0; i < WARP_KEYS / ROWS; ++i) copy16(va + i * ROWS * S::V_PITCH * (int)sizeof(T), (const char*)at[WARP_KEYS + i * ROWS] + c);
    } else {
      const uint32_t kw0 = smem_addr(raw) + stage * S::STAGE + WARP_KEYS * warp * S::K_PITCH * (int)sizeof(T);
      const uint32_t vw0 = smem_addr(raw) + stage * S::STAGE + (BLOCK_KEYS * S::K_PITCH + WARP_KEYS * warp * S::V_PITCH) * (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < CHUNKS * WARP_KEYS / 32; ++i) {
        const int n = lane + 32 * i, row = n / CHUNKS, c = n % CHUNKS * 16;
        copy16(kw0 + row * S::K_PITCH * (int)sizeof(T) + c, (const char*)my_rows[row] + c);
        copy16(vw0 + row * S::V_PITCH * (int)sizeof(T) + c, (const char*)my_rows[WARP_KEYS + row] + c);
      }
    }
    __syncwarp();
  };
  uint32_t qf[S::Q_IN_REGS ? KSTEPS : 1][4];
  float o[OT][4], m[2], l[2];
  bool any[2];
  uint32_t from[2], from_most = 0;                                                                      // the first position in a row's window
  int local[2];
  bool live[2];
  const float c2 = scale * LOG2_E;
  uint32_t piece_begin = begin;
  Place next_place;
  auto begin_unit = [&](uint32_t at) {                                                                   // a new unit: its rows
    const int row_tile = use.row_tile, hk = use.hk;
    piece_begin = at;
    from_most = 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = row_tile * TILE_ROWS + 16 * mw + quad + 8 * x;
      live[x] = r < use.r.fresh * group;
      local[x] = live[x] ? r / group : 0;
      const int64_t t = use.r.first + local[x];
      from[x] = 0;
      if (ix.window > 0) {
        const uint32_t place = ix.positions ? ix.positions[t] : use.r.cached + (uint32_t)local[x];
        from[x] = place >= ix.window ? place - (uint32_t)ix.window + 1 : 0;
        if (live[x] && place < use.r.cached) bad = true;
        if (live[x]) from_most = max(from_most, from[x]);
      }
      m[x] = -INFINITY; l[x] = 0.0f; any[x] = false;
      if (S::Q_IN_REGS) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(q.ptr + t * q.sn + (int64_t)(hk * group + (live[x] ? r % group : 0)) * q.sh);
#pragma unroll
        for (int k = 0; k < KSTEPS; ++k) { qf[k][x] = live[x] ? p[8 * k + pair] : 0u; qf[k][2 + x] = live[x] ? p[8 * k + 4 + pair] : 0u; }
      }
    }
    if (ix.window > 0) from_most = __reduce_max_sync(0xffffffffu, from_most);
    if (!S::Q_IN_REGS) {                                                                                 // by copies: the first unit's ride with the first block's
      __syncthreads();
      for (int i = tid; i < TILE_ROWS * CHUNKS; i += TILE_WARPS * 32) {
        const int r = i / CHUNKS, c = i % CHUNKS, g = row_tile * TILE_ROWS + r;
        T* dst = q_tile + r * S::K_PITCH + c * PER;
        if (g < use.r.fresh * group) copy16(smem_addr(dst), q.ptr + (int64_t)(use.r.first + g / group) * q.sn + (int64_t)(hk * group + g % group) * q.sh + c * PER);
        else *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
      }
      if (at != begin) { copies_commit(); copies_wait<0>(); __syncthreads(); }
    }
#pragma unroll
    for (int n = 0; n < OT; ++n) { o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f; }
  };
  {
    Place p[STAGES];                                                                                    // all look-ups, the queries, then the copies
#pragma unroll
    for (int i = 0; i < STAGES; ++i) if (i < todo) p[i] = look_up();
    begin_unit(begin);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (i < todo) copy_block(i, p[i]);
      copies_commit();
    }
    next_place = p[STAGES - 1];
  }

  int stage = 0;
  for (int f = 0; f < todo; ++f) {
    if (f > 0 && use.block == 0) begin_unit(begin + f);
    const int row_tile = use.row_tile, hk = use.hk;

    copies_wait<STAGES - 2>();
    if (MW == 1 && (S::Q_IN_REGS || f > 0)) __syncwarp(); else __syncthreads();
    {                                                                                                   // the stage that the last block left
      const int next = f + STAGES - 1;
      if (next < todo) { copy_block(stage == 0 ? STAGES - 1 : stage - 1, next_place); if (next + 1 < todo) next_place = look_up(); }
      copies_commit();
    }
    const T* kt = reinterpret_cast<const T*>(raw + stage * S::STAGE) + kw * KEYS * S::K_PITCH;
    const T* vt = reinterpret_cast<const T*>(raw + stage * S::STAGE) + BLOCK_KEYS * S::K_PITCH + kw * KEYS * S::V_PITCH;
    const uint32_t j0 = (uint32_t)((use.r.first_block + use.block) * BLOCK_KEYS + kw * KEYS);
    stage = stage + 1 == STAGES ? 0 : stage + 1;

    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f; }
    if (!F32) {
      const uint32_t ka = smem_addr(kt) + ((((lane >> 4) & 1) * 8 + (lane & 7)) * S::K_PITCH + ((lane >> 3) & 1) * 8) * 2;
      const uint32_t qa = smem_addr(q_tile) + ((16 * mw + (lane & 15)) * S::K_PITCH + (lane >> 4) * 8) * 2;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        uint32_t a[4];
        if (S::Q_IN_REGS) { a[0] = qf[k][0]; a[1] = qf[k][1]; a[2] = qf[k][2]; a[3] = qf[k][3]; }
        else ldmatrix4(a, qa + k * 32);
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          uint32_t b4[4];
          ldmatrix4(b4, ka + (n * 8 * S::K_PITCH + k * 16) * 2);
          mma_bf16(s[n], a, b4[0], b4[1]);
          mma_bf16(s[n + 1], a, b4[2], b4[3]);
        }
      }
    } else {
      // with few tiles to a warp the three products of a step have sums of their own: a third of the chain of dependent products
      constexpr bool APART = NT <= 4;
      float s1[APART ? NT : 1][4], s2[APART ? NT : 1][4];
#pragma unroll
      for (int n = 0; n < (APART ? NT : 1); ++n) { s1[n][0] = s1[n][1] = s1[n][2] = s1[n][3] = 0.0f; s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0.0f; }
      const float* qa = reinterpret_cast<const float*>(q_tile) + (16 * mw + quad) * S::K_PITCH + pair;
      const float* ka = reinterpret_cast<const float*>(kt) + quad * S::K_PITCH + pair;
#pragma unroll 4
      for (int k = 0; k < KSTEPS; ++k) {
        uint32_t ah[4], al[4];
        split_tf32(qa[8 * k], &ah[0], &al[0]); split_tf32(qa[8 * S::K_PITCH + 8 * k], &ah[1], &al[1]);
        split_tf32(qa[8 * k + 4], &ah[2], &al[2]); split_tf32(qa[8 * S::K_PITCH + 8 * k + 4], &ah[3], &al[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t bh0, bl0, bh1, bl1;
          split_tf32(ka[n * 8 * S::K_PITCH + 8 * k], &bh0, &bl0); split_tf32(ka[n * 8 * S::K_PITCH + 8 * k + 4], &bh1, &bl1);
          mma_tf32(APART ? s1[APART ? n : 0] : s[n], al, bh0, bh1);
          mma_tf32(APART ? s2[APART ? n : 0] : s[n], ah, bl0, bl1);
          mma_tf32(s[n], ah, bh0, bh1);
        }
      }
      if (APART) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] += s1[APART ? n : 0][e] + s2[APART ? n : 0][e];
        }
      }
      // An operand that is infinite, or rounds up to it, is not the sum of its two parts: scores that are not finite are formed once more from the operands
      float odd[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) odd[e] = fmaf(s[n][e], 0.0f, odd[e]);
      }
      if (__any_sync(0xffffffffu, (odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.0f)) {
#pragma unroll 1
        for (int n = 0; n < NT; ++n) {                                                                  // the tile in work is s[0]: they move on
          float now[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float* qr = reinterpret_cast<const float*>(q_tile) + (16 * mw + quad + 8 * (e >> 1)) * S::K_PITCH;
            const float* kr = reinterpret_cast<const float*>(kt) + (8 * n + 2 * pair + (e & 1)) * S::K_PITCH;
            now[e] = s[0][e];
            if (!isfinite(now[e])) {
              now[e] = 0.0f;
#pragma unroll 1
              for (int d = 0; d < D; ++d) now[e] = fmaf(qr[d], kr[d], now[e]);
            }
          }
#pragma unroll
          for (int i = 0; i + 1 < NT; ++i) { s[i][0] = s[i + 1][0]; s[i][1] = s[i + 1][1]; s[i][2] = s[i + 1][2]; s[i][3] = s[i + 1][3]; }
          s[NT - 1][0] = now[0]; s[NT - 1][1] = now[1]; s[NT - 1][2] = now[2]; s[NT - 1][3] = now[3];
        }
      }
    }

    // ---- what the rows see: everything in a block below the cached length and inside every row's window
    uint32_t sees = 0xffffffffu;                                                                        // bit 4 n + element
    bool poisoned = false;
    if (j0 + KEYS > use.r.cached || j0 < from_most) {
      sees = 0;
#pragma unroll 1
      for (int i = 0; i < 4 * NT; ++i) {                                                                // a loop, for the code's size: few blocks come here
        const int x = (i >> 1) & 1;
        const uint32_t j = j0 + 8 * (i >> 2) + 2 * pair + (i & 1), mine_from = x ? from[1] : from[0];
        const uint32_t row = (uint32_t)(x ? local[1] : local[0]);
        bool v = x ? live[1] : live[0];
        if (j < use.r.cached) v = v && j >= mine_from;
        else {
          const uint32_t d = j - use.r.cached;
          v = v && d < (uint32_t)use.r.fresh;
          if (v) v = ix.masks ? (d >> 5) < (uint32_t)ix.words && (ix.masks[(int64_t)(use.r.first + row) * ix.words + (d >> 5)] >> (d & 31) & 1u) : d <= row;
          if (v && ix.window > 0) v = (ix.positions ? ix.positions[use.r.first + d] : j) >= mine_from;
        }
        sees |= (uint32_t)v << i;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (!(sees >> (4 * n + e) & 1u)) s[n][e] = -INFINITY;
      }
      // a value that only some rows see must not reach the others as 0 x NaN: such a block's second product goes without the tensor cores
      const uint32_t* w = reinterpret_cast<const uint32_t*>(vt);
      constexpr int WORDS = D * (int)sizeof(T) / 4, PITCH_WORDS = S::V_PITCH * (int)sizeof(T) / 4;
      for (int i = lane; i < KEYS * WORDS; i += 32) {
        const uint32_t x = w[(i / WORDS) * PITCH_WORDS + i % WORDS];
        if (F32) poisoned |= (x & 0x7f800000u) == 0x7f800000u;
        else poisoned |= (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
      }
      poisoned = __any_sync(0xffffffffu, poisoned);
    }

    // ---- running maximum and sum
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) top = fmaxf(top, fmaxf(s[n][2 * x], s[n][2 * x + 1]));
      top = fmaxf(m[x], quad_max(top));
      const float base = top == -INFINITY ? 0.0f : top * c2;
      const float corr = exp2_fast(fmaf(m[x], c2, -base));
      float sum = 0.0f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        s[n][2 * x] = exp2_fast(fmaf(s[n][2 * x], c2, -base));
        s[n][2 * x + 1] = exp2_fast(fmaf(s[n][2 * x + 1], c2, -base));
        sum += s[n][2 * x] + s[n][2 * x + 1];
      }
      any[x] |= (sees & (0x33333333u << (2 * x)) & (NT == 8 ? 0xffffffffu : (1u << (4 * NT & 31)) - 1u)) != 0;
      if (__any_sync(0xffffffffu, top != m[x])) {
#pragma unroll
        for (int n = 0; n < OT; ++n) { o[n][2 * x] *= corr; o[n][2 * x + 1] *= corr; }
      }
      l[x] = l[x] * corr + sum;
      m[x] = top;
    }

    // ---- O += P V
    if (poisoned) {
#pragma unroll 1
      for (int k = 0; k < KEYS; ++k) {                                                                  // the key's weights lie in s[0]: the tile moves on every eight keys
        const int from_lane = (lane & ~3) | ((k & 7) >> 1);
        float p[2];
        bool v[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          p[x] = __shfl_sync(0xffffffffu, (k & 1) ? s[0][2 * x + 1] : s[0][2 * x], from_lane);
          v[x] = __shfl_sync(0xffffffffu, sees >> (4 * (k >> 3) + 2 * x + (k & 1)) & 1u, from_lane);
        }
#pragma unroll
        for (int i = 0; i < OT; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float val = ldf(vt, k * S::V_PITCH + 8 * i + 2 * pair + (e & 1));
            if (v[e >> 1]) o[i][e] = fmaf(p[e >> 1], val, o[i][e]);
          }
        }
        if ((k & 7) == 7) {
#pragma unroll
          for (int n = 0; n + 1 < NT; ++n) { s[n][0] = s[n + 1][0]; s[n][1] = s[n + 1][1]; s[n][2] = s[n + 1][2]; s[n][3] = s[n + 1][3]; }
        }
      }
    } else if (!F32) {
      const uint32_t va = smem_addr(vt) + ((((lane >> 3) & 1) * 8 + (lane & 7)) * S::V_PITCH + ((lane >> 4) & 1) * 8) * 2;
#pragma unroll
      for (int k = 0; k < NT / 2; ++k) {
        const uint32_t a[4] = {pack_bf16(s[2 * k][0], s[2 * k][1]), pack_bf16(s[2 * k][2], s[2 * k][3]), pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]),
                               pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
        for (int n = 0; n < OT; n += 2) {
          uint32_t b4[4];
          ldmatrix4_trans(b4, va + (k * 16 * S::V_PITCH + n * 8) * 2);
          mma_bf16(o[n], a, b4[0], b4[1]);
          mma_bf16(o[n + 1], a, b4[2], b4[3]);
        }
      }
    } else {
      // the k index of the product runs over keys in the order 0 2 4 6 1 3 5 7 of a tile of eight: the order in which the scores lie in the registers
      const float* va = reinterpret_cast<const float*>(vt) + 2 * pair * S::V_PITCH + quad;
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        uint32_t ah[4], al[4];
        split_tf32(s[k][0], &ah[0], &al[0]); split_tf32(s[k][2], &ah[1], &al[1]); split_tf32(s[k][1], &ah[2], &al[2]); split_tf32(s[k][3], &ah[3], &al[3]);
#pragma unroll
        for (int n = 0; n < OT; ++n) {
          uint32_t bh0, bl0, bh1, bl1;
          split_tf32_value(va[k * 8 * S::V_PITCH + 8 * n], &bh0, &bl0); split_tf32_value(va[(k * 8 + 1) * S::V_PITCH + 8 * n], &bh1, &bl1);
          mma_tf32(o[n], al, bh0, bh1);
          mma_tf32(o[n], ah, bl0, bl1);
          mma_tf32(o[n], ah, bh0, bh1);
        }
      }
    }

    // ---- the end of the unit, or of this CTA's piece of it
    const bool unit_done = use.block + 1 == use.r.blocks;
    if (unit_done || f + 1 == todo) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        l[x] = quad_sum(l[x]);
        int seen = any[x];
        seen |= __shfl_xor_sync(0xffffffffu, seen, 1); seen |= __shfl_xor_sync(0xffffffffu, seen, 2);
        l[x] = only_minus_inf(seen, m[x], l[x]);
      }
      if (KW > 1) {                                                                                     // the warps that share a row tile add up in order
        const int rows = min(16, use.r.fresh * group - row_tile * TILE_ROWS);                            // of a row tile of 16 (MW 1)
        const bool at_once = MW == 1 && rows * (KW - 1) <= 16;                                           // all warps' rows fit next to one another
        float* jm = joint + 16 * D;
        auto give = [&](int at) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = quad + 8 * x;
            if (!live[x]) continue;
            if (pair == 0) { jm[2 * (at + r)] = m[x]; jm[2 * (at + r) + 1] = l[x]; }
#pragma unroll
            for (int n = 0; n < OT; ++n) *reinterpret_cast<float2*>(joint + (at + r) * D + 8 * n + 2 * pair) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
          }
        };
        auto take = [&](int at) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = at + quad + 8 * x;
            if (!live[x]) continue;
            const float m2 = jm[2 * r], l2 = jm[2 * r + 1], top = fmaxf(m[x], m2), base = top == -INFINITY ? 0.0f : top * c2;
            const float ca = exp2_fast(fmaf(m[x], c2, -base)), cb = exp2_fast(fmaf(m2, c2, -base));
            l[x] = joined_sum(top, l[x], ca, l2, cb);
            m[x] = top;
#pragma unroll
            for (int n = 0; n < OT; ++n) {
              const float2 v = *reinterpret_cast<const float2*>(joint + r * D + 8 * n + 2 * pair);
              o[n][2 * x] = o[n][2 * x] * ca + v.x * cb;
              o[n][2 * x + 1] = o[n][2 * x + 1] * ca + v.y * cb;
            }
          }
        };
        __syncthreads();                                                                                 // what a unit before left has been taken
        if (at_once) {
          if (kw > 0) give((kw - 1) * rows);
          __syncthreads();
          if (kw == 0) {
#pragma unroll 1
            for (int w = 1; w < KW; ++w) take((w - 1) * rows);
          }
        } else {
#pragma unroll 1
          for (int w = 1; w < KW; ++w) {
#pragma unroll 1
            for (int g = 0; g < MW; ++g) {
              if (kw == w && mw == g) give(0);
              __syncthreads();
              if (kw == 0 && mw == g) take(0);
              __syncthreads();
            }
          }
        }
      }
      const uint32_t unit_begin = begin + f - use.block;
      const bool whole = unit_done && piece_begin == unit_begin;
      if (kw == 0) {
        const int slot = 2 * blockIdx.x + (piece_begin == unit_begin ? 1 : 0);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!live[x]) continue;
          const int r = row_tile * TILE_ROWS + 16 * mw + quad + 8 * x;
          const int64_t t = use.r.first + local[x];
          const int h = hk * group + r % group;
          if (whole) {
            const bool seen = !(m[x] == -INFINITY && l[x] == 0.0f);
            const float inv = inverse_sum(m[x], l[x]);
            T* p = out.ptr + t * out.sn + h * out.sh;
#pragma unroll
            for (int n = 0; n < OT; ++n) {
              const float u = o[n][2 * x] * inv, v = o[n][2 * x + 1] * inv;
              wrong |= !isfinite(u) || !isfinite(v);
              if (F32) *reinterpret_cast<float2*>(p + 8 * n + 2 * pair) = make_float2(u, v);
              else *reinterpret_cast<uint32_t*>(p + 8 * n + 2 * pair) = pack_bf16(u, v);
            }
            if (pair == 0 && lse) lse[t * heads + h] = seen ? m[x] * scale + logf(l[x]) : -INFINITY;
          } else {
            const int64_t row = (int64_t)slot * TILE_ROWS + 16 * mw + quad + 8 * x;
            if (pair == 0) work.ml[row] = make_float2(m[x] * c2, l[x]);
#pragma unroll
            for (int n = 0; n < OT; ++n) *reinterpret_cast<float2*>(work.o + row * D + 8 * n + 2 * pair) = make_float2(o[n][2 * x], o[n][2 * x + 1]);
          }
        }
      }
      if (!unit_done && piece_begin == unit_begin && tid == 0) {                                        // this CTA holds the unit's first piece
        work.split[blockIdx.x] = SplitUnit{(int)(share.of_block(unit_begin + use.r.blocks - 1) - blockIdx.x) + 1, hk, row_tile * TILE_ROWS,
                                               min(TILE_ROWS, use.r.fresh * group - row_tile * TILE_ROWS), use.r.first};
      }
    }
    use.step(ix, group, TILE_ROWS, kv_heads, &bad);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
  else if (wrong) raise_fault(fault, OP_PAGED_ATTN);
}

// ======================================================================== few rows in F32
// Up to four rows to a KV head in F32, where the tiles' split products (three MMAs on 16 rows, each operand taken apart) cost more than the bytes: plain
// fused multiply-adds. A warp takes 16 keys of a block of 64: for the scores a pair of lanes shares a key, alternating chunks of 16 bytes (rows of D + 8
// words: no bank conflicts); for the output a lane keeps D / 32 columns and the keys' weights come by shuffles. The line of work, the copies and the joining are the
// tiles kernel's. Bound by the cache's bytes: 12 x 64 heads over 60,000 places 65 us, 5.7 TB/s, against 113 on the
// tiles; 8 x 4000 places of 12 x 128 51 us against 97.
template <int D, int R> struct FewShape {
  static constexpr int PITCH = D + 8, KEYS = 64, STAGE = 2 * KEYS * PITCH * 4, JOINT = 3 * R * (D + 2) * 4, OFFSETS = 2 * KEYS * 8, Q_TILE = R * D * 4;
  static constexpr int REST = JOINT + OFFSETS + Q_TILE, HALF_SM = 113 * 1024;
  static constexpr int STAGES = 3 * STAGE + REST <= HALF_SM ? 3 : 2 * STAGE + REST <= HALF_SM ? 2 : 3;
  static constexpr int SMEM = STAGES * STAGE + REST, CTAS_PER_SM = SMEM <= HALF_SM ? 2 : 1;
};

template <int D, int R>
__global__ void __launch_bounds__(TILE_WARPS * 32, FewShape<D, R>::CTAS_PER_SM)
paged_attention_few_kernel(RowsView<const float> q, PagesView<const float> kp, PagesView<const float> vp, PassIndex ix, RowsView<float> out, float* __restrict__ lse, TileWork work, int heads,
                           int group, int kv_heads, float scale, uint32_t* fault) {
  using S = FewShape<D, R>;
  constexpr int KEYS = S::KEYS, STAGES = S::STAGES, COLS = D / 32, CHUNKS = D / 4;
  extern __shared__ __align__(128) uint8_t raw[];
  uint64_t* rows_at = reinterpret_cast<uint64_t*>(raw + STAGES * S::STAGE);
  float* q_tile = reinterpret_cast<float*>(rows_at + 2 * KEYS);
  float* joint = q_tile + R * D;                                             // [3 R][D], then (m, l) of each
  float* jm = joint + 3 * R * D;
  __shared__ ShareScratch s_share;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  bool bad = false, wrong = false;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tid == 0) work.split[blockIdx.x].pieces = 0;
  Share<KEYS> share;
  const bool any_work = find_share<KEYS, TILE_WARPS * 32>(ix, group, R, kv_heads, &s_share, &share, &bad);
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
  if (!any_work) return;
  const uint32_t begin = share.begin;
  const int todo = share.todo;
  Cursor<KEYS> use = share.at, ahead = use;
  // copies: lane l looks up key l's row of K, lane 16 + l its row of V; places behind the last one repeat it, those before the first
  // that a row can see repeat that one
  struct Place { uint32_t id, off; int hk; };
  auto look_up = [&]() {
    Place p;
    const uint32_t last = ahead.r.cached + (uint32_t)ahead.r.fresh - 1;
    const uint32_t j = max(min((uint32_t)((ahead.r.first_block + ahead.block) * KEYS + 16 * warp + (lane & 15)), last), first_place(ix, ahead.r.cached));
    const uint32_t pi = ix.page_shift >= 0 ? j >> ix.page_shift : j / ix.page;
    p.off = j - pi * ix.page;
    p.id = ix.tables[(int64_t)ahead.b * ix.width + pi];
    p.hk = ahead.hk;
    ahead.step(ix, group, R, kv_heads, &bad);
    return p;
  };
  uint64_t* my_rows = rows_at + warp * 32;
  auto copy_block = [&](int stage, Place p) {
    if (p.id >= ix.pages) { bad = true; p.id = 0; }
    my_rows[lane] = lane < 16 ? (uint64_t)(kp.ptr + p.id * kp.sp + p.off * kp.st + p.hk * kp.sh) : (uint64_t)(vp.ptr + p.id * vp.sp + p.off * vp.st + p.hk * vp.sh);
    __syncwarp();
    const uint32_t k0 = smem_addr(raw) + stage * S::STAGE + 16 * warp * S::PITCH * 4, v0 = k0 + KEYS * S::PITCH * 4;
#pragma unroll
    for (int i = 0; i < CHUNKS / 2; ++i) {
      const int n = lane + 32 * i, row = n / CHUNKS, c = n % CHUNKS * 16;
      copy16(k0 + row * S::PITCH * 4 + c, (const char*)my_rows[row] + c);
      copy16(v0 + row * S::PITCH * 4 + c, (const char*)my_rows[16 + row] + c);
    }
    __syncwarp();
  };
  float o[R][COLS], m[R], l[R];
  bool any[R];
  uint32_t from[R], from_most = 0;
  int local[R], rows = 0;
  const float c2 = scale * LOG2_E;
  uint32_t piece_begin = begin;
  auto begin_unit = [&](uint32_t at) {
    piece_begin = at;
    from_most = 0;
    rows = min(R, use.r.fresh * group - use.row_tile * R);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int n = use.row_tile * R + (r < rows ? r : 0);
      local[r] = n / group;
      from[r] = 0;
      if (ix.window > 0) {
        const uint32_t place = ix.positions ? ix.positions[use.r.first + local[r]] : use.r.cached + (uint32_t)local[r];
        if (place < use.r.cached) bad = true;
        from[r] = place >= ix.window ? place - (uint32_t)ix.window + 1 : 0;
        from_most = max(from_most, from[r]);
      }
      m[r] = -INFINITY; l[r] = 0.0f; any[r] = false;
#pragma unroll
      for (int i = 0; i < COLS; ++i) o[r][i] = 0.0f;
    }
    __syncthreads();                                                          // the unit before has been computed
    for (int i = tid; i < R * CHUNKS; i += TILE_WARPS * 32) {
      const int r = i / CHUNKS, c = i % CHUNKS, n = use.row_tile * R + (r < rows ? r : 0);   // rows that are not there repeat the first
      copy16(smem_addr(q_tile + r * D + 4 * c), q.ptr + (int64_t)(use.r.first + n / group) * q.sn + (int64_t)(use.hk * group + n % group) * q.sh + 4 * c);
    }
    if (at != begin) { copies_commit(); copies_wait<0>(); __syncthreads(); }
  };
  Place next_place;
  {
    Place p[STAGES];
#pragma unroll
    for (int i = 0; i < STAGES; ++i) if (i < todo) p[i] = look_up();
    begin_unit(begin);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (i < todo) copy_block(i, p[i]);
      copies_commit();
    }
    next_place = p[STAGES - 1];
  }
  int stage = 0;
  for (int f = 0; f < todo; ++f) {
    if (f > 0 && use.block == 0) begin_unit(begin + f);
    copies_wait<STAGES - 2>();
    if (f > 0) __syncwarp(); else __syncthreads();
    const int next = f + STAGES - 1;
    if (next < todo) { copy_block(stage == 0 ? STAGES - 1 : stage - 1, next_place); if (next + 1 < todo) next_place = look_up(); }
    copies_commit();
    const float* kt = reinterpret_cast<const float*>(raw + stage * S::STAGE) + 16 * warp * S::PITCH;
    const float* vt = kt + KEYS * S::PITCH;
    const uint32_t j0 = (uint32_t)((use.r.first_block + use.block) * KEYS + 16 * warp), j = j0 + (lane >> 1);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    // scores: lanes 2 k and 2 k + 1 share key k
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = 0.0f;
    const float* krow = kt + (lane >> 1) * S::PITCH + 4 * (lane & 1);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(krow + 8 * i);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 y = *reinterpret_cast<const float4*>(q_tile + r * D + 8 * i + 4 * (lane & 1));
        s[r] = fmaf(x.x, y.x, s[r]); s[r] = fmaf(x.y, y.y, s[r]); s[r] = fmaf(x.z, y.z, s[r]); s[r] = fmaf(x.w, y.w, s[r]);
      }
    }
    const bool masked = j0 + 16 > use.r.cached || j0 < from_most;
    uint32_t sees[R];                                                          // by lanes
    float p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], 1);
      bool v = true;
      if (masked) {
        if (j < use.r.cached) v = j >= from[r];
        else {
          const uint32_t d = j - use.r.cached;
          v = d < (uint32_t)use.r.fresh;
          if (v) v = ix.masks ? (d >> 5) < (uint32_t)ix.words && (ix.masks[(int64_t)(use.r.first + local[r]) * ix.words + (d >> 5)] >> (d & 31) & 1u) : d <= (uint32_t)local[r];
          if (v && ix.window > 0) v = (ix.positions ? ix.positions[use.r.first + d] : j) >= from[r];
        }
      }
      sees[r] = __ballot_sync(0xffffffffu, v);
      any[r] |= sees[r] != 0;
      const float top = fmaxf(m[r], warp_max(v ? s[r] : -INFINITY)), base = top == -INFINITY ? 0.0f : top * c2, corr = exp2_fast(fmaf(m[r], c2, -base));
      p[r] = v ? exp2_fast(fmaf(s[r], c2, -base)) : 0.0f;
      l[r] = fmaf(l[r], corr, 0.5f * warp_sum(p[r]));                          // every key stands twice
      if (top != m[r]) {
#pragma unroll
        for (int i = 0; i < COLS; ++i) o[r][i] *= corr;
      }
      m[r] = top;
    }
    // output: a key's weight from its lanes; places that a row does not see are left out, whatever they hold
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float v[COLS];
      const float* vrow = vt + k * S::PITCH + lane * COLS;
      if constexpr (COLS == 4) { const float4 x = *reinterpret_cast<const float4*>(vrow); v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
      else if constexpr (COLS == 2) { const float2 x = *reinterpret_cast<const float2*>(vrow); v[0] = x.x; v[1] = x.y; }
      else {
#pragma unroll
        for (int i = 0; i < COLS; ++i) v[i] = vrow[i];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float w = __shfl_sync(0xffffffffu, p[r], 2 * k);
        if (sees[r] >> (2 * k) & 1u) {
#pragma unroll
          for (int i = 0; i < COLS; ++i) o[r][i] = fmaf(w, v[i], o[r][i]);
        }
      }
    }
    const bool unit_done = use.block + 1 == use.r.blocks;
    if (unit_done || f + 1 == todo) {
#pragma unroll
      for (int r = 0; r < R; ++r) l[r] = only_minus_inf(any[r], m[r], l[r]);
      __syncthreads();                                                          // what a unit before left has been taken
      if (warp > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int at = (warp - 1) * R + r;
#pragma unroll
          for (int i = 0; i < COLS; ++i) joint[at * D + lane * COLS + i] = o[r][i];
          if (lane == 0) { jm[2 * at] = m[r]; jm[2 * at + 1] = l[r]; }
        }
      }
      __syncthreads();
      const uint32_t unit_begin = begin + f - use.block;
      const bool starts = piece_begin == unit_begin, whole = unit_done && starts;
      if (warp == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r >= rows) continue;
#pragma unroll
          for (int w = 0; w < TILE_WARPS - 1; ++w) {
            const int at = w * R + r;
            const float m2 = jm[2 * at], l2 = jm[2 * at + 1], top = fmaxf(m[r], m2), base = top == -INFINITY ? 0.0f : top * c2;
            const float ca = exp2_fast(fmaf(m[r], c2, -base)), cb = exp2_fast(fmaf(m2, c2, -base));
            l[r] = joined_sum(top, l[r], ca, l2, cb);
            m[r] = top;
#pragma unroll
            for (int i = 0; i < COLS; ++i) o[r][i] = o[r][i] * ca + joint[at * D + lane * COLS + i] * cb;
          }
          const int n = use.row_tile * R + r, h = use.hk * group + n % group;
          const int64_t t = use.r.first + local[r];
          if (whole) {
            const bool seen = !(m[r] == -INFINITY && l[r] == 0.0f);
            const float inv = inverse_sum(m[r], l[r]);
            float* po = out.ptr + t * out.sn + h * out.sh + lane * COLS;
#pragma unroll
            for (int i = 0; i < COLS; ++i) { const float x = o[r][i] * inv; wrong |= !isfinite(x); po[i] = x; }
            if (lane == 0 && lse) lse[t * heads + h] = seen ? m[r] * scale + logf(l[r]) : -INFINITY;
          } else {
            const int64_t row = (int64_t)(2 * blockIdx.x + (starts ? 1 : 0)) * R + r;
            if (lane == 0) work.ml[row] = make_float2(m[r] * c2, l[r]);
#pragma unroll
            for (int i = 0; i < COLS; ++i) work.o[row * D + lane * COLS + i] = o[r][i];
          }
        }
      }
      if (!unit_done && starts && tid == 0)
        work.split[blockIdx.x] = SplitUnit{(int)(share.of_block(unit_begin + use.r.blocks - 1) - blockIdx.x) + 1, use.hk, use.row_tile * R, rows, use.r.first};
    }
    use.step(ix, group, R, kv_heads, &bad);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
  else if (wrong) raise_fault(fault, OP_PAGED_ATTN);
}

// Joins the pieces of the units that several CTAs shared: blocks (c, .) take the unit whose first piece CTA c left. A warp takes a row, or where a unit has
// many pieces a 2nd, 4th or 8th part of a row's (joined in a fixed order); lanes are columns. The loads of four pieces, maxima and outputs, are in
// flight together: two round trips to memory for a unit of up to four pieces (latency is all there is to this kernel, so registers are kept few: with
// eight pieces at 110 registers it took three times as long for units of 256 rows). COLS: 128 columns of four to a lane.
constexpr int JOIN_WARPS = 8, JOIN_PIECES = 4;

template <class T, int COLS>
__global__ void __launch_bounds__(JOIN_WARPS * 32, COLS == 1 ? 6 : 4)
paged_attention_join_kernel(RowsView<T> out, float* __restrict__ lse, TileWork work, int heads, int group, int tile_rows, int dim, uint32_t* fault) {
  __shared__ float s_l[JOIN_WARPS], s_m[JOIN_WARPS];
  extern __shared__ float acc[];                                          // [JOIN_WARPS][dim]
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const SplitUnit u = work.split[blockIdx.x];
  if (u.pieces == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int shares = 1;                                                         // warps to a row
  while (shares < JOIN_WARPS && shares * JOIN_PIECES < u.pieces) shares *= 2;
  const int part = warp % shares, step = JOIN_WARPS / shares;
  bool wrong = false;
  for (int r0 = blockIdx.y * step; r0 < u.rows; r0 += gridDim.y * step) {
    const int r = r0 + warp / shares;
    const bool live = r < u.rows;
    float top = -INFINITY, l = 0.0f;                                      // maxima in log2 units
    bool minus = false;                                                   // a piece saw scores of -inf alone
    float4 o[COLS];                                                       // columns 4 lane .. 4 lane + 3, and 128 more for a head of 256
#pragma unroll
    for (int i = 0; i < COLS; ++i) o[i] = make_float4(0, 0, 0, 0);
    for (int p0 = part; live && p0 < u.pieces; p0 += JOIN_PIECES * shares) {
      float4 v[COLS][JOIN_PIECES];
      float2 ml[JOIN_PIECES];
#pragma unroll
      for (int k = 0; k < JOIN_PIECES; ++k) {
        const int p = p0 + k * shares;
        const bool there = p < u.pieces;
        const int64_t row = (int64_t)(2 * (blockIdx.x + p) + (p == 0 ? 1 : 0)) * tile_rows + r;
        ml[k] = there ? work.ml[row] : make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int i = 0; i < COLS; ++i) {
          const int d = 4 * lane + 128 * i;
          v[i][k] = there && d < dim ? *reinterpret_cast<const float4*>(work.o + row * dim + d) : make_float4(0, 0, 0, 0);
        }
      }
      float most = top;
#pragma unroll
      for (int k = 0; k < JOIN_PIECES; ++k) most = fmaxf(most, ml[k].x);
      const float base = most == -INFINITY ? 0.0f : most, c = exp2_fast(top - base);
      l *= c;
#pragma unroll
      for (int i = 0; i < COLS; ++i) { o[i].x *= c; o[i].y *= c; o[i].z *= c; o[i].w *= c; }
      top = most;
#pragma unroll
      for (int k = 0; k < JOIN_PIECES; ++k) {
        if (p0 + k * shares >= u.pieces) break;
        const float w = exp2_fast(ml[k].x - base);
        l = fmaf(ml[k].y, w, l);
        minus |= ml[k].y < 0.0f;
#pragma unroll
        for (int i = 0; i < COLS; ++i) {
          o[i].x = fmaf(v[i][k].x, w, o[i].x); o[i].y = fmaf(v[i][k].y, w, o[i].y); o[i].z = fmaf(v[i][k].z, w, o[i].z); o[i].w = fmaf(v[i][k].w, w, o[i].w);
        }
      }
    }
    l = only_minus_inf(minus, top, l);
    if (shares > 1) {                                                     // the same for all warps: a block-wide exchange
      if (lane == 0) { s_m[warp] = top; s_l[warp] = l; }
#pragma unroll
      for (int i = 0; i < COLS; ++i) { const int d = 4 * lane + 128 * i; if (d < dim) *reinterpret_cast<float4*>(acc + warp * dim + d) = o[i]; }
      __syncthreads();
      if (part == 0 && live) {
        for (int w = 1; w < shares; ++w) top = fmaxf(top, s_m[warp + w]);
        const float base = top == -INFINITY ? 0.0f : top;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < COLS; ++i) o[i] = make_float4(0, 0, 0, 0);
        for (int w = 0; w < shares; ++w) {
          const float c = exp2_fast(s_m[warp + w] - base);
          l = fmaf(s_l[warp + w], c, l);
          minus |= s_l[warp + w] < 0.0f;
#pragma unroll
          for (int i = 0; i < COLS; ++i) {
            const int d = 4 * lane + 128 * i;
            if (d >= dim) continue;
            const float4 v = *reinterpret_cast<const float4*>(acc + (warp + w) * dim + d);
            o[i].x = fmaf(v.x, c, o[i].x); o[i].y = fmaf(v.y, c, o[i].y); o[i].z = fmaf(v.z, c, o[i].z); o[i].w = fmaf(v.w, c, o[i].w);
          }
        }
      }
      __syncthreads();
      l = only_minus_inf(minus, top, l);
    }
    if (live && part == 0) {
      const int g = u.row + r;
      const int64_t t = u.first + g / group;
      const int h = u.kv_head * group + g % group;
      const bool seen = !(top == -INFINITY && l == 0.0f);
      const float inv = inverse_sum(top, l);
      T* po = out.ptr + t * out.sn + h * out.sh;
#pragma unroll
      for (int i = 0; i < COLS; ++i) {
        const int d = 4 * lane + 128 * i;
        if (d >= dim) continue;
        const float4 v = make_float4(o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv);
        wrong |= !isfinite(v.x) || !isfinite(v.y) || !isfinite(v.z) || !isfinite(v.w);
        if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float4*>(po + d) = v;
        else *reinterpret_cast<uint2*>(po + d) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
      }
      if (lane == 0 && lse) lse[t * heads + h] = seen ? top * LN_2 + logf(l) : -INFINITY;
    }
  }
  if (wrong) raise_fault(fault, OP_PAGED_ATTN);
}

ojc_status u32_table(const char* op, const char* what, const ojc_tensor* t, int rank) {
  OJC_TRY(check_tensor(op, what, t));
  if (t->dtype != OJC_U32) return ojc_fail(OJC_ERR_DTYPE, op, std::string(what) + " is U32");
  if (t->rank != rank) return ojc_fail(OJC_ERR_SHAPE, op, std::string(what) + " has the wrong rank");
  return OJC_OK;
}

ojc_status attn_dims(const char* op, const ojc_tensor* q, const ojc_tensor* k_pages, AttnDims* a) {
  OJC_TRY(check_tensor(op, "q", q, false)); OJC_TRY(check_tensor(op, "k_pages", k_pages, false));
  if (q->rank != 3 || k_pages->rank != 4 || q->shape[2] != k_pages->shape[3]) return ojc_fail(OJC_ERR_SHAPE, op, "q [N, H, D]; k_pages, v_pages [P, page, Hkv, D]");
  *a = AttnDims{q->shape[0], q->shape[1], k_pages->shape[2], q->shape[2], k_pages->shape[0], k_pages->shape[1]};
  if (numel(q) == 0 || numel(k_pages) == 0) return ojc_fail(OJC_ERR_SHAPE, op, "empty tensor");
  if (a->heads % a->kv_heads != 0) return ojc_fail(OJC_ERR_SHAPE, op, "heads must be a multiple of KV heads");
  if (a->dim > 32 * MAX_HEAD_COLUMNS) return ojc_fail(OJC_ERR_UNSUPPORTED_HEAD_DIM, op, "head_dim above 256");
  if (a->tokens > INT32_MAX / a->heads || a->page > (1 << 24) || a->pages > (int64_t)OJC_NONE / a->page) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "extent out of range");
  if (q->dtype != k_pages->dtype || !is_float(q)) return ojc_fail(OJC_ERR_DTYPE, op, "q and the pages share F32 or BF16");
  return OJC_OK;
}

// The workspace: the split units, then (m, l) and outputs of two row tiles for each CTA.
constexpr uint64_t SPLIT_BYTES = (MAX_SHARES * sizeof(SplitUnit) + 255) / 256 * 256;
uint64_t attn_workspace(int64_t dim) { return SPLIT_BYTES + (uint64_t)2 * MAX_SHARE_ROWS * (dim + 2) * 4; }

// 16-byte rows: base and strides aligned
bool rows_aligned(const ojc_tensor* t, int axes) {
  const int64_t per = 16 / (int64_t)dtype_size(t->dtype);
  if ((uintptr_t)t->data & 15) return false;
  for (int i = 0; i < axes; ++i) if (t->stride[i] < 0 || t->stride[i] % per) return false;
  return true;
}

bool tiles_take(const ojc_tensor* q, const ojc_tensor* k, const ojc_tensor* v, const ojc_tensor* out, int64_t dim) {
  // tiles_by_dim's list
  const bool shape = dim == 32 || dim == 48 || dim == 64 || dim == 80 || dim == 96 || dim == 112 || dim == 128 ||
                     (q->dtype == OJC_BF16 && (dim == 160 || dim == 192 || dim == 256));
  return shape && rows_aligned(q, 2) && rows_aligned(k, 3) && rows_aligned(v, 3) && rows_aligned(out, 2);
}

// Launches a kernel with the shape S on tiles of `tile_rows` rows, and the join behind it.
template <class T, class S, class Kernel>
ojc_status shares_launch(const AttnCall& c, Kernel kernel, int tile_rows) {
  static PerDeviceFlag attr;                                                 // one for each S, and so for each kernel
  if (!attr[c.be->device]) {
    OJC_CUDA(c.be, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM), c.op);
    attr[c.be->device] = true;
  }
  const unsigned ctas = attn_ctas(c, S::CTAS_PER_SM * REDUCE_SMS, tile_rows, S::KEYS);
  const int group = (int)(c.a.heads / c.a.kv_heads);
  // queued while the kernel before still runs; it waits for that one's end before it looks at memory
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(TILE_WARPS * 32);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = c.be->stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  OJC_CUDA(c.be, cudaLaunchKernelEx(&cfg, kernel, rows_view<const T>(c.q), pages_view<const T>(c.k), pages_view<const T>(c.v), c.ix, rows_view<T>(c.out), c.lse, c.work, (int)c.a.heads, group,
                                    (int)c.a.kv_heads, c.scale, c.be->fault_dev), c.op);
  OJC_LAUNCHED(c.be, c.op);
  return c.ix.width * c.ix.page <= S::KEYS ? OJC_OK : paged_attention_join(c, ctas, tile_rows);   // no unit of one block is ever shared
}

template <class T, int D, int MW>
ojc_status tiles_launch(const AttnCall& c) {
  using S = TileShape<T, D, MW>;
  static_assert(S::CTAS_PER_SM * REDUCE_SMS <= MAX_SHARES && S::CTAS_PER_SM * REDUCE_SMS * 16 * MW <= MAX_SHARE_ROWS, "workspace");
  return shares_launch<T, S>(c, paged_attention_tiles_kernel<T, D, MW>, 16 * MW);
}

template <int D, int R>
ojc_status few_launch(const AttnCall& c) { return shares_launch<float, FewShape<D, R>>(c, paged_attention_few_kernel<D, R>, R); }

template <class T, int D>
ojc_status tiles_by_rows(const AttnCall& c) {
  // rows of a KV head in a request of average length: what the host knows without a readback
  const int64_t rows = (c.a.tokens + c.ix.batch - 1) / c.ix.batch * (c.a.heads / c.a.kv_heads);
  // More than 32 rows: tcgen05 (48 drafts over 4000 cached, 16 heads of 128: 55 us against 76; 100 drafts 61 against 117).
  // 17 to 32 rows, tiles here against tcgen05 in us, 31 drafts of 16 heads of 128: one request of 300, 4095 and 65536 cached 18/15, 40/28 and 135/107; 16 requests
  // 35/37, 99/103 and, of 16384, 291/249; 64 requests of 300 84/120, of 4095 316/320 (4 tokens of 32/4 heads: 64 of 300 31/38, of 16384 288/248). So tcgen05
  // while units do not queue behind one another, each paying for a tile of 128 rows that is mostly empty, and else where the tables are made for long
  // requests (how long they are is not known here). At 64 columns its copies are half as large and its empty rows count for more: one request of 131
  // thousand, 5 drafts of 32/8 heads, 85/102; 8 of 4095, 31 drafts, 46/60. (Ahead only for a single request of up to 16384: 36/32.)
  // Heads that leave columns of the operands empty, 63 rows: 68 us here against 63 at 96 columns and 4000 cached, 77 against 83 at 300 cached, 43 against 56 at
  // 32 columns; from 65 rows on a unit here is two row tiles (255 rows: 573 us against 208 at 96 columns, 282 against 180 at 32).
  const bool few_units = c.ix.batch * c.a.kv_heads <= REDUCE_SMS, long_tables = c.ix.width * c.ix.page >= 32768;
  const bool wide = D == 128 ? rows > 32 || (rows > 16 && (few_units || long_tables)) : rows > (D == 64 ? 32 : 64);
  if (D <= 128 && wide && paged_attention_tcgen05_takes(c)) return paged_attention_tcgen05(c, rows > 128 ? 2 : 1);
  if constexpr (std::is_same<T, float>::value && D % 32 == 0) {
    if (rows == 1) return few_launch<D, 1>(c);
    if (rows == 2) return few_launch<D, 2>(c);
    if (rows <= 4) return few_launch<D, 4>(c);
  }
  if (rows <= 16) return tiles_launch<T, D, 1>(c);
  if (rows <= 32) return tiles_launch<T, D, 2>(c);
  return tiles_launch<T, D, 4>(c);
}

template <class T>
ojc_status tiles_by_dim(const AttnCall& c) {
  switch (c.a.dim) {
    case 32: return tiles_by_rows<T, 32>(c);
    case 48: return tiles_by_rows<T, 48>(c);
    case 64: return tiles_by_rows<T, 64>(c);
    case 80: return tiles_by_rows<T, 80>(c);
    case 96: return tiles_by_rows<T, 96>(c);
    case 112: return tiles_by_rows<T, 112>(c);
    default: break;
  }
  if constexpr (std::is_same<T, bf16>::value) {
    if (c.a.dim == 160) return tiles_by_rows<T, 160>(c);
    if (c.a.dim == 192) return tiles_by_rows<T, 192>(c);
    if (c.a.dim == 256) return tiles_by_rows<T, 256>(c);
  }
  return tiles_by_rows<T, 128>(c);
}

}  // namespace

ojc_status paged_attention_join(const AttnCall& c, unsigned shares, int tile_rows) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(shares, std::max(1, tile_rows / (tile_rows <= 64 ? 4 : 8)));   // rows go round: any grid does, these leave a warp one row of most units
  cfg.blockDim = dim3(JOIN_WARPS * 32);
  cfg.dynamicSmemBytes = JOIN_WARPS * c.a.dim * 4;
  cfg.stream = c.be->stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const int group = (int)(c.a.heads / c.a.kv_heads), heads = (int)c.a.heads, dim = (int)c.a.dim;
  auto run = [&](auto t, auto kernel) {
    using T = decltype(t);
    return cudaLaunchKernelEx(&cfg, kernel, rows_view<T>(c.out), c.lse, c.work, heads, group, tile_rows, dim, c.be->fault_dev);
  };
  OJC_CUDA(c.be, c.q->dtype == OJC_F32 ? run(float(), paged_attention_join_kernel<float, 1>) : dim <= 128 ? run(bf16(), paged_attention_join_kernel<bf16, 1>)
                                       : run(bf16(), paged_attention_join_kernel<bf16, 2>), c.op);   // the F32 tiles end at 128 columns
  OJC_LAUNCHED(c.be, c.op);
  return OJC_OK;
}

extern "C" {

ojc_status ojc_paged_attention_workspace_bytes(ojc_backend* be, const ojc_tensor* q, const ojc_tensor* k_pages, uint64_t* bytes) {
  const char* op = "paged_attention_workspace_bytes";
  OJC_ALIVE(be, op);
  if (!bytes) return ojc_fail(OJC_ERR_BACKEND, op, "null out pointer");
  AttnDims a;
  OJC_TRY(attn_dims(op, q, k_pages, &a));
  *bytes = attn_workspace(a.dim);
  return OJC_OK;
}

ojc_status ojc_paged_attention_forward(ojc_backend* be, const ojc_tensor* q, const ojc_tensor* k_pages, const ojc_tensor* v_pages, const ojc_tensor* block_tables, const ojc_tensor* cached_lens,
                                       const ojc_tensor* starts, const ojc_tensor* masks, const ojc_tensor* positions, int64_t window, ojc_tensor* out, ojc_tensor* lse, void* workspace,
                                       uint64_t workspace_bytes) {
  const char* op = "paged_attention_forward";
  OJC_ALIVE(be, op);
  AttnDims a;
  OJC_TRY(attn_dims(op, q, k_pages, &a));
  OJC_TRY(check_tensor(op, "v_pages", v_pages, false)); OJC_TRY(check_tensor(op, "out", out, false));
  if (!same_shape(k_pages, v_pages) || !same_shape(q, out)) return ojc_fail(OJC_ERR_SHAPE, op, "q, out [N, H, D]; k_pages, v_pages [P, page, Hkv, D]");
  if (v_pages->dtype != q->dtype || out->dtype != q->dtype) return ojc_fail(OJC_ERR_DTYPE, op, "q, out and the pages share F32 or BF16");
  if (q->stride[2] != 1 || out->stride[2] != 1 || k_pages->stride[3] != 1 || v_pages->stride[3] != 1) return ojc_fail(OJC_ERR_SHAPE, op, "the head_dim axis must be contiguous");
  OJC_TRY(own_places(op, "out", out));
  OJC_TRY(u32_table(op, "block_tables", block_tables, 2)); OJC_TRY(u32_table(op, "cached_lens", cached_lens, 1)); OJC_TRY(u32_table(op, "starts", starts, 1));
  const int64_t batch = cached_lens->shape[0], width = block_tables->shape[1];
  if (batch == 0 || width == 0) return ojc_fail(OJC_ERR_SHAPE, op, "every dimension must be non-zero");
  if (block_tables->shape[0] != batch || starts->shape[0] != batch + 1) return ojc_fail(OJC_ERR_SHAPE, op, "block_tables [B, W], cached_lens [B], starts [B + 1]");
  if (batch > INT32_MAX || width > INT32_MAX / a.page) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "extent out of range");
  if (masks) {
    OJC_TRY(u32_table(op, "masks", masks, 2));
    if (masks->shape[0] != a.tokens || masks->shape[1] == 0 || masks->shape[1] > INT32_MAX / 32) return ojc_fail(OJC_ERR_SHAPE, op, "masks is [N, words]");
  }
  if (positions) {
    OJC_TRY(u32_table(op, "positions", positions, 1));
    if (positions->shape[0] != a.tokens) return ojc_fail(OJC_ERR_SHAPE, op, "positions is [N]");
  }
  if (window == 0) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "window must be at least 1");
  if (lse) {
    OJC_TRY(check_tensor(op, "lse", lse));
    if (lse->dtype != OJC_F32 || lse->rank != 2 || lse->shape[0] != a.tokens || lse->shape[1] != a.heads) return ojc_fail(OJC_ERR_SHAPE, op, "lse must be F32 [N, H]");
  }
  uint64_t need = 0;
  OJC_TRY(ojc_paged_attention_workspace_bytes(be, q, k_pages, &need));
  if (workspace) {
    if (workspace_bytes < need || ((uintptr_t)workspace & 255)) return ojc_fail(OJC_ERR_SHAPE, op, "the workspace is too small or not 256-byte aligned");
  }
  OJC_CUDA(be, cudaSetDevice(be->device), op);   // the caller's current device may be another backend's
  if (!workspace) {
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    OJC_CUDA(be, cudaStreamIsCapturing(be->stream, &capturing), op);
    if (capturing != cudaStreamCaptureStatusNone) return ojc_fail(OJC_ERR_UNSUPPORTED, op, "a call that is captured into a graph needs a workspace of its own");
    OJC_TRY(ojc_scratch(be, need, &workspace));
  }
  const PassIndex ix{(const uint32_t*)block_tables->data, (const uint32_t*)cached_lens->data, (const uint32_t*)starts->data, masks ? (const uint32_t*)masks->data : nullptr,
                     positions ? (const uint32_t*)positions->data : nullptr, (int)batch, masks ? (int)masks->shape[1] : 0, a.tokens, width, a.pages, (uint32_t)a.page,
                     (a.page & (a.page - 1)) ? -1 : __builtin_ctzll((unsigned long long)a.page), window < 0 ? 0 : window};
  const float scale = 1.0f / sqrtf((float)a.dim);
  float* lse_out = lse ? (float*)lse->data : nullptr;
  TileWork work;
  work.split = (SplitUnit*)workspace;
  work.ml = (float2*)((char*)workspace + SPLIT_BYTES);
  work.o = (float*)(work.ml + (size_t)2 * MAX_SHARE_ROWS);
  const AttnCall call{be, op, q, k_pages, v_pages, out, lse_out, ix, a, scale, work};
  const bool tiles = tiles_take(q, k_pages, v_pages, out, a.dim);
  return dispatch_float(op, q->dtype, [&](auto t) {
    using T = decltype(t);
    if (tiles) return tiles_by_dim<T>(call);
    paged_attention_rows_kernel<T><<<(unsigned)((a.tokens * a.heads + 3) / 4), 128, 4 * a.dim * 4, be->stream>>>(
        rows_view<const T>(q), pages_view<const T>(k_pages), pages_view<const T>(v_pages), ix, rows_view<T>(out), lse_out, (int)a.heads, (int)(a.heads / a.kv_heads), (int)a.dim,
        scale, be->fault_dev);
    OJC_LAUNCHED(be, op);
    return OJC_OK;
  });
}

}  // extern "C"
