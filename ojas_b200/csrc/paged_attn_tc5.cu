// Paged attention for many rows to a KV head on the Blackwell tensor cores (tcgen05 + TMEM): trees of drafts times the query heads of a group, and
// pieces of prompts. BF16, head dims of the tiles up to 128: the operands have D = 64 or 128 columns, those behind the head's are zeros (TMA fills them
// in for K and V).
//
// A CTA walks its stretch of the line of work (paged_attn.cuh) in blocks of 128 keys with T = 1 or 2 tiles of 128 rows:
//   warps 0 .. 4T-1  softmax, one thread per row (= TMEM lane): at a unit's start the row of Q into shared memory (swizzled K-major operand) and zeros
//                    into its lane of O; per block the S row in one TMEM pass, exponentials in the log2 domain against a row scale that moves only
//                    when the maximum outgrew it by 2^8 (O is then rescaled in place), P packed to BF16 over the S columns (the A operand of the second
//                    product comes from tensor memory); at the end the normalised row, or the piece's (m, l, O)
//   warp 4T          TMA producer: every lane looks up one page of the block and fetches its rows as 64-column boxes (K and V on rings of stages);
//                    the next block's look-ups are under way meanwhile
//   warp 4T+1        issues S = Q K^T (M128 N128, K-major operands) and O += P V (V MN-major)
// With T 1, S has two buffers: the next block's S is computed under this block's softmax. With T 2 the tiles take turns: one tile's products run
// under the other's softmax.
//
// What bounds it: with one tile of 64 rows or so the cache's bytes (64 KB of K and V per block and SM); with two tiles of 128 columns the issue of the
// products: 32 MMAs of N 128 at 96 cycles each and four changes of accumulator at about 277, 4200 cycles a block, where the exponentials of both tiles at 16 a
// cycle take 2048. Over longer contexts a block costs 4060 cycles (16 trees of 128 drafts x 32/4 heads, 8000 -> 32000 cached: 880 to 930 TFLOP/s). Below
// that lie some 60 us that do not grow: 20 us of joining (a piece of 256 rows at either end of most CTAs' stretches), blocks with masks, first loads.
//
// V's rows behind a request's last place are whatever the page held, and no box is fetched for pages before its first one: the softmax threads overwrite
// all those rows with zeros before P V reads them. A place that some rows see and others do not may hold NaN or infinity: the blocks with masks are
// searched for such values; where there are any, each row adds its own share of them to O by itself and the operand's are replaced by zeros.
// Every mbarrier wait is bounded; on expiry the CTA raises the fault word, drains and frees its TMEM.
#include "paged_attn.cuh"
#include "tc_common.cuh"

namespace {

using namespace tc;

constexpr int KEYS = 128, ROWS = 128;
constexpr int SUB_BYTES = 128 * 128;                           // one 64-column sub-tile of 128 rows: 128-byte swizzled rows
constexpr uint32_t HI = desc_hi(1024);                         // 8-row groups 1024 bytes apart
constexpr uint32_t KSTEP = 32 >> 4, MNSTEP = 2048 >> 4, SUB16 = SUB_BYTES >> 4;
constexpr float RESCALE_STEP = 8.0f;                           // log2 units the row maximum may run ahead of the scale in use

template <int D, int T> struct Shape {
  static constexpr int NSUB = D / 64, TILE_BYTES = NSUB * SUB_BYTES, STAGES = D == 64 ? 4 : T == 1 ? 3 : 2;
  static constexpr int OFF_K = T * TILE_BYTES, OFF_V = OFF_K + STAGES * TILE_BYTES, OFF_BAR = OFF_V + STAGES * TILE_BYTES;
  static constexpr int QFULL = 0, KFULL = 2, KEMPTY = 6, VFULL = 10, VEMPTY = 14, SFULL = 18, PREADY = 20, PVFULL = 22, SYNC = 24, BARRIERS = 25;
  static constexpr int SMEM = OFF_BAR + 512;
  static constexpr int THREADS = T == 1 ? 192 : 384;              // T 2: whole warpgroups, so that registers can be shared out (two warps idle)
  static constexpr uint32_t COL_O = 256;
};

// tcgen05.mma with the A operand in tensor memory (lane = row, two bf16 per 32-bit column, 8 columns per K = 16 step)
__device__ __forceinline__ void umma_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, 1, 0;\n\tmov.b64 db, {%2, %3};\n\t"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
               ::"r"(tmem_d), "r"(tmem_a), "r"(b_lo), "r"(hi), "r"(idesc) : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}

struct TcArgs {
  RowsView<const bf16> q;
  RowsView<bf16> out;
  float* lse;
  PassIndex ix;
  TileWork work;
  int heads, group, kv_heads, dim;
  int k_heads_inside, v_heads_inside;   // tensor-map order: (D, Hkv, page, P) or (D, page, Hkv, P)
  int out_sectors;                      // out's rows start at 32-byte boundaries
  int box_rows;                         // rows of a page that one box holds: min(page, 128)
  float scale;
  uint32_t* fault;
};

// What a row sees of the 128 places from j on, as bits: the row's mask words are loaded together, then shifted to the places
struct RowMask { uint32_t local, from; bool live; };
__device__ __forceinline__ void seen_bits(const PassIndex& ix, const Request& r, const RowMask& row, uint32_t j, uint32_t (&bits)[4]) {
  const int32_t d0 = (int32_t)(j - r.cached);                  // the first place's number among the new tokens (below 0: cached)
  uint32_t m[5] = {0, 0, 0, 0, 0};
  if (ix.masks) {
    const uint32_t* p = ix.masks + (int64_t)(r.first + row.local) * ix.words;
    const int32_t w0 = d0 >> 5;
#pragma unroll
    for (int k = 0; k < 5; ++k) if (row.live && w0 + k >= 0 && w0 + k < ix.words) m[k] = p[w0 + k];
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int32_t d = d0 + 32 * k;                             // this word's first place
    auto below = [&](int64_t n) { return n <= d ? 0u : n >= (int64_t)d + 32 ? 0xffffffffu : (1u << (uint32_t)(n - d)) - 1u; };   // places with numbers under n
    uint32_t fresh = ix.masks ? __funnelshift_r(m[k], m[k + 1], d0 & 31) : below((int64_t)row.local + 1);
    fresh &= below(r.fresh) & ~below(0);
    uint32_t old = below(0);
    if (ix.window > 0) {
      old &= ~below((int64_t)row.from - r.cached);
      for (uint32_t left = fresh; left; left &= left - 1) {
        const uint32_t e = __ffs(left) - 1, n = (uint32_t)d + e;
        if ((ix.positions ? ix.positions[r.first + n] : r.cached + n) < row.from) fresh &= ~(1u << e);
      }
    }
    bits[k] = row.live ? old | fresh : 0u;
  }
}

// A store of 32 bytes: a whole sector to a thread, where a warp's threads write to rows of their own
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

// A warp's 32 rows of a Q tile, asynchronously into the swizzled operand at `tile` (row pointers from the lanes that own the rows). Not inlined: it runs once
// to a unit, and its addresses would cost the softmax loop its registers.
template <int D, bool WHOLE>
__device__ __noinline__ void fetch_q_rows(RowsView<const bf16> q, uint32_t first, int fresh, int hk, int row0, int group, int dim, uint32_t tile) {
  const int lane = threadIdx.x & 31, t0 = threadIdx.x & 96, n = row0 + t0 + lane;
  const uint64_t mine = n < fresh * group ? (uint64_t)(q.ptr + (int64_t)(first + (uint32_t)(n / group)) * q.sn + (int64_t)(hk * group + n % group) * q.sh) : 0;
  const int c = lane % (D / 8);
  const uint32_t dst = tile + (c >> 3) * SUB_BYTES + t0 * 128;
#pragma unroll 4
  for (int i = 0; i < D / 8; ++i) {
    const int row = i * (256 / D) + lane / (D / 8);
    const uint64_t from = __shfl_sync(0xffffffffu, mine, row);
    const uint32_t to = dst + row * 128 + (((c & 7) ^ (row & 7)) << 4);
    if (!WHOLE && 8 * c >= dim) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
    else if (from) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from + c * 16) : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

// WHOLE: the head has all D columns (asked at run time, a tree of 63 drafts took 2 % longer, most of it in the fetching of Q)
template <int D, int T, bool WHOLE>
__global__ void __launch_bounds__(Shape<D, T>::THREADS, 1)
paged_attention_tcgen05_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const TcArgs args) {
  const int dim = WHOLE ? D : args.dim;
  using C = Shape<D, T>;
  constexpr int STAGES = C::STAGES, TILE_ROWS = ROWS * T;
  constexpr uint32_t TILE16 = C::TILE_BYTES >> 4;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  __shared__ ShareScratch s_share;
  __shared__ uint32_t s_found[3], s_from[8];
  __shared__ Share<KEYS> s_line;
  const PassIndex& ix = args.ix;
  uint32_t* const fault = args.fault;
  auto bar = [&](int i) { return base + C::OFF_BAR + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + C::OFF_BAR + 8 * C::BARRIERS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (base & 1023u) { if (tid == 0) raise_fault(fault, OP_PAGED_ATTN); return; }   // the swizzled tiles need 1024-byte alignment (the whole CTA leaves)
  if (warp == 4 * T && lane == 0) {
    prefetch_tmap(&tm_k); prefetch_tmap(&tm_v);
    for (int i = 0; i < C::BARRIERS; ++i)
      mbar_init(bar(i), i < C::KFULL || (i >= C::PREADY && i < C::PVFULL) ? ROWS : i == C::SYNC ? TILE_ROWS : 1);
    *abort_flag = 0;
    s_found[0] = s_found[1] = s_found[2] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * T + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (tid == 0) args.work.split[blockIdx.x].pieces = 0;
  bool bad = false;
  int todo = 0;
  Cursor<KEYS> use;
  {
    Share<KEYS> share;
    if (find_share<KEYS, C::THREADS>(ix, args.group, TILE_ROWS, args.kv_heads, &s_share, &share, &bad)) {
      todo = share.todo;
      use = share.at;
      if (tid == 0) s_line = share;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // T 2: launched with 168 registers a thread (384 x 168 = 64,512); two softmax warpgroups of 216 and one of 72 take 128 x (2 x 216 + 72) = 64,512
  if (warp >= 4 * T) {
  if (T == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 4 * T) {
    // ------------------------------------------------------------------ TMA producer
    const uint32_t pg = (uint32_t)args.box_rows;
    uint32_t id = 0, off = 0;
    bool there = false;
    auto look_up = [&]() {
      const uint32_t last = use.r.cached + (uint32_t)use.r.fresh - 1, j = (uint32_t)(use.r.first_block + use.block) * KEYS + lane * pg;
      there = lane * pg < KEYS && j <= last && j + pg > first_place(ix, use.r.cached);
      if (there) {
        const uint32_t pi = ix.page_shift >= 0 ? j >> ix.page_shift : j / ix.page;
        off = j - pi * ix.page;
        id = ix.tables[(int64_t)use.b * ix.width + pi];
      }
    };
    if (todo > 0) look_up();
    for (int f = 0; f < todo; ++f) {
      const uint32_t s = f % STAGES, ph = ((f / STAGES) & 1) ^ 1;
      if (there && id >= ix.pages) { bad = true; id = 0; }
      const uint32_t now_id = id, now_off = off;
      const bool now = there;
      const int hk = use.hk;
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, now)) * pg * 128 * C::NSUB;
      use.step(ix, args.group, TILE_ROWS, args.kv_heads, &bad);
      if (f + 1 < todo) look_up();
      // a K stage is free once the S products that read it finished, a V stage once its P V products did
      bool ok = true;
      if (lane == 0) {
        ok = f < STAGES || mbar_wait(bar(C::KEMPTY + s), ph, fault, abort_flag);
        if (ok) mbar_expect_tx(bar(C::KFULL + s), bytes);
      }
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
      if (now) {
#pragma unroll
        for (int i = 0; i < C::NSUB; ++i)
          tma_load_4d(base + C::OFF_K + s * C::TILE_BYTES + i * SUB_BYTES + lane * pg * 128, &tm_k, bar(C::KFULL + s), 64 * i, args.k_heads_inside ? hk : (int)now_off,
                      args.k_heads_inside ? (int)now_off : hk, (int)now_id);
      }
      if (lane == 0) {
        ok = f < STAGES || mbar_wait(bar(C::VEMPTY + s), ph, fault, abort_flag);
        if (ok) mbar_expect_tx(bar(C::VFULL + s), bytes);
      }
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
      if (now) {
#pragma unroll
        for (int i = 0; i < C::NSUB; ++i)
          tma_load_4d(base + C::OFF_V + s * C::TILE_BYTES + i * SUB_BYTES + lane * pg * 128, &tm_v, bar(C::VFULL + s), 64 * i, args.v_heads_inside ? hk : (int)now_off,
                      args.v_heads_inside ? (int)now_off : hk, (int)now_id);
      }
      __syncwarp();
    }
  } else if (warp == 4 * T + 1) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      const uint32_t idesc_s = make_idesc(ROWS, KEYS, 0, 0), idesc_pv = make_idesc(ROWS, D, 0, 1);
      const uint32_t q_lo = desc_lo(base, 0), k_lo = desc_lo(base + C::OFF_K, 0), v_lo = desc_lo(base + C::OFF_V, SUB_BYTES);
      // The roles' loops together have to stay small for the instruction cache (the softmax warps waited for instructions more than for anything else). With T 1,
      // where the MMA thread has time, its products are rolled loops at one site each (trees of 63 67 -> 62 us); with T 2 it is on the way, and they are not
      // (213 us against 231).
      constexpr int UNROLL = T == 1 ? 2 : 8;
      int units = 0;                                             // units begun so far: their Q tiles' barrier phase
      auto issue_s = [&](int g, int f, bool first) -> bool {     // S of block f for tile g
        const uint32_t s = f % STAGES, col = T == 1 ? (f & 1) * 128 : g * 128;
        if (first && !mbar_wait(bar(C::QFULL + g), units & 1, fault, abort_flag)) return false;
        if (!mbar_wait(bar(C::KFULL + s), (f / STAGES) & 1, fault, abort_flag)) return false;
        fence_after();
#pragma unroll UNROLL
        for (uint32_t kk = 0; kk < D / 16; ++kk)
          umma_lh(tmem_base + col, q_lo + g * TILE16 + (kk >> 2) * SUB16 + (kk & 3) * KSTEP, k_lo + s * TILE16 + (kk >> 2) * SUB16 + (kk & 3) * KSTEP, HI, idesc_s, kk > 0);
        umma_commit(bar(C::SFULL + (T == 1 ? f & 1 : g)));
        if (g == T - 1) umma_commit(bar(C::KEMPTY + s));
        return true;
      };
      auto issue_pv = [&](int g, int f) -> bool {                // O += P V of block f for tile g
        const uint32_t s = f % STAGES, col = T == 1 ? (f & 1) * 128 : g * 128;
        if (!mbar_wait(bar(C::PREADY + (T == 1 ? f & 1 : g)), T == 1 ? (f >> 1) & 1 : f & 1, fault, abort_flag)) return false;
        if (!mbar_wait(bar(C::VFULL + s), (f / STAGES) & 1, fault, abort_flag)) return false;
        fence_after();
#pragma unroll UNROLL
        for (uint32_t kk = 0; kk < KEYS / 16; ++kk) umma_a_tmem(tmem_base + C::COL_O + g * D, tmem_base + col + kk * 8, v_lo + s * TILE16 + kk * MNSTEP, HI, idesc_pv);
        umma_commit(bar(C::PVFULL + g));
        if (g == T - 1) umma_commit(bar(C::VEMPTY + s));
        return true;
      };
      bool ok = true;
      if constexpr (T == 1) {
        for (int f = -1; f < todo && ok; ++f) {
          const bool begins = f < 0 || use.block + 1 == use.r.blocks, more = f + 1 < todo;   // the next block begins a unit (or the first one)
          if (f >= 0) use.step(ix, args.group, TILE_ROWS, args.kv_heads, &bad);
#pragma unroll 1
          for (int k = 0; k < 2 && ok; ++k) {
            // the next S goes first, into the other buffer, under this block's softmax; but before a unit's first S the last P V of the one before: its Q
            // comes from rows that first wait for that
            if ((k == 0) != begins) { if (more) ok = issue_s(0, f + 1, begins); }
            else if (f >= 0) { ok = issue_pv(0, f); units += begins; }
          }
        }
      } else {
        for (int g = 0; g < T && ok && todo > 0; ++g) ok = issue_s(g, 0, true);
        for (int f = 0; f < todo && ok; ++f) {
          const bool unit_ends = use.block + 1 == use.r.blocks, more = f + 1 < todo;
          use.step(ix, args.group, TILE_ROWS, args.kv_heads, &bad);
          if (unit_ends) {
            // the next unit's Q comes from rows that first wait for this unit's last O: both tiles' products before either's S
            for (int g = 0; g < T && ok; ++g) ok = issue_pv(g, f);
            ++units;
            for (int g = 0; g < T && ok && more; ++g) ok = issue_s(g, f + 1, true);
          } else {
            for (int g = 0; g < T && ok; ++g) {
              ok = issue_pv(g, f);
              if (ok && more) ok = issue_s(g, f + 1, false);       // over the P just consumed: the pipe runs the two in order
            }
          }
        }
      }
    }
  }
  } else {
    if (T == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------------ softmax + output rows
    const int g = warp >> 2, t = tid & 127;
    const uint32_t lane_base = tmem_base + ((uint32_t)((warp & 3) * 32) << 16), o_addr = lane_base + C::COL_O + g * D;
    const float sl2 = args.scale * LOG2_E;
    float m = 0.0f, l = 0.0f;
    bool have = false, any = false, wrong = false, ok = true;
    RowMask row = {0, 0, false};
    uint32_t from_most = 0;
    int votes = 0, syncs = 0, piece = 0;                          // piece: the block at which this CTA's piece of the unit begins
    auto sync_rows = [&]() -> bool {                              // all softmax threads, bounded
      mbar_arrive(bar(C::SYNC));
      return mbar_wait(bar(C::SYNC), syncs++ & 1, fault, abort_flag);
    };
    // The Q tile of a unit: a warp fetches its 32 rows together (row pointers from the lanes that own them), asynchronously, straight into the swizzled
    // operand. It is called as soon as the last S of the unit before is there, so the copies run under that unit's last softmax.
    auto fetch_q = [&](const Cursor<KEYS>& u) { fetch_q_rows<D, WHOLE>(args.q, u.r.first, u.r.fresh, u.hk, u.row_tile * TILE_ROWS + g * ROWS, args.group, dim, base + g * C::TILE_BYTES); };
    auto give_q = [&]() {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      fence_async_smem();
      mbar_arrive(bar(C::QFULL + g));
    };
    if (todo > 0) { fetch_q(use); give_q(); }
    for (int f = 0; f < todo && ok; ++f) {
      const uint32_t stage = f % STAGES;
      if (f == 0 || use.block == 0) {
        // ---- a new unit: this thread's row
        piece = f;
        const int n = use.row_tile * TILE_ROWS + g * ROWS + t;
        row.live = n < use.r.fresh * args.group;
        row.local = row.live ? (uint32_t)(n / args.group) : 0u;
        row.from = 0;
        m = l = 0.0f;
        have = any = false;
        if (ix.window > 0) {
          const uint32_t place = ix.positions ? ix.positions[use.r.first + row.local] : use.r.cached + row.local;
          if (row.live && place < use.r.cached) bad = true;
          row.from = place >= ix.window ? place - (uint32_t)ix.window + 1 : 0;
          const uint32_t most = __reduce_max_sync(0xffffffffu, row.live ? row.from : 0u);
          if (!sync_rows()) { ok = false; break; }                // the unit before has been read
          if (lane == 0) s_from[warp] = most;
          if (!sync_rows()) { ok = false; break; }
          from_most = 0;
#pragma unroll
          for (int w = 0; w < 4 * T; ++w) from_most = max(from_most, s_from[w]);
        }
        uint32_t zero[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) zero[e] = 0;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) tmem_st32(o_addr + c * 32, zero);
        tmem_wait_st();
      }
      const bool warp_live = __any_sync(0xffffffffu, row.live);
      const uint32_t s_addr = lane_base + (T == 1 ? (f & 1) * 128 : g * 128);
      const uint32_t j0 = (uint32_t)(use.r.first_block + use.block) * KEYS, places = use.r.cached + (uint32_t)use.r.fresh;
      const bool masked = j0 + KEYS > use.r.cached || j0 < from_most;
      const bool unit_done = use.block + 1 == use.r.blocks;
      bool poisoned = false;
      uint32_t bits[4];
      if (masked) {
        seen_bits(ix, use.r, row, j0, bits);
        // V's rows behind the last place, and those before the first that a row can see, become zeros; the others are searched for values that are not finite
        if (!mbar_wait(bar(C::VFULL + stage), (f / STAGES) & 1, fault, abort_flag)) { ok = false; break; }
        uint32_t odd = 0;
        const bool outside = j0 + t >= places || j0 + t < first_place(ix, use.r.cached);
        for (int part = g; part < C::NSUB; part += T) {           // T 2 and one sub-tile: the first tile's threads do it all
          uint8_t* v = smem_raw + C::OFF_V + stage * C::TILE_BYTES + part * SUB_BYTES + t * 128;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint4* w = reinterpret_cast<uint4*>(v + ((c ^ (t & 7)) << 4));
            if (outside) *w = make_uint4(0, 0, 0, 0);
            else {
              const uint4 x = *w;
              const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) odd |= (u[k] & 0x7f80u) == 0x7f80u || (u[k] & 0x7f800000u) == 0x7f800000u;
            }
          }
        }
        fence_async_smem();
        if (tid == 0) s_found[(votes + 1) % 3] = 0;               // last read before the vote before this one
        if (odd) atomicOr(&s_found[votes % 3], 1u);
        if (!sync_rows()) { ok = false; break; }
        poisoned = *(volatile uint32_t*)&s_found[votes % 3] != 0;
        ++votes;
      }
      if (!mbar_wait(bar(C::SFULL + (T == 1 ? f & 1 : g)), T == 1 ? (f >> 1) & 1 : f & 1, fault, abort_flag)) { ok = false; break; }
      fence_after();
      if (unit_done && f + 1 < todo) {                            // every S that reads this unit's Q is there
        Cursor<KEYS> next = use;
        next.step(ix, args.group, TILE_ROWS, args.kv_heads, &bad);
        fetch_q(next);
      }
      if (warp_live) {
        uint32_t r[KEYS];
#pragma unroll
        for (int c = 0; c < KEYS / 32; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&r[c * 32]));
        tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int w = 0; w < KEYS / 32; ++w) {
            any |= bits[w] != 0;
#pragma unroll
            for (int e = 0; e < 32; ++e) if (!(bits[w] >> e & 1u)) r[32 * w + e] = 0xff800000u;
          }
        } else any = true;
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < KEYS; e += 4) {
#pragma unroll
          for (int k = 0; k < 4; ++k) mx4[k] = fmaxf(mx4[k], __uint_as_float(r[e + k]));
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl2;
        const bool grow = mx != -INFINITY && (!have || mx > m + RESCALE_STEP);
        if (__any_sync(0xffffffffu, grow)) {
          const float m_new = !grow ? m : have ? fmaxf(m, mx) : mx, corr = have ? fast_exp2(m - m_new) : 1.0f;   // a row without a score yet has O = 0
          have |= grow;
          m = m_new;
          l *= corr;
          if (f != piece) {
            if (!mbar_wait(bar(C::PVFULL + g), (f - 1) & 1, fault, abort_flag)) { ok = false; break; }   // O of the blocks before has landed
            fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(o_addr + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st32(o_addr + c * 32, o);
            }
          }
        }
        float rs4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float p0 = fast_exp2(fmaf(__uint_as_float(r[c * 64 + 2 * e]), sl2, -m)), p1 = fast_exp2(fmaf(__uint_as_float(r[c * 64 + 2 * e + 1]), sl2, -m));
            rs4[e & 3] += p0 + p1;
            w[e] = pack2_bf16(p0, p1);                            // the operand's type; the sum above takes the weights unrounded
          }
          tmem_st32(s_addr + c * 32, w);
        }
        l += (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]);
        tmem_wait_st();
      }
      if (poisoned) {
        // ---- every row adds its own share of what is not finite, then the operand's are replaced by zeros
        if (f != piece) { if (!mbar_wait(bar(C::PVFULL + g), (f - 1) & 1, fault, abort_flag)) { ok = false; break; } fence_after(); }
        const uint8_t* v = smem_raw + C::OFF_V + stage * C::TILE_BYTES;
#pragma unroll 1
        for (int k = 0; k < KEYS && warp_live; ++k) {
          const bool sees = (k < 64 ? k < 32 ? bits[0] : bits[1] : k < 96 ? bits[2] : bits[3]) >> (k & 31) & 1u;
          const uint32_t pw = tmem_ld1(s_addr + (k >> 1));
          tmem_wait_ld();
          const float p = __uint_as_float((k & 1) ? pw & 0xffff0000u : pw << 16);
#pragma unroll 1
          for (int d = 0; d < D; ++d) {
            const uint32_t x = *reinterpret_cast<const uint16_t*>(v + (d >> 6) * SUB_BYTES + k * 128 + ((((d & 63) >> 3) ^ (k & 7)) << 4) + (d & 7) * 2);
            if ((x & 0x7f80u) != 0x7f80u) continue;               // the same for all threads
            uint32_t o = tmem_ld1(o_addr + d);
            tmem_wait_ld();
            if (sees) o = __float_as_uint(fmaf(p, __uint_as_float(x << 16), __uint_as_float(o)));
            asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(o_addr + d), "r"(o) : "memory");
            tmem_wait_st();
          }
        }
        if (!sync_rows()) { ok = false; break; }
        for (int part = g; part < C::NSUB; part += T) {
          uint16_t* w = reinterpret_cast<uint16_t*>(smem_raw + C::OFF_V + stage * C::TILE_BYTES + part * SUB_BYTES + t * 128);
#pragma unroll 1
          for (int e = 0; e < 64; ++e) if ((w[e] & 0x7f80u) == 0x7f80u) w[e] = 0;
        }
        fence_async_smem();
        if (!sync_rows()) { ok = false; break; }
      }
      // A parity tells two phases apart only for one who knows that the phase before has passed and the one behind it has not: with T 1 this block's S may
      // be there before the last block's P V, so whoever is about to wait for this block's P V waits for the last one's first, while P is still held back.
      if (T == 1 && f > 0 && (unit_done || f + 1 == todo) && !mbar_wait(bar(C::PVFULL + g), (f - 1) & 1, fault, abort_flag)) { ok = false; break; }
      fence_before();
      // T 1: a warp may be a block ahead of another (the next S is there early), so the two S buffers have a barrier each; two blocks ahead it cannot be,
      // since the S after next is issued behind this block's P V
      mbar_arrive(bar(C::PREADY + (T == 1 ? f & 1 : g)));
      if (unit_done && f + 1 < todo) give_q();                    // the next unit's first S runs while this one's rows are written

      // ---- the end of the unit, or of this CTA's piece of it
      if (unit_done || f + 1 == todo) {
        if (!mbar_wait(bar(C::PVFULL + g), f & 1, fault, abort_flag)) { ok = false; break; }
        fence_after();
        if (!have) l = only_minus_inf(any, -INFINITY, l);
        const bool starts = f - piece == use.block, whole = unit_done && starts;
        const int n = use.row_tile * TILE_ROWS + g * ROWS + t, h = use.hk * args.group + (row.live ? n % args.group : 0);
        const int64_t token = use.r.first + row.local;
        const float inv = inverse_sum(have ? m : -INFINITY, l);
        bf16* dst = args.out.ptr + token * args.out.sn + h * args.out.sh;
        const int64_t at = (int64_t)(2 * blockIdx.x + (starts ? 1 : 0)) * TILE_ROWS + g * ROWS + t;
        if (warp_live) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(o_addr + c * 32, o);
            tmem_wait_ld();
            if (row.live && whole) {
#pragma unroll
              for (int i = 0; i < 32; i += 16) {
                if (!WHOLE && c * 32 + i >= dim) break;
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const float x = any ? __uint_as_float(o[i + 2 * e]) * inv : 0.0f, y = any ? __uint_as_float(o[i + 2 * e + 1]) * inv : 0.0f;
                  wrong |= !isfinite(x) || !isfinite(y);
                  w[e] = pack2_bf16(x, y);
                }
                if (args.out_sectors) store32(dst + c * 32 + i, w);
                else { uint4* d = reinterpret_cast<uint4*>(dst + c * 32 + i); d[0] = make_uint4(w[0], w[1], w[2], w[3]); d[1] = make_uint4(w[4], w[5], w[6], w[7]); }
              }
            } else if (row.live) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                if (!WHOLE && c * 32 + i >= dim) break;
                const uint32_t w[8] = {o[i], o[i + 1], o[i + 2], o[i + 3], o[i + 4], o[i + 5], o[i + 6], o[i + 7]};
                store32(args.work.o + at * dim + c * 32 + i, w);
              }
            }
          }
          if (row.live && whole && args.lse) args.lse[token * args.heads + h] = any ? m * LN_2 + logf(l) : -INFINITY;
          if (row.live && !whole) args.work.ml[at] = make_float2(have ? m : -INFINITY, l);
        }
        if (!unit_done && starts && tid == 0)
          args.work.split[blockIdx.x] = SplitUnit{(int)(s_line.of_block(s_line.begin + f - use.block + use.r.blocks - 1) - blockIdx.x) + 1, use.hk, use.row_tile * TILE_ROWS,
                                                    min(TILE_ROWS, use.r.fresh * args.group - use.row_tile * TILE_ROWS), use.r.first};
      }
      use.step(ix, args.group, TILE_ROWS, args.kv_heads, &bad);
    }
    if (wrong && !bad) raise_fault(fault, OP_PAGED_ATTN);
  }
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
  if (*abort_flag) __nanosleep(200000);
  fence_before();
  __syncthreads();
  if (warp == 4 * T + 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Pages as a 4-D tensor map whose boxes are `rows` places x 64 columns of one head of one page (one 128-byte swizzle span per row)
ojc_status pages_map(const AttnCall& c, CUtensorMap* map, const ojc_tensor* t, bool heads_inside, uint32_t rows) {
  const cuuint64_t page_bytes = (cuuint64_t)t->stride[1] * 2, head_bytes = (cuuint64_t)t->stride[2] * 2;
  const cuuint64_t page = (cuuint64_t)t->shape[1], kv_heads = (cuuint64_t)t->shape[2];
  cuuint64_t dims[4] = {(cuuint64_t)t->shape[3], heads_inside ? kv_heads : page, heads_inside ? page : kv_heads, (cuuint64_t)t->shape[0]};
  cuuint64_t strides[3] = {heads_inside ? head_bytes : page_bytes, heads_inside ? page_bytes : head_bytes, (cuuint64_t)t->stride[0] * 2};
  cuuint32_t box[4] = {64, heads_inside ? 1u : rows, heads_inside ? rows : 1u, 1}, steps[4] = {1, 1, 1, 1};
  const CUresult r = ((EncodeTiledFn)c.be->tmap_encode)(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, t->data, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return ojc_fail(OJC_ERR_BACKEND, c.op, "cuTensorMapEncodeTiled refused the pages (code " + std::to_string((int)r) + ")");
  return OJC_OK;
}

template <int D, int T, bool WHOLE>
ojc_status launch(const AttnCall& c) {
  using S = Shape<D, T>;
  static PerDeviceFlag attr;
  if (!attr[c.be->device]) {
    // the register shares of T 2 add up to 168 for each of the launched threads: with fewer their second half would wait for ever
    cudaFuncAttributes made;
    OJC_CUDA(c.be, cudaFuncGetAttributes(&made, paged_attention_tcgen05_kernel<D, T, WHOLE>), c.op);
    if (T == 2 && made.numRegs < 168) return ojc_fail(OJC_ERR_BACKEND, c.op, "the kernel was built with fewer registers than its warps share out");
    OJC_CUDA(c.be, cudaFuncSetAttribute(paged_attention_tcgen05_kernel<D, T, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM), c.op);
    attr[c.be->device] = true;
  }
  TcArgs args{rows_view<const bf16>(c.q), rows_view<bf16>(c.out), c.lse, c.ix, c.work, (int)c.a.heads, (int)(c.a.heads / c.a.kv_heads), (int)c.a.kv_heads, (int)c.a.dim,
              c.k->stride[2] < c.k->stride[1], c.v->stride[2] < c.v->stride[1],
              (uintptr_t)c.out->data % 32 == 0 && c.out->stride[0] % 16 == 0 && c.out->stride[1] % 16 == 0, (int)std::min<int64_t>(c.a.page, KEYS), c.scale, c.be->fault_dev};
  CUtensorMap mk, mv;
  OJC_TRY(pages_map(c, &mk, c.k, args.k_heads_inside, args.box_rows));
  OJC_TRY(pages_map(c, &mv, c.v, args.v_heads_inside, args.box_rows));
  static_assert(REDUCE_SMS * ROWS * T <= MAX_SHARE_ROWS && REDUCE_SMS <= MAX_SHARES, "workspace");
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  const unsigned ctas = attn_ctas(c, REDUCE_SMS, ROWS * T, KEYS);
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = c.be->stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  OJC_CUDA(c.be, cudaLaunchKernelEx(&cfg, paged_attention_tcgen05_kernel<D, T, WHOLE>, mk, mv, args), c.op);
  OJC_LAUNCHED(c.be, c.op);
  return c.ix.width * c.ix.page <= KEYS ? OJC_OK : paged_attention_join(c, ctas, ROWS * T);   // no unit of one block is ever shared
}

}  // namespace

bool paged_attention_tcgen05_takes(const AttnCall& c) {
  if (!c.be->tmap_encode || c.q->dtype != OJC_BF16 || c.a.dim > 128 || c.a.dim % 16) return false;
  if (c.a.page % 8 || (KEYS % c.a.page && c.a.page % KEYS)) return false;    // boxes of whole 8-row swizzle groups that tile a block
  for (const ojc_tensor* t : {c.k, c.v})
    for (int i = 0; i < 3; ++i) if (t->stride[i] <= 0 || t->stride[i] >= 1ll << 38) return false;   // what a tensor map can say
  return true;
}

ojc_status paged_attention_tcgen05(const AttnCall& c, int tiles) {
  if (c.a.dim == 64) return tiles == 1 ? launch<64, 1, true>(c) : launch<64, 2, true>(c);
  if (c.a.dim == 128) return tiles == 1 ? launch<128, 1, true>(c) : launch<128, 2, true>(c);
  if (c.a.dim < 64) return tiles == 1 ? launch<64, 1, false>(c) : launch<64, 2, false>(c);
  return tiles == 1 ? launch<128, 1, false>(c) : launch<128, 2, false>(c);
}
