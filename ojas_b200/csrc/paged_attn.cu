// Attention of new tokens (one decoded token, a tree of drafts, a piece of a prompt) over a paged KV cache.
//
// out_i = sum_j p_ij v_j, p_ij = exp(s_ij - max_j s_ij) / sum, s_ij = q_i . k_j / sqrt(D) over the places j that row i sees: the cached ones inside
// its window, and of its request's new tokens those in its ancestor mask (or up to itself). One pass over the keys with a running maximum and sum.
#include "dispatch.cuh"
#include "paged.cuh"

namespace {

constexpr int MAXI = 8;  // head_dim <= 256: each lane owns columns lane + 32 i

struct PassIndex {       // the pass's index tables (all U32)
  const uint32_t *tables, *cached, *starts, *masks, *positions;
  int batch, words;
  int64_t tokens, width, pages;
  uint32_t page;
  int64_t window;        // 0: none
};

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
  if (t >= ix.tokens || t >= ix.starts[ix.batch]) return;
  const int b = request_of(ix.starts, ix.batch, (uint32_t)t);
  const uint32_t first = ix.starts[b], end = ix.starts[b + 1], local = (uint32_t)t - first;
  const int64_t cached = ix.cached[b], room = ix.width * ix.page;
  bool bad = first > t || end <= t || end > ix.tokens || cached + (end - first) > room;
  const int64_t fresh = bad ? 0 : end - first, total = bad ? 0 : cached + fresh;
  const int64_t place = ix.positions ? ix.positions[t] : cached + local;
  const int64_t low = ix.window > 0 ? place - ix.window : -1;   // keys at positions above `low` are in the window
  float* qs = sm + warp * dim;
  const T* qp = q.ptr + t * q.sn + h * q.sh;
  for (int d = lane; d < dim; d += 32) qs[d] = ldf(qp, d);
  __syncwarp();
  float m = -INFINITY, l = 0.0f, o[MAXI];
  bool any = false;
#pragma unroll
  for (int i = 0; i < MAXI; ++i) o[i] = 0.0f;
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
    // every score -inf so far (or NaN among them): the sum shows it below
    const float corr = m_new == -INFINITY ? 1.0f : expf(m - m_new);
    const float p = sees ? expf(s - m_new) : 0.0f;
    l = l * corr + warp_sum(p);
#pragma unroll
    for (int i = 0; i < MAXI; ++i) o[i] *= corr;
    for (uint32_t left = seen; left; left &= left - 1) {
      const int jj = __ffs(left) - 1;
      const float pj = __shfl_sync(0xffffffffu, p, jj);
      const T* pv = vp.ptr + __shfl_sync(0xffffffffu, at, jj) + hk * vp.sh;
#pragma unroll
      for (int i = 0; i < MAXI; ++i) { const int d = lane + 32 * i; if (d < dim) o[i] = fmaf(pj, ldf(pv, d), o[i]); }
    }
    m = m_new;
  }
  bool wrong = any && !(isfinite(l) && l > 0.0f && isfinite(m));
  const float inv = any ? 1.0f / l : 0.0f;
  T* po = out.ptr + t * out.sn + h * out.sh;
#pragma unroll
  for (int i = 0; i < MAXI; ++i) {
    const int d = lane + 32 * i;
    if (d < dim) { const float v = any ? o[i] * inv : 0.0f; wrong |= !isfinite(v); stf(po, d, v); }
  }
  if (lane == 0 && lse) lse[t * heads + h] = any ? m + logf(l) : -INFINITY;
  if (bad) raise_fault(fault, OP_PAGED_RANGE);
  else if (wrong) raise_fault(fault, OP_PAGED_ATTN);
}

ojc_status u32_table(const char* op, const char* what, const ojc_tensor* t, int rank) {
  OJC_TRY(check_tensor(op, what, t));
  if (t->dtype != OJC_U32) return ojc_fail(OJC_ERR_DTYPE, op, std::string(what) + " is U32");
  if (t->rank != rank) return ojc_fail(OJC_ERR_SHAPE, op, std::string(what) + " has the wrong rank");
  return OJC_OK;
}

struct AttnDims { int64_t tokens, heads, kv_heads, dim, pages, page; };

ojc_status attn_dims(const char* op, const ojc_tensor* q, const ojc_tensor* k_pages, AttnDims* a) {
  OJC_TRY(check_tensor(op, "q", q, false)); OJC_TRY(check_tensor(op, "k_pages", k_pages, false));
  if (q->rank != 3 || k_pages->rank != 4 || q->shape[2] != k_pages->shape[3]) return ojc_fail(OJC_ERR_SHAPE, op, "q [N, H, D]; k_pages, v_pages [P, page, Hkv, D]");
  *a = AttnDims{q->shape[0], q->shape[1], k_pages->shape[2], q->shape[2], k_pages->shape[0], k_pages->shape[1]};
  if (numel(q) == 0 || numel(k_pages) == 0) return ojc_fail(OJC_ERR_SHAPE, op, "empty tensor");
  if (a->heads % a->kv_heads != 0) return ojc_fail(OJC_ERR_SHAPE, op, "heads must be a multiple of KV heads");
  if (a->dim > 32 * MAXI) return ojc_fail(OJC_ERR_UNSUPPORTED_HEAD_DIM, op, "head_dim above 256");
  if (a->tokens > INT32_MAX / a->heads || a->page > (1 << 24) || a->pages > (int64_t)OJC_NONE / a->page) return ojc_fail(OJC_ERR_OUT_OF_RANGE, op, "extent out of range");
  if (q->dtype != k_pages->dtype || !is_float(q)) return ojc_fail(OJC_ERR_DTYPE, op, "q and the pages share F32 or BF16");
  return OJC_OK;
}

}  // namespace

extern "C" {

ojc_status ojc_paged_attention_workspace_bytes(ojc_backend* be, const ojc_tensor* q, const ojc_tensor* k_pages, uint64_t* bytes) {
  const char* op = "paged_attention_workspace_bytes";
  OJC_ALIVE(be, op);
  if (!bytes) return ojc_fail(OJC_ERR_BACKEND, op, "null out pointer");
  AttnDims a;
  OJC_TRY(attn_dims(op, q, k_pages, &a));
  *bytes = 256;
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
  } else {
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    OJC_CUDA(be, cudaStreamIsCapturing(be->stream, &capturing), op);
    if (capturing != cudaStreamCaptureStatusNone) return ojc_fail(OJC_ERR_UNSUPPORTED, op, "a call that is captured into a graph needs a workspace of its own");
    OJC_TRY(ojc_scratch(be, need, &workspace));
  }
  const PassIndex ix{(const uint32_t*)block_tables->data, (const uint32_t*)cached_lens->data, (const uint32_t*)starts->data, masks ? (const uint32_t*)masks->data : nullptr,
                     positions ? (const uint32_t*)positions->data : nullptr, (int)batch, masks ? (int)masks->shape[1] : 0, a.tokens, width, a.pages, (uint32_t)a.page,
                     window < 0 ? 0 : window};
  const float scale = 1.0f / sqrtf((float)a.dim);
  float* lse_out = lse ? (float*)lse->data : nullptr;
  return dispatch_float(op, q->dtype, [&](auto t) {
    using T = decltype(t);
    paged_attention_rows_kernel<T><<<(unsigned)((a.tokens * a.heads + 3) / 4), 128, 4 * a.dim * 4, be->stream>>>(
        rows_view<const T>(q), pages_view<const T>(k_pages), pages_view<const T>(v_pages), ix, rows_view<T>(out), lse_out, (int)a.heads, (int)(a.heads / a.kv_heads), (int)a.dim,
        scale, be->fault_dev);
    OJC_LAUNCHED(be, op);
    return OJC_OK;
  });
}

}  // extern "C"
