// Attention of new tokens over a paged cache: what a call is, its plan, and the merge of units that several CTAs share.  The
// kernels are in paged_tokens.cu and paged_chunk.cu, the list of work they walk in paged_common.cuh.
#include <cstring>

#include "paged_common.cuh"

namespace b200 {

// Adds up the partial rows of the units that were cut: o = sum_i exp(lse_i - lse) part_i.  Block x looks after the unit that
// begins in CTA x and goes on in others, a thread 8 columns of a row.
constexpr int kMergeRows = 16;   // of a block

template <int D, bool kBf16>
__global__ void __launch_bounds__(2 * D) paged_merge_kernel(const __grid_constant__ PagedParams p, int ctas) {
  pdl_launch_dependents();
  const int c_lo = blockIdx.x, row = blockIdx.y * kMergeRows + threadIdx.x % kMergeRows, col = threadIdx.x / kMergeRows * 8;
  const int t = row / kPgTile, r = row - t * kPgTile;   // query tile and its row
  const int g = p.head_major ? r / p.tile_pos : r % p.group, qi = p.head_major ? r % p.tile_pos : r / p.group;
  pdl_wait();
  const int4 cut = __ldcg(p.cut + c_lo);
  if (cut.w < 0 || row >= p.rows || r >= p.tile_pos * p.group) return;
  const int tok = cut.z * p.per_tile + t * p.tile_pos + qi, head = cut.y * p.group + g;
  // rows as the kernel in front of this one counted them: those of p.cu may go backwards
  const int2 seq_rows = __ldcg(p.cut_rows + c_lo);
  const int row0 = seq_rows.x, fresh = seq_rows.y;
  if (tok >= fresh) return;
  const int c_hi = min(cut.w, ctas - 1);
  float mx = -INFINITY, den = 0.0f, acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
  // four shares at a time, their statistics and rows loaded together, added up against a running maximum
#pragma unroll 1
  for (int c0 = c_lo; c0 <= c_hi; c0 += 4) {
    float l[4];
    float4 x[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = c0 + k <= c_hi;
      const int c = in ? c0 + k : c_hi;
      const long long slot = (2LL * c + (c == c_lo ? 1 : 0)) * p.rows;
      const float4* src = reinterpret_cast<const float4*>(p.part_o + slot * D) + col / 4 * p.rows + row;
      l[k] = __ldcg(p.part_lse + slot + row);
      x[k][0] = __ldcg(src);
      x[k][1] = __ldcg(src + p.rows);
      if (!in) l[k] = -INFINITY;
    }
    // shares in which the row saw nothing count nothing; NaN passes through: the maxima ignore it, its weight does not
    const float m = fmaxf(mx, fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])));
    const float old = mx == -INFINITY ? 0.0f : __expf(mx - m);
    den *= old;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= old;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (l[k] == -INFINITY) continue;
      const float wgt = __expf(l[k] - m);
      const float v[8] = {x[k][0].x, x[k][0].y, x[k][0].z, x[k][0].w, x[k][1].x, x[k][1].y, x[k][1].z, x[k][1].w};
      den += wgt;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = fmaf(wgt, v[e], acc[e]);
    }
    mx = m;
  }
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  const long long at = row0 + tok;
  uint16_t* orow = static_cast<uint16_t*>(p.o) + (p.cu != nullptr ? 0 : cut.x * p.o_sb) + at * p.o_ss + head * p.o_sh + col;
  *reinterpret_cast<uint4*>(orow) = make_uint4(pack2<kBf16>(acc[0] * inv, acc[1] * inv), pack2<kBf16>(acc[2] * inv, acc[3] * inv),
                                               pack2<kBf16>(acc[4] * inv, acc[5] * inv), pack2<kBf16>(acc[6] * inv, acc[7] * inv));
  if (col == 0 && p.lse != nullptr)
    p.lse[(p.cu != nullptr ? static_cast<long long>(head) : static_cast<long long>(cut.x) * p.heads + head) * p.seq + at] = den == 0.0f ? -INFINITY : mx + logf(den);
}

int paged_merge(const AttnB200PagedAttnArgs* a, const PagedPlan& d, const PagedParams& p, cudaStream_t stream) {
  if (d.ctas == 1 || d.whole) return ATTN_B200_OK;   // nothing was cut
  const bool bf16 = a->dtype == ATTN_B200_DTYPE_BF16;
  auto kernel = a->cache.head_dim == 64 ? (bf16 ? paged_merge_kernel<64, true> : paged_merge_kernel<64, false>)
                                        : (bf16 ? paged_merge_kernel<128, true> : paged_merge_kernel<128, false>);
  return launch_pdl(kernel, dim3(d.ctas, (d.rows + kMergeRows - 1) / kMergeRows), dim3(2 * a->cache.head_dim), 0, stream, p, d.ctas) ? ATTN_B200_OK : ATTN_B200_E_LAUNCH;
}

constexpr int kPgFew = 32;       // rows of a unit of paged_tokens.cu
constexpr int kPgWholeTiles = 4; // KV tiles of a unit that is not cut: the merge behind it costs 3 us, a tile 0.8

inline int plan_paged(const AttnB200PagedAttnArgs* a, int sms, PagedPlan* d) {
  const AttnB200PagedCache& c = a->cache;
  if (c.batch <= 0 || c.heads_kv <= 0 || a->heads <= 0 || a->seq <= 0 || a->heads % c.heads_kv != 0) return ATTN_B200_E_INVALID_ARG;
  if (c.num_pages <= 0 || c.page_size <= 0 || c.max_blocks <= 0) return ATTN_B200_E_INVALID_ARG;
  if (c.head_dim != 64 && c.head_dim != 128) return ATTN_B200_E_UNSUPPORTED;
  if (c.page_size < 8 || (c.page_size & (c.page_size - 1)) != 0) return ATTN_B200_E_UNSUPPORTED;
  if (c.batch > kPgMaxBatch || a->heads > 65535) return ATTN_B200_E_UNSUPPORTED;
  d->group = a->heads / c.heads_kv;
  if (d->group > kPgTile) return ATTN_B200_E_UNSUPPORTED;
  const bool packed = a->cu_seqlens != nullptr;
  const long long all = packed ? a->seq : static_cast<long long>(c.batch) * a->seq;   // new tokens
  if (all > 0x7fffffff / 2) return ATTN_B200_E_UNSUPPORTED;
  // A few rows a sequence: their own kernel (16 sequences of 16384, 20 rows: 168 us where paged_chunk.cu takes 183, 64 columns 97 for
  // 177, 8 bits 165 for 281).  How many a packed sequence has the host does not know; where they are less than two on average a
  // longer one among them costs a walk over its keys for each kPgFew of its rows (64 sequences of up to 8192, single tokens: 208 us
  // for 230, 8 bits 212 for 352; 63 and one of 60 tokens: 229 for 291, 274 for 469).
  d->few = d->group <= kPgFew && (packed ? a->seq < 2LL * c.batch : static_cast<long long>(d->group) * a->seq <= kPgFew);
  // packed tokens, most of them alone: the narrower score tile
  const int most_rows = !d->few ? kPgTile : packed && d->group <= kPgFew / 2 ? kPgFew / 2 : kPgFew;
  d->tile_pos = std::min(most_rows / d->group, a->seq);
  d->per_tile = d->few || a->seq <= d->tile_pos ? d->tile_pos : 2 * d->tile_pos;
  d->rows = (d->per_tile > d->tile_pos ? kPgTile : 0) + d->tile_pos * d->group;
  const long long most_kv = static_cast<long long>(c.max_blocks) * c.page_size;
  if (most_kv > 0x3fffffff) return ATTN_B200_E_UNSUPPORTED;
  const long long q_tiles = packed ? a->seq / d->per_tile + c.batch : static_cast<long long>(c.batch) * ((a->seq + d->per_tile - 1) / d->per_tile);
  long long unit_tiles = (most_kv + kPgTile - 1) / kPgTile;   // at most
  if (a->window > 0) unit_tiles = std::min<long long>(unit_tiles, (static_cast<long long>(a->window) + d->per_tile - 2) / kPgTile + 2);
  d->whole = unit_tiles <= kPgWholeTiles;
  const long long most = q_tiles * c.heads_kv * (d->whole ? 1 : unit_tiles + kPgUnitCost);
  if (most > 0x3fffffff) return ATTN_B200_E_UNSUPPORTED;
  d->ctas = static_cast<int>(std::min<long long>(sms, most));
  const long long parts = d->whole ? 0 : 2LL * d->ctas * d->rows;
  d->off_lse = parts * c.head_dim * 4;
  d->off_cut = (d->off_lse + parts * 4 + 15) / 16 * 16;
  d->off_rows = d->off_cut + 16LL * d->ctas;
  d->bytes = (d->off_rows + 8LL * d->ctas + 255) / 256 * 256;
  return ATTN_B200_OK;
}

// Tensor map over a pool of codes [page][row][head][dim] of bytes: a box is a row of one head by `box_rows` rows of a page.
inline int encode_codes_map(CUtensorMap* tm, CoordOrder* order, const void* base, const AttnB200PagedCache& c, const int64_t stride[3], int box_rows,
                            CUtensorMapSwizzle swizzle) {
  TensorMapEncodeTiledFn enc = tensor_map_encoder();
  if (enc == nullptr) return ATTN_B200_E_LAUNCH;
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0) return ATTN_B200_E_UNSUPPORTED;
  const cuuint64_t size[3] = {(cuuint64_t)c.num_pages, (cuuint64_t)c.page_size, (cuuint64_t)c.heads_kv};
  int idx[3] = {0, 1, 2};
  for (int i = 0; i < 3; ++i)
    if (size[i] > 1 && (stride[i] <= 0 || stride[i] % 16 != 0)) return ATTN_B200_E_UNSUPPORTED;
  std::stable_sort(idx, idx + 3, [&](int x, int y) {   // extent-1 dimensions last: their strides say nothing
    if ((size[x] <= 1) != (size[y] <= 1)) return size[y] <= 1;
    return size[x] > 1 && stride[x] < stride[y];
  });
  cuuint64_t gdim[4] = {(cuuint64_t)c.head_dim, 1, 1, 1}, gstride[3];
  cuuint32_t box[4] = {(cuuint32_t)c.head_dim, 1, 1, 1}, estr[4] = {1, 1, 1, 1};
  cuuint64_t next = c.head_dim;
  int pos[3];
  for (int i = 0; i < 3; ++i) {
    const int w = idx[i];
    gdim[i + 1] = size[w];
    gstride[i] = size[w] > 1 ? (cuuint64_t)stride[w] : next;
    next = std::max(next, gstride[i] * size[w]);
    pos[w] = i + 1;
    if (w == 1) box[i + 1] = (cuuint32_t)box_rows;
  }
  order->pos_b = pos[0];
  order->pos_s = pos[1];
  order->pos_h = pos[2];
  const CUresult r = enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), gdim, gstride, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ATTN_B200_OK : ATTN_B200_E_UNSUPPORTED;
}

int paged_setup(const AttnB200PagedAttnArgs* a, const PagedPlan& d, int* status, PagedParams* out, PagedMaps* m) {
  const AttnB200PagedCache& c = a->cache;
  PagedParams& p = *out;
  std::memset(&p, 0, sizeof(p));
  std::memset(m, 0, sizeof(*m));
  const bool packed = a->cu_seqlens != nullptr, codes = c.dtype == ATTN_B200_DTYPE_E4M3;
  const int D = c.head_dim, box = std::min(c.page_size, kPgTile);
  int rc;
  if (codes && d.few) {   // queries are read and split into parts
    const bool aligned = (reinterpret_cast<uintptr_t>(a->q) & 15) == 0;
    const int extent[3] = {packed ? 1 : c.batch, a->seq, a->heads};
    for (int i = 0; i < 3; ++i) {
      if (!aligned || (extent[i] > 1 && a->q_stride[i] % 8 != 0)) return ATTN_B200_E_UNSUPPORTED;
      p.qs[i] = extent[i] > 1 ? a->q_stride[i] : 0;
    }
    rc = ATTN_B200_OK;
  } else {
    rc = encode_rows_map(&m->q, &p.oq, a->q, a->dtype, D, packed ? 1 : c.batch, a->seq, a->heads, a->q_stride, d.tile_pos, d.group);
    p.head_major = p.oq.pos_s < p.oq.pos_h ? 1 : 0;
  }
  if (rc != ATTN_B200_OK) return rc;
  if (codes) {   // keys are an operand as they come for a few rows; else they are widened first, as values are
    rc = encode_codes_map(&m->k, &p.ok, c.k, c, c.k_stride, box, !d.few ? CU_TENSOR_MAP_SWIZZLE_NONE : D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    if (rc == ATTN_B200_OK) rc = encode_codes_map(&m->v, &p.ov, c.v, c, c.v_stride, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    const int pool[3] = {c.num_pages, c.page_size, c.heads_kv};
    for (int i = 0; i < 3; ++i) {
      p.scale_stride[0][i] = pool[i] > 1 ? c.k_scale_stride[i] : 0;
      p.scale_stride[1][i] = pool[i] > 1 ? c.v_scale_stride[i] : 0;
    }
  } else {
    rc = encode_rows_map(&m->k, &p.ok, c.k, a->dtype, D, c.num_pages, c.page_size, c.heads_kv, c.k_stride, box);
    if (rc == ATTN_B200_OK) rc = encode_rows_map(&m->v, &p.ov, c.v, a->dtype, D, c.num_pages, c.page_size, c.heads_kv, c.v_stride, box);
  }
  if (rc != ATTN_B200_OK) return rc;
  p.q = static_cast<const uint16_t*>(a->q);
  p.scale8[0] = c.k_scale;
  p.scale8[1] = c.v_scale;
  p.o = a->o;
  p.lse = a->lse;
  p.o_sb = packed ? 0 : a->o_stride[0];
  p.o_ss = a->o_stride[1];
  p.o_sh = a->o_stride[2];
  p.cu = a->cu_seqlens;
  p.lens = c.seq_lens;
  p.table = c.block_table;
  p.table_stride = c.batch > 1 ? c.block_table_stride : 0;
  p.batch = c.batch;
  p.heads = a->heads;
  p.heads_kv = c.heads_kv;
  p.group = d.group;
  p.seq = a->seq;
  p.per_tile = d.per_tile;
  p.rows = d.rows;
  p.tile_pos = d.tile_pos;
  p.max_blocks = c.max_blocks;
  p.pages = c.num_pages;
  while ((1 << p.page_shift) < c.page_size) ++p.page_shift;
  while ((1 << p.box_shift) < box) ++p.box_shift;
  p.causal = a->causal != 0;
  p.window = std::min(a->window, 0x3fffffff);   // no sequence is longer, and a position less it stays in 32 bits
  p.whole = d.whole ? 1 : 0;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_lse = reinterpret_cast<float*>(ws + d.off_lse);
  p.cut = reinterpret_cast<int4*>(ws + d.off_cut);
  p.cut_rows = reinterpret_cast<int2*>(ws + d.off_rows);
  p.status = status;
  p.scale = a->scale;
  return ATTN_B200_OK;
}

}  // namespace b200

extern "C" {

int64_t attn_b200_paged_workspace_bytes(const AttnB200PagedAttnArgs* a) {
  if (a == nullptr) return -1;
  const int sms = b200::device_sms();
  if (sms <= 0) return -1;
  b200::PagedPlan d;
  return b200::plan_paged(a, sms, &d) == ATTN_B200_OK ? d.bytes : -1;
}

int attn_b200_paged_attention(const AttnB200PagedAttnArgs* a, void* cuda_stream) {
  if (a == nullptr || a->q == nullptr || a->o == nullptr) return ATTN_B200_E_INVALID_ARG;
  const AttnB200PagedCache& c = a->cache;
  if (c.k == nullptr || c.v == nullptr || c.block_table == nullptr || c.seq_lens == nullptr) return ATTN_B200_E_INVALID_ARG;
  if (a->dtype != ATTN_B200_DTYPE_FP16 && a->dtype != ATTN_B200_DTYPE_BF16) return ATTN_B200_E_INVALID_ARG;
  const bool codes = c.dtype == ATTN_B200_DTYPE_E4M3;
  if (codes ? c.k_scale == nullptr || c.v_scale == nullptr : c.dtype != a->dtype) return ATTN_B200_E_INVALID_ARG;
  if (!(a->scale > 0.0f) || a->scale > 3.4028235e38f || a->window < 0 || (a->window > 0 && !a->causal)) return ATTN_B200_E_INVALID_ARG;
  const int sms = b200::device_sms();
  if (sms <= 0) return ATTN_B200_E_LAUNCH;
  b200::PagedPlan d;
  const int rc = b200::plan_paged(a, sms, &d);
  if (rc != ATTN_B200_OK) return rc;
  if ((reinterpret_cast<uintptr_t>(a->o) & 15) != 0) return ATTN_B200_E_UNSUPPORTED;
  const int extent[3] = {a->cu_seqlens != nullptr ? 1 : c.batch, a->seq, a->heads};
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && a->o_stride[i] % 8 != 0) return ATTN_B200_E_UNSUPPORTED;
  if (a->workspace == nullptr || a->workspace_bytes < d.bytes || (reinterpret_cast<uintptr_t>(a->workspace) & 15) != 0) return ATTN_B200_E_WORKSPACE;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ATTN_B200_E_LAUNCH;
  int* status = b200::device_status_word(dev);
  if (status == nullptr) return ATTN_B200_E_LAUNCH;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  return d.few ? b200::launch_paged_tokens(a, d, stream, status) : b200::launch_paged_chunk(a, d, stream, status);
}

}  // extern "C"
