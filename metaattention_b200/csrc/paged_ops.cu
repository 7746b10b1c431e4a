// Writing tokens into a paged cache and reading it back (sm_100a).  Both are bound by HBM, and by their launch where a call
// is one token a sequence: every value is read once and written once, in one kernel for keys and values.
//
//   append:  row (page, token % page) of each head = k or v of a new token, k turned by its position first where asked; into
//            16-bit pages as it is, into 8-bit ones as codes q = e4m3(x 2^-e) with the least e >= -127 that keeps |x| 2^-e <= 448.
//            A power of two loses nothing against a scale of amax / 448 (the codes are floating point, their relative step is
//            the same anywhere in the range), divides exactly and makes code * 2^e exact in 16 bits again.
//   read:    the rows of each sequence one after the other, code * 2^e rounded once to 16 bits, zeros behind the end.
// Measured: 4 x 2048 tokens of 8 heads of 128, turned, into 16-bit pages 15.0 us = 4.5 TB/s, ragged prompts of 6 sequences into 8-bit ones
// 9.3; 64 single tokens in 8 bits 3.8-4.1 us, of which 3.3 are the host's; 8 sequences of up to 8192 tokens out of 8 bits 68 us = 5.4 TB/s
// (a copy's rate: 6.55).
#include <algorithm>

#include <cuda_fp8.h>

#include "common_host.cuh"
#include "rotary.cuh"

namespace b200 {

struct PagedView {   // what the kernels need of AttnB200PagedCache
  uint8_t* kv[2];
  uint8_t* scale[2];
  long long stride[2][3], scale_stride[2][3];   // elements of (page, token, head)
  const int* table;
  long long table_stride;
  const int* lens;
  int pages, page_shift, heads, max_blocks, batch;
};

// Page of position `pos` of sequence b, or -1 where the table holds none.
__device__ __forceinline__ int page_of(const PagedView& c, int b, int pos) {
  const int block = pos >> c.page_shift;
  if (block >= c.max_blocks) return -1;
  const int page = c.table[b * c.table_stride + block];
  return page >= 0 && page < c.pages ? page : -1;
}

struct AppendParams {
  PagedView c;
  const uint16_t* in[2];
  long long is[2][3];       // (batch, seq, head)
  const int* cu;
  int seq, rows;            // rows: tokens of the call, batch * seq or the packed ones
  int lanes;                // groups of threads that share the heads of a token
  AttnB200Rotary rot;
};

// 16 values of a head as floats
template <bool kBf16>
__device__ __forceinline__ void unpack16(const uint4 lo, const uint4 hi, float (&x)[16]) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = unpack2<kBf16>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint32_t codes4(const float* x) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// A thread owns 16 columns of a token and walks its heads, so that a k's angles are made once; the D / 16 threads of a row
// are neighbours in a warp, for the row's largest magnitude.
constexpr int kAppendThreads = 128;

template <int D, bool kBf16, bool k8Bit>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kUnits = D / 16;
  const long long id = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int unit = threadIdx.x % kUnits;
  const long long group = id / kUnits;
  const long long row = group / p.lanes;
  const int lane = static_cast<int>(group - row * p.lanes);
  bool live = row < p.rows;
  int b = 0, t = static_cast<int>(row), pos = -1;
  if (live && p.cu == nullptr) {
    b = t / p.seq;
    t -= b * p.seq;
  }
  // columns of k: two pieces of 8 whose pairs this thread turns; v: 16 in a row
  int c0 = unit * 16, c1 = c0 + 8;
  const bool mine = unit < p.rot.dim / 16;   // its columns of k turn
  if (mine && !p.rot.interleaved) {
    c0 = unit * 8;
    c1 = c0 + p.rot.dim / 2;
  }
  const long long in_b = p.cu == nullptr ? b : 0;
  uint4 lo[2], hi[2];
  auto load = [&](int h, uint4 (&lo)[2], uint4 (&hi)[2]) {
    if (live && h < p.c.heads) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint16_t* src = p.in[w] + in_b * p.is[w][0] + t * p.is[w][1] + h * p.is[w][2];
        lo[w] = *reinterpret_cast<const uint4*>(src + (w == 0 ? c0 : unit * 16));
        hi[w] = *reinterpret_cast<const uint4*>(src + (w == 0 ? c1 : unit * 16 + 8));
      }
    }
  };
  lo[0] = lo[1] = hi[0] = hi[1] = make_uint4(0, 0, 0, 0);
  load(lane, lo, hi);   // on its way while the row's place and angles are found
  if (live) {
    if (p.cu == nullptr) {
      pos = p.c.lens[b] - p.seq + t;
    } else {
      int first = 0, behind = p.c.batch;   // the last sequence that begins at or before the row
      while (behind - first > 1) {
        const int mid = (first + behind) >> 1;
        if (p.cu[mid] <= t) first = mid; else behind = mid;
      }
      b = first;
      const int end = p.cu[b + 1];
      live = t >= p.cu[b] && t < end;
      pos = p.c.lens[b] - (end - t);
    }
  }
  live = live && pos >= 0;
  const int page = live ? page_of(p.c, b, pos) : -1;
  live = live && page >= 0;
  // the threads of a row agree, and rows that have no place stay for the shuffles
  const int in_page = pos & ((1 << p.c.page_shift) - 1);
  float2 cs[8];
  if (mine && live) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = rotary_cos_sin<false>(p.rot.turns[unit * 8 + i], pos, p.rot.magnitude, false);
  }
#pragma unroll 1
  for (int h0 = 0; h0 < p.c.heads; h0 += p.lanes) {
    const int h = h0 + lane;
    const bool on = live && h < p.c.heads;
    uint4 lo_next[2], hi_next[2];
    load(h + p.lanes, lo_next, hi_next);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int a0 = w == 0 ? c0 : unit * 16, a1 = w == 0 ? c1 : unit * 16 + 8;
      uint8_t* dst = p.c.kv[w] + (page * p.c.stride[w][0] + in_page * p.c.stride[w][1] + h * p.c.stride[w][2]) * (k8Bit ? 1 : 2);
      const bool turned = w == 0 && mine;
      if (!k8Bit && !turned) {
        if (on) {
          *reinterpret_cast<uint4*>(dst + 2 * a0) = lo[w];
          *reinterpret_cast<uint4*>(dst + 2 * a1) = hi[w];
        }
        lo[w] = lo_next[w];
        hi[w] = hi_next[w];
        continue;
      }
      float x[16];
      unpack16<kBf16>(lo[w], hi[w], x);
      if (turned) {
        if (p.rot.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) rotary_turn(x[2 * i], x[2 * i + 1], cs[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) rotary_turn(x[i], x[8 + i], cs[i]);
        }
      }
      if constexpr (!k8Bit) {
        if (on) {
          *reinterpret_cast<uint4*>(dst + 2 * a0) = make_uint4(pack2<kBf16>(x[0], x[1]), pack2<kBf16>(x[2], x[3]), pack2<kBf16>(x[4], x[5]), pack2<kBf16>(x[6], x[7]));
          *reinterpret_cast<uint4*>(dst + 2 * a1) = make_uint4(pack2<kBf16>(x[8], x[9]), pack2<kBf16>(x[10], x[11]), pack2<kBf16>(x[12], x[13]), pack2<kBf16>(x[14], x[15]));
        }
      } else {
        // the largest magnitude as the bits of a float, which order like the magnitudes do; NaN and infinities on top
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
        for (int d = 1; d < kUnits; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
        const bool finite = top < 0x7f800000u;
        const int e = max(code_exponent(top), -127);
        const int byte = finite ? e + 127 : 255;
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);   // 2^-e; e is at most 121
        if (on) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = finite ? x[i] * inv : __uint_as_float(0x7fffffffu);
          *reinterpret_cast<uint2*>(dst + a0) = make_uint2(codes4(x), codes4(x + 4));
          *reinterpret_cast<uint2*>(dst + a1) = make_uint2(codes4(x + 8), codes4(x + 12));
          if (unit == 0)
            p.c.scale[w][page * p.c.scale_stride[w][0] + in_page * p.c.scale_stride[w][1] + h * p.c.scale_stride[w][2]] = static_cast<uint8_t>(byte);
        }
      }
      lo[w] = lo_next[w];
      hi[w] = hi_next[w];
    }
  }
}

struct ReadParams {
  PagedView c;
  uint8_t* out[2];
  int max_len;
  long long items;   // batch * max_len * heads * D / 16
};

// 16 codes of a row times 2^(byte - 127), rounded to 16 bits.  In 32 bits the factor may be a subnormal (byte 0) and the
// product is exact but for the last rounding; a NaN code or byte 255 gives NaN.
template <bool kBf16>
__device__ __forceinline__ void widen16(const uint4 codes, int byte, uint4& lo, uint4& hi) {
  const float f = byte == 255 ? __uint_as_float(0x7fffffffu) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(byte) << 23);
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i / 2] >> (16 * (i % 2))), __NV_E4M3);
    const float2 x = __half22float2(__half2(h));
    r[i] = pack2<kBf16>(x.x * f, x.y * f);
  }
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}

template <int D, bool kBf16, bool k8Bit>
__global__ void __launch_bounds__(256) paged_read_kernel(const ReadParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kUnits = D / 16;
  for (long long id = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; id < p.items; id += static_cast<long long>(gridDim.x) * blockDim.x) {
    int unit, h, b, t;
    if (p.items <= 0x7fffffff) {   // 64-bit divisions cost ten times as much
      const int i = static_cast<int>(id), row = i / kUnits, token = row / p.c.heads;
      unit = i - row * kUnits;
      h = row - token * p.c.heads;
      b = token / p.max_len;
      t = token - b * p.max_len;
    } else {
      const long long row = id / kUnits, token = row / p.c.heads;
      unit = static_cast<int>(id - row * kUnits);
      h = static_cast<int>(row - token * p.c.heads);
      b = static_cast<int>(token / p.max_len);
      t = static_cast<int>(token - static_cast<long long>(b) * p.max_len);
    }
    const int page = t < p.c.lens[b] ? page_of(p.c, b, t) : -1;
    const int in_page = t & ((1 << p.c.page_shift) - 1);
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
      if (page >= 0) {
        const uint8_t* src = p.c.kv[w] + (page * p.c.stride[w][0] + in_page * p.c.stride[w][1] + h * p.c.stride[w][2] + unit * 16) * (k8Bit ? 1 : 2);
        if constexpr (k8Bit) {
          const int byte = p.c.scale[w][page * p.c.scale_stride[w][0] + in_page * p.c.scale_stride[w][1] + h * p.c.scale_stride[w][2]];
          widen16<kBf16>(*reinterpret_cast<const uint4*>(src), byte, lo, hi);
        } else {
          lo = reinterpret_cast<const uint4*>(src)[0];
          hi = reinterpret_cast<const uint4*>(src)[1];
        }
      }
      uint4* dst = reinterpret_cast<uint4*>(p.out[w] + id * 32);
      dst[0] = lo;
      dst[1] = hi;
    }
  }
}

// The cache as the kernels see it, or an error.  All strides are whole 16-byte pieces.
inline int view_cache(const AttnB200PagedCache& c, PagedView* v) {
  if (c.k == nullptr || c.v == nullptr || c.block_table == nullptr || c.seq_lens == nullptr) return ATTN_B200_E_INVALID_ARG;
  if (c.num_pages <= 0 || c.page_size <= 0 || c.heads_kv <= 0 || c.max_blocks <= 0 || c.batch <= 0) return ATTN_B200_E_INVALID_ARG;
  if (c.dtype != ATTN_B200_DTYPE_FP16 && c.dtype != ATTN_B200_DTYPE_BF16 && c.dtype != ATTN_B200_DTYPE_E4M3) return ATTN_B200_E_INVALID_ARG;
  const bool codes = c.dtype == ATTN_B200_DTYPE_E4M3;
  if (codes && (c.k_scale == nullptr || c.v_scale == nullptr)) return ATTN_B200_E_INVALID_ARG;
  if ((c.page_size & (c.page_size - 1)) != 0 || (c.head_dim != 64 && c.head_dim != 128)) return ATTN_B200_E_UNSUPPORTED;
  if (static_cast<long long>(c.max_blocks) * c.page_size > 0x7fffffff) return ATTN_B200_E_UNSUPPORTED;
  void* const kv[2] = {c.k, c.v};
  uint8_t* const scale[2] = {c.k_scale, c.v_scale};
  const int64_t* const strides[2] = {c.k_stride, c.v_stride};
  const int64_t* const scales[2] = {c.k_scale_stride, c.v_scale_stride};
  const int64_t extent[3] = {c.num_pages, c.page_size, c.heads_kv};
  for (int w = 0; w < 2; ++w) {
    v->kv[w] = static_cast<uint8_t*>(kv[w]);
    v->scale[w] = codes ? scale[w] : nullptr;
    if ((reinterpret_cast<uintptr_t>(kv[w]) & 15) != 0) return ATTN_B200_E_UNSUPPORTED;
    for (int i = 0; i < 3; ++i) {
      v->stride[w][i] = extent[i] > 1 ? strides[w][i] : 0;
      v->scale_stride[w][i] = codes && extent[i] > 1 ? scales[w][i] : 0;
      if (v->stride[w][i] % (codes ? 16 : 8) != 0) return ATTN_B200_E_UNSUPPORTED;
    }
  }
  v->table = c.block_table;
  v->table_stride = c.batch > 1 ? c.block_table_stride : 0;
  v->lens = c.seq_lens;
  v->pages = c.num_pages;
  v->page_shift = 0;
  while ((1 << v->page_shift) < c.page_size) ++v->page_shift;
  v->heads = c.heads_kv;
  v->max_blocks = c.max_blocks;
  v->batch = c.batch;
  return ATTN_B200_OK;
}

template <int D>
int launch_append(const AppendParams& p, bool bf16, bool codes, dim3 grid, cudaStream_t stream) {
  auto kernel = codes ? (bf16 ? paged_append_kernel<D, true, true> : paged_append_kernel<D, false, true>)
                      : (bf16 ? paged_append_kernel<D, true, false> : paged_append_kernel<D, false, false>);
  return launch_pdl(kernel, grid, dim3(kAppendThreads), 0, stream, p) ? ATTN_B200_OK : ATTN_B200_E_LAUNCH;
}

template <int D>
int launch_read(const ReadParams& p, bool bf16, bool codes, dim3 grid, cudaStream_t stream) {
  auto kernel = codes ? (bf16 ? paged_read_kernel<D, true, true> : paged_read_kernel<D, false, true>)
                      : (bf16 ? paged_read_kernel<D, true, false> : paged_read_kernel<D, false, false>);
  return launch_pdl(kernel, grid, dim3(256), 0, stream, p) ? ATTN_B200_OK : ATTN_B200_E_LAUNCH;
}

}  // namespace b200

extern "C" {

int attn_b200_paged_append(const AttnB200PagedAppendArgs* a, void* cuda_stream) {
  using namespace b200;
  if (a == nullptr || a->k == nullptr || a->v == nullptr || a->seq <= 0) return ATTN_B200_E_INVALID_ARG;
  AppendParams p = {};
  const int rc = view_cache(a->cache, &p.c);
  if (rc != ATTN_B200_OK) return rc;
  const bool codes = a->cache.dtype == ATTN_B200_DTYPE_E4M3, packed = a->cu_seqlens != nullptr;
  if (a->dtype != ATTN_B200_DTYPE_FP16 && a->dtype != ATTN_B200_DTYPE_BF16) return ATTN_B200_E_INVALID_ARG;
  if (!codes && a->dtype != a->cache.dtype) return ATTN_B200_E_UNSUPPORTED;
  if (a->rotary.dim < 0 || a->rotary.dim > a->cache.head_dim || (a->rotary.dim > 0 && a->rotary.turns == nullptr)) return ATTN_B200_E_INVALID_ARG;
  if (a->rotary.dim % 16 != 0) return ATTN_B200_E_UNSUPPORTED;
  const void* const in[2] = {a->k, a->v};
  const int64_t* const strides[2] = {a->k_stride, a->v_stride};
  const int extent[3] = {packed ? 1 : a->cache.batch, a->seq, a->cache.heads_kv};
  for (int w = 0; w < 2; ++w) {
    p.in[w] = static_cast<const uint16_t*>(in[w]);
    if ((reinterpret_cast<uintptr_t>(in[w]) & 15) != 0) return ATTN_B200_E_UNSUPPORTED;
    for (int i = 0; i < 3; ++i) {
      p.is[w][i] = extent[i] > 1 ? strides[w][i] : 0;
      if (p.is[w][i] % 8 != 0) return ATTN_B200_E_UNSUPPORTED;
    }
  }
  const long long rows = packed ? a->seq : static_cast<long long>(a->cache.batch) * a->seq;
  if (rows > 0x7fffffff) return ATTN_B200_E_UNSUPPORTED;
  p.cu = a->cu_seqlens;
  p.seq = a->seq;
  p.rows = static_cast<int>(rows);
  p.rot = a->rotary;
  const int sms = device_sms();
  if (sms <= 0) return ATTN_B200_E_LAUNCH;
  // heads are shared out evenly until there is work for two thirds of the chip's threads; with 90 to 96 registers 640 of an SM's are
  // resident at a time, so that a full call goes in up to 2.8 rounds of blocks (4 x 2048 tokens: 2048 blocks, 740 at a time)
  const long long one = rows * (a->cache.head_dim / 16), want = std::min<long long>(a->cache.heads_kv, (sms * 1365LL + one - 1) / one);
  const int rounds = static_cast<int>(a->cache.heads_kv / want);
  p.lanes = (a->cache.heads_kv + rounds - 1) / rounds;
  const long long blocks = (one * p.lanes + kAppendThreads - 1) / kAppendThreads;
  if (blocks > 0x7fffffff) return ATTN_B200_E_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool bf16 = a->dtype == ATTN_B200_DTYPE_BF16;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  return a->cache.head_dim == 64 ? launch_append<64>(p, bf16, codes, grid, stream) : launch_append<128>(p, bf16, codes, grid, stream);
}

int attn_b200_paged_read(const AttnB200PagedReadArgs* a, void* cuda_stream) {
  using namespace b200;
  if (a == nullptr || a->k == nullptr || a->v == nullptr || a->max_len <= 0) return ATTN_B200_E_INVALID_ARG;
  ReadParams p = {};
  const int rc = view_cache(a->cache, &p.c);
  if (rc != ATTN_B200_OK) return rc;
  const bool codes = a->cache.dtype == ATTN_B200_DTYPE_E4M3;
  if (a->dtype != ATTN_B200_DTYPE_FP16 && a->dtype != ATTN_B200_DTYPE_BF16) return ATTN_B200_E_INVALID_ARG;
  if (!codes && a->dtype != a->cache.dtype) return ATTN_B200_E_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15) != 0) return ATTN_B200_E_UNSUPPORTED;
  const int sms = device_sms();
  if (sms <= 0) return ATTN_B200_E_LAUNCH;
  p.out[0] = static_cast<uint8_t*>(a->k);
  p.out[1] = static_cast<uint8_t*>(a->v);
  p.max_len = a->max_len;
  p.items = static_cast<long long>(a->cache.batch) * a->max_len * a->cache.heads_kv * (a->cache.head_dim / 16);
  const long long blocks = std::min<long long>((p.items + 255) / 256, sms * 64LL);
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool bf16 = a->dtype == ATTN_B200_DTYPE_BF16;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  return a->cache.head_dim == 64 ? launch_read<64>(p, bf16, codes, grid, stream) : launch_read<128>(p, bf16, codes, grid, stream);
}

}  // extern "C"
