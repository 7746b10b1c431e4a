// Rotary positions of q and k in one launch, forward and backward (the opposite angle): y = x with the first `dim` columns of
// every head turned by position.  Bound by HBM: every value is read and written once.  4 x 4096 tokens of 40 heads of 128, there
// and back: 123 us = 5.5 TB/s; in 32 bits 217-222 us, 6.1 TB/s.
//
// A thread owns a unit of a token -- 16 bytes from each half of the turning columns, or 32 bytes of interleaved pairs -- and
// walks the heads of q and k with it, so that the angles, cosines and sines of its pairs are made once for all heads and
// nothing is read but the tensors, the positions and dim / 2 frequencies.  Columns that do not turn are units of their own.
#include <algorithm>

#include "common_host.cuh"
#include "rotary.cuh"

namespace b200 {

struct RotaryParams {
  const void* x[2];
  void* y[2];
  const void* positions;
  long long xs[2][3], ys[2][3], ps[2];
  int heads0, heads, seq, dim, head_dim, pos64, inverse;
  int units, copies;        // turning and copied units of a head
  int lanes;                // threads that share the heads of a (token, unit)
  long long threads;        // tokens * lanes * (units + copies)
  const uint64_t* turns;
  float magnitude;
};

constexpr int kRotaryThreads = 128;   // of a CTA; 256: 125 us where these take 122 (4 x 4096 x 40 x 128, there and back)

template <class T, int V>
struct alignas(sizeof(T) * V) Piece {
  T e[V];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// V: values of a piece (a unit is two of them), 16 bytes where dims, strides and addresses are multiples of it, else one value
template <class T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const long long id = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (id >= p.threads) return;
  const int per = p.units + p.copies;
  int unit, lane, b, t;
  if (p.threads <= 0x7fffffff) {   // 64-bit divisions cost ten times as much
    const int i = static_cast<int>(id), rest = i / per, token = rest / p.lanes;
    unit = i - rest * per;
    lane = rest - token * p.lanes;
    b = token / p.seq;
    t = token - b * p.seq;
  } else {
    const long long rest = id / per, token = rest / p.lanes;
    unit = static_cast<int>(id - rest * per);
    lane = static_cast<int>(rest - token * p.lanes);
    b = static_cast<int>(token / p.seq);
    t = static_cast<int>(token - static_cast<long long>(b) * p.seq);
  }
  const bool turns = unit < p.units;
  // columns of the unit's two pieces
  int c0, c1;
  bool second = true;
  if (!turns) {
    c0 = p.dim + (unit - p.units) * 2 * V;
    c1 = c0 + V;
    second = c1 < p.head_dim;
  } else if (kInterleaved) {
    c0 = unit * 2 * V;
    c1 = c0 + V;
  } else {
    c0 = unit * V;
    c1 = c0 + p.dim / 2;
  }
  using P = Piece<T, V>;
  const long long x_at[2] = {b * p.xs[0][0] + t * p.xs[0][1], b * p.xs[1][0] + t * p.xs[1][1]};
  const long long y_at[2] = {b * p.ys[0][0] + t * p.ys[0][1], b * p.ys[1][0] + t * p.ys[1][1]};
  P u, v;
  auto load = [&](int h, P& u, P& v) {
    const int w = h < p.heads0 ? 0 : 1;
    const T* x = static_cast<const T*>(p.x[w]) + x_at[w] + (w == 0 ? h : h - p.heads0) * p.xs[w][2];
    u = *reinterpret_cast<const P*>(x + c0);
    if (second) v = *reinterpret_cast<const P*>(x + c1);
  };
  // A head is on its way while the angles are made, and the next one while a head is turned: 126 -> 121 us of that case.
  // (Four heads at once take the registers of half of the warps: 170.)
  load(lane, u, v);
  float2 cs[V];
  if (turns) {
    long long pos = t;
    if (p.positions != nullptr) {
      const long long at = b * p.ps[0] + t * p.ps[1];
      pos = p.pos64 ? static_cast<const long long*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) cs[i] = rotary_cos_sin<sizeof(T) == 4>(p.turns[unit * V + i], pos, p.magnitude, p.inverse != 0);
  }
#pragma unroll 1
  for (int h = lane; h < p.heads; h += p.lanes) {
    P u_next, v_next;
    if (h + p.lanes < p.heads) load(h + p.lanes, u_next, v_next);
    if (turns) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        T& a = kInterleaved ? (2 * i < V ? u.e[(2 * i) % V] : v.e[(2 * i) % V]) : u.e[i];
        T& c = kInterleaved ? (2 * i + 1 < V ? u.e[(2 * i + 1) % V] : v.e[(2 * i + 1) % V]) : v.e[i];
        float fa = to_float(a), fc = to_float(c);
        rotary_turn(fa, fc, cs[i]);
        a = from_float<T>(fa);
        c = from_float<T>(fc);
      }
    }
    const int w = h < p.heads0 ? 0 : 1;
    T* y = static_cast<T*>(p.y[w]) + y_at[w] + (w == 0 ? h : h - p.heads0) * p.ys[w][2];
    *reinterpret_cast<P*>(y + c0) = u;
    if (second) *reinterpret_cast<P*>(y + c1) = v;
    u = u_next;
    v = v_next;
  }
}

template <class T, int V>
int launch_rotary(RotaryParams& p, bool interleaved, bool copy, long long tokens, int sms, cudaStream_t stream) {
  p.units = p.dim / (2 * V);
  p.copies = copy ? (p.head_dim - p.dim + 2 * V - 1) / (2 * V) : 0;
  const long long per = p.units + p.copies;
  if (per == 0) return ATTN_B200_OK;
  // heads are shared out until the chip is full (two thirds of its threads), down to one head a thread; beyond that up to ten
  // heads share one set of angles
  const long long one = tokens * per, want = (sms * 1365LL + one - 1) / one;
  p.lanes = static_cast<int>(std::min<long long>(p.heads, std::max<long long>(want, (p.heads + 9) / 10)));
  p.threads = one * p.lanes;
  const long long blocks = (p.threads + kRotaryThreads - 1) / kRotaryThreads;
  if (blocks > 0x7fffffff) return ATTN_B200_E_UNSUPPORTED;
  auto kernel = interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>;
  return launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kRotaryThreads), 0, stream, p) ? ATTN_B200_OK : ATTN_B200_E_LAUNCH;
}

}  // namespace b200

extern "C" int attn_b200_rotary(const AttnB200RotaryArgs* a, void* cuda_stream) {
  using namespace b200;
  if (a == nullptr || a->x[0] == nullptr || a->y[0] == nullptr || (a->x[1] != nullptr && a->y[1] == nullptr)) return ATTN_B200_E_INVALID_ARG;
  const AttnB200Rotary& r = a->rotary;
  if (a->batch <= 0 || a->seq <= 0 || a->head_dim <= 0 || a->heads[0] <= 0 || (a->x[1] != nullptr && a->heads[1] <= 0)) return ATTN_B200_E_INVALID_ARG;
  if (r.dim <= 0 || r.dim % 2 != 0 || r.dim > a->head_dim || r.turns == nullptr) return ATTN_B200_E_INVALID_ARG;
  if (a->dtype != ATTN_B200_DTYPE_FP16 && a->dtype != ATTN_B200_DTYPE_BF16 && a->dtype != ATTN_B200_DTYPE_FP32) return ATTN_B200_E_INVALID_ARG;
  if (static_cast<long long>(a->heads[0]) + a->heads[1] > 0x7fffff) return ATTN_B200_E_UNSUPPORTED;
  const int sms = device_sms();
  if (sms <= 0) return ATTN_B200_E_LAUNCH;
  const int n = a->x[1] != nullptr ? 2 : 1;
  const int size = a->dtype == ATTN_B200_DTYPE_FP32 ? 4 : 2, wide = 16 / size;
  RotaryParams p = {};
  bool whole = a->head_dim % wide == 0 && r.dim % (2 * wide) == 0, copy = false;
  for (int w = 0; w < n; ++w) {
    p.x[w] = a->x[w];
    p.y[w] = a->y[w];
    whole = whole && (reinterpret_cast<uintptr_t>(a->x[w]) & 15) == 0 && (reinterpret_cast<uintptr_t>(a->y[w]) & 15) == 0;
    if (a->x[w] != a->y[w]) copy = copy || a->head_dim > r.dim;
    const int extent[3] = {a->batch, a->seq, a->heads[w]};
    for (int i = 0; i < 3; ++i) {
      p.xs[w][i] = extent[i] > 1 ? a->x_stride[w][i] : 0;   // the stride of an axis of one entry says nothing
      p.ys[w][i] = extent[i] > 1 ? a->y_stride[w][i] : 0;
      if (a->x[w] == a->y[w] && p.xs[w][i] != p.ys[w][i]) return ATTN_B200_E_INVALID_ARG;
      whole = whole && p.xs[w][i] % wide == 0 && p.ys[w][i] % wide == 0;
    }
  }
  p.positions = a->positions;
  p.ps[0] = a->pos_stride[0];
  p.ps[1] = a->pos_stride[1];
  p.heads0 = a->heads[0];
  p.heads = a->heads[0] + (n == 2 ? a->heads[1] : 0);
  p.seq = a->seq;
  p.dim = r.dim;
  p.head_dim = a->head_dim;
  p.pos64 = a->positions_64;
  p.inverse = a->inverse;
  p.turns = r.turns;
  p.magnitude = r.magnitude;
  const long long tokens = static_cast<long long>(a->batch) * a->seq;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  const bool inter = r.interleaved != 0;
#define ATTN_B200_ROTARY(T) \
  return whole ? launch_rotary<T, 16 / sizeof(T)>(p, inter, copy, tokens, sms, stream) : launch_rotary<T, 1>(p, inter, copy, tokens, sms, stream)
  if (a->dtype == ATTN_B200_DTYPE_FP32) { ATTN_B200_ROTARY(float); }
  if (a->dtype == ATTN_B200_DTYPE_BF16) { ATTN_B200_ROTARY(__nv_bfloat16); }
  ATTN_B200_ROTARY(__half);
#undef ATTN_B200_ROTARY
}
