// Attention of new tokens over a paged cache for sm_100a: softmax(scale * Q.K^T).V with grouped KV heads, for single tokens
// and for chunks of prompts, all sequences of a batch in one launch; 16-bit pages, or 8-bit ones with a scale for each row.
//
// One list of work: a unit is a tile of 128 query rows -- the (position, head of the group) pairs of one KV head of one
// sequence, so that K and V are read once for the group -- with the 128-row KV tiles that any of its rows sees.  The KV
// tiles of all units, in order, are cut into one equal share per SM: a long context against a single token is split over the
// chip, the units of a prompt are spread over it evenly whatever their lengths, and a share walks its units with every ring
// and barrier phase carried across them.  A unit that lies in one share writes its rows; the others leave fp32 partial rows
// that a second small kernel adds up.  Each CTA counts the list itself from the lengths on the device, so a captured call
// follows them.
// Pages are fetched by TMA, a box of up to 128 rows of one page, its index from the block table; boxes without a row that
// counts are not fetched.  V rows behind the last key of a unit, or in front of its window, hold anything: they are zeroed in
// shared memory (0 * NaN would reach the row), the scores there are masked.
#include <cstring>

#include "../../include/attn_b200.h"
#include "common_host.cuh"
#include "functors.cuh"
#include "parallel_launch.cuh"

namespace b200 {

constexpr int kPgTile = 128;       // KV rows of a tile
constexpr int kPgMaxBatch = 1024;  // sequences of a call
constexpr int kPgConvWarps = 8;    // 8-bit caches: warps that widen codes

struct PagedParams {
  void* o;
  float* lse;
  long long o_sb, o_ss, o_sh;
  const int* cu;                 // packed rows, or null
  const int* lens;
  const int* table;
  long long table_stride;
  int batch, heads, heads_kv, group, seq;
  int per_tile;                  // query positions of a tile
  int rows, rows_pad;            // group * per_tile; padded to a multiple of 8
  int q_bufs, q_bytes;
  int head_major;                // row = g * per_tile + i (1) or i * group + g (0): the order the tensor map delivers
  int max_blocks, page_shift, pages, box_shift;   // rows of a box: min(page, 128)
  int causal, window;
  const uint8_t* scale[2];       // 8-bit caches: exponents of k and v
  long long scale_stride[2][3];
  float* part_o;                 // [2 * CTAs][rows][D]
  float* part_lse;               // [2 * CTAs][rows]
  int4* cut;                     // [CTAs] sequence, KV head, query tile and last CTA of the unit that begins in a CTA and goes on, or w = -1
  CoordOrder oq, ok, ov;
  int* status;
  FunctorArgs fa;
};

enum PagedWaitSite {
  kPgQFull = 101, kPgQEmpty, kPgKFull, kPgKEmpty, kPgVFull, kPgVEmpty, kPgSFull, kPgPReady, kPgODone, kPgStats, kPgOFree, kPgRawFull, kPgRawEmpty,
  kPgScaleFull, kPgScaleEmpty
};

template <int D, bool k8Bit>
struct PagedSmem {
  static constexpr int kThreads = 320 + (k8Bit ? 32 + 32 * kPgConvWarps : 0);
  static constexpr int kTileBytes = kPgTile * D * 2;
  static constexpr int kRawBytes = kPgTile * D;
  static constexpr int kStagesK = k8Bit ? 2 : D == 128 ? 3 : 6, kStagesV = k8Bit ? 2 : D == 128 ? 2 : 5;
  static constexpr int kRaw = k8Bit ? (D == 128 ? 3 : 10) : 0;       // tiles of codes, keys and values in turn
  static constexpr int kScales = k8Bit ? 3 : 0;                     // tiles of factors
  // query tiles; an MMA reads 128 rows from a tile's start whatever its rows, so what follows must be shared memory too
  static constexpr int kOffK = D * 256;
  static constexpr int kOffV = kOffK + kStagesK * kTileBytes;
  static constexpr int kOffRaw = kOffV + kStagesV * kTileBytes;
  static constexpr int kOffScale = kOffRaw + kRaw * kRawBytes;      // uint32 [kScales][2][128]
  static constexpr int kOffBar = kOffScale + kScales * 2 * kPgTile * 4;
  static constexpr int kQFull = 0, kQEmpty = 2, kSFull = 4, kPReady = 6, kODone = 8, kStats = 10, kOFree = 11, kKFull = 12;
  static constexpr int kKEmpty = kKFull + kStagesK, kVFull = kKEmpty + kStagesK, kVEmpty = kVFull + kStagesV;
  static constexpr int kRawFull = kVEmpty + kStagesV, kRawEmpty = kRawFull + kRaw, kScaleFull = kRawEmpty + kRaw;
  static constexpr int kScaleEmpty = kScaleFull + kScales, kNumBars = kScaleEmpty + kScales;
  static constexpr int kOffMisc = kOffBar + 8 * kNumBars;
  static constexpr int kOffMl = (kOffMisc + 16 + 15) / 16 * 16;     // float2 [128]: group 1's (reference maximum, sum) of a row
  static constexpr int kOffCum = kOffMl + 128 * 8;                  // int [batch + 1] tiles in front, [batch] lengths, [batch + 1] first rows
  static constexpr int kBytes = kOffCum + (3 * kPgMaxBatch + 2) * 4 + 1024;
  static_assert(kBytes <= 232448, "shared memory layout exceeds an SM");
};

__host__ __device__ __forceinline__ int pg_share(int total, int c, int n) { return static_cast<int>(static_cast<long long>(total) * c / n); }
__device__ __forceinline__ int pg_owner(int t, int n, int total) { return static_cast<int>((static_cast<long long>(t + 1) * n - 1) / total); }

// Keys [begin, end) that any row of a query tile sees, and the KV tiles they lie in; one (masked) tile where there are none,
// so that every unit is somebody's.
struct PagedSpan {
  int begin, end, lo, n;
  __device__ PagedSpan(const PagedParams& p, int len, int fresh, int qt) {
    const int first = len - fresh + qt * p.per_tile, last = len - fresh + min((qt + 1) * p.per_tile, fresh) - 1;
    end = p.causal ? min(len, last + 1) : len;
    begin = p.window > 0 ? max(0, first - p.window + 1) : 0;
    if (end <= begin) {
      begin = end = 0;
      lo = 0;
      n = 1;
    } else {
      lo = begin / kPgTile;
      n = (end + kPgTile - 1) / kPgTile - lo;
    }
  }
};

// The units of one CTA, in order.
struct PagedWalk {
  const PagedParams& p;
  const int *cum, *lens, *row0;
  int t, t_end;
  int b, h, qt, len, fresh, tiles;   // sequence, KV head, query tile; its length, new tokens, query tiles
  int begin, end, lo, total, t0, n;  // keys and KV tiles of the unit; this share's: n from t0 on
  bool started = false;
  __device__ PagedWalk(const PagedParams& p_, const int* cum_, const int* lens_, const int* row0_, int t_, int t_end_)
      : p(p_), cum(cum_), lens(lens_), row0(row0_), t(t_), t_end(t_end_) {
    if (t >= t_end) return;
    int a = 0, z = p.batch;   // last sequence with cum[b] <= t: it has tiles
    while (z - a > 1) {
      const int mid = (a + z) >> 1;
      if (cum[mid] <= t) a = mid; else z = mid;
    }
    b = a;
    sequence();
    const int per_head = (cum[b + 1] - cum[b]) / p.heads_kv;
    int rest = t - cum[b];
    h = rest / per_head;
    rest -= h * per_head;
    for (qt = 0;; ++qt) {
      const PagedSpan s(p, len, fresh, qt);
      if (rest < s.n || qt + 1 >= tiles) break;
      rest -= s.n;
    }
    t0 = rest;
  }
  __device__ void sequence() {
    len = lens[b];
    fresh = row0[b + 1] - row0[b];
    tiles = (fresh + p.per_tile - 1) / p.per_tile;
  }
  __device__ bool next() {
    if (t >= t_end) return false;
    if (started) {
      t0 = 0;
      if (++qt >= tiles) {
        qt = 0;
        if (++h >= p.heads_kv) {
          h = 0;
          do ++b; while (b + 1 < p.batch && cum[b + 1] <= t);   // sequences without new tokens
          sequence();
        }
      }
    }
    started = true;
    const PagedSpan s(p, len, fresh, qt);
    begin = s.begin;
    end = s.end;
    lo = s.lo;
    total = s.n;
    n = min(total - t0, t_end - t);
    t += n;
    return true;
  }
  // rows [a, e) of the unit's i-th tile that any of its rows sees
  __device__ void rows_of(int i, int& a, int& e) const {
    const int kv0 = (lo + t0 + i) * kPgTile;
    a = max(begin - kv0, 0);
    e = max(min(end - kv0, kPgTile), 0);
  }
};

// Four e4m3 codes as 16-bit values.  A code's bits, moved to where a wider format has its sign, exponent and mantissa, are the
// code's value times 2^-120 (bf16) or 2^-8 (fp16), subnormals among them; the row's factor takes that back.
template <bool kBf16>
__device__ __forceinline__ uint2 widen4(uint32_t codes) {
  constexpr int kShift = kBf16 ? 4 : 1;
  const uint32_t lo = __byte_perm(codes, 0, 0x1404), hi = __byte_perm(codes, 0, 0x3424);
  return make_uint2((lo & 0x80008000u) | ((lo & 0x7f007f00u) >> kShift), (hi & 0x80008000u) | ((hi & 0x7f007f00u) >> kShift));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  if constexpr (kBf16) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
// The factor of a row in two 16-bit powers of two (their product may be outside the format): low and high half of a word.
template <bool kBf16>
__device__ __forceinline__ uint32_t row_factor(int byte) {
  if (byte == 255) return kBf16 ? 0x3f807fffu : 0x3c007fffu;
  int e = byte - 127 + (kBf16 ? 120 : 8);
  if constexpr (kBf16) {
    const int first = min(e, 127), second = e - first;   // e from -7 to 247
    return static_cast<uint32_t>((first + 127) << 7) | (static_cast<uint32_t>((second + 127) << 7) << 16);
  } else {
    e = min(max(e, -38), 30);   // beyond: under half of the least value, or infinite
    const int first = min(max(e, -14), 15), second = e - first;   // -24 to 15
    const uint32_t s = second >= -14 ? static_cast<uint32_t>(second + 15) << 10 : 1u << (second + 24);
    return (static_cast<uint32_t>(first + 15) << 10) | (s << 16);
  }
}

template <int D, bool kBf16, bool k8Bit>
__global__ void __launch_bounds__(PagedSmem<D, k8Bit>::kThreads, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const __grid_constant__ PagedParams p) {
  using L = PagedSmem<D, k8Bit>;
  using F = SoftmaxFunctor;
  constexpr int N = kPgTile, KC = D / 64, kChunk = N * 128, kThreads = L::kThreads;
  constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::kOffK;
  uint8_t* sV = smem + L::kOffV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 8);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::kOffMl);
  int* s_cum = reinterpret_cast<int*>(smem + L::kOffCum);
  int* s_len = s_cum + kPgMaxBatch + 1;
  int* s_row = s_len + kPgMaxBatch;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AbortState ab{abort_flag, p.status};
  const int active_warps = (p.rows + 31) / 32;   // of each softmax group

  // The merge kernel may be made ready ahead of this kernel's own tensor memory: shared memory keeps every other kernel with
  // tensor memory off the SM.
  static_assert(L::kBytes + 65536 > 233472, "a CTA with tensor memory could share the SM");
  pdl_launch_dependents();

  const int cta = static_cast<int>(blockIdx.x);
  if (warp == 8) {
    for (int i = lane; i < L::kNumBars; i += 32) {
      int count = 1;
      if (i == L::kPReady || i == L::kPReady + 1 || i == L::kStats || i == L::kOFree) count = active_warps * 32;
      if constexpr (k8Bit) {   // written, or read, by the warps that widen
        if ((i >= L::kKFull && i < L::kKEmpty) || (i >= L::kVFull && i < L::kVEmpty) || (i >= L::kRawEmpty && i < L::kScaleFull) || i >= L::kScaleEmpty)
          count = kPgConvWarps;
      }
      mbar_init(bars + i, count);
    }
    fence_barrier_init();
    __syncwarp();
    if (lane == 0) {
      tma_prefetch_desc(&tmQ);
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  if (tid == 0) {
    *abort_flag = (*reinterpret_cast<volatile int*>(p.status) != 0) ? 1 : 0;
    p.cut[cta].w = -1;   // this thread writes the real one, too
  }
  // ---- lengths, and the tiles in front of every sequence ----
  const int most = p.max_blocks << p.page_shift;
  for (int b = tid; b <= p.batch; b += kThreads) {
    s_row[b] = p.cu != nullptr ? min(max(p.cu[b], 0), p.seq) : b * p.seq;
    if (b < p.batch) s_len[b] = min(max(p.lens[b], 0), most);
  }
  __syncthreads();
  if (p.cu != nullptr) {   // first rows that go backwards count as their predecessors: no row is two sequences'
    if (warp == 0) {
      int run = 0;
      for (int i0 = 0; i0 <= p.batch; i0 += 32) {
        int x = i0 + lane <= p.batch ? s_row[i0 + lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, d);
          if (lane >= d) x = max(x, y);
        }
        x = max(x, run);
        if (i0 + lane <= p.batch) s_row[i0 + lane] = x;
        run = __shfl_sync(0xffffffffu, x, 31);
      }
    }
    __syncthreads();
  }
  for (int b = warp; b < p.batch; b += kThreads / 32) {
    const int fresh = s_row[b + 1] - s_row[b], tiles = (fresh + p.per_tile - 1) / p.per_tile;
    int sum = 0;
    for (int qt = lane; qt < tiles; qt += 32) sum += PagedSpan(p, s_len[b], fresh, qt).n;
    if (tiles > 1) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    }
    if (lane == 0) s_cum[b] = sum * p.heads_kv;
  }
  __syncthreads();
  if (warp == 0) {
    int run = 0;
    for (int i0 = 0; i0 < p.batch; i0 += 32) {
      const int tiles = i0 + lane < p.batch ? s_cum[i0 + lane] : 0;
      int x = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (i0 + lane < p.batch) s_cum[i0 + lane] = run + x - tiles;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) s_cum[p.batch] = run;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const int total = s_cum[p.batch];
  const int shares = min(static_cast<int>(gridDim.x), total);   // none is empty
  const int T0 = cta < shares ? pg_share(total, cta, shares) : 0, T1 = cta < shares ? pg_share(total, cta + 1, shares) : 0;
  const bool run_cta = warp_all(T1 > T0 && !*abort_flag);
  auto make_walk = [&]() { return PagedWalk(p, s_cum, s_len, s_row, T0, T1); };
  const int box = 1 << p.box_shift, bpt = N >> p.box_shift;   // rows of a box, boxes of a tile

  if (warp == 8) {
    // ======================= loading warp =======================
    if (run_cta) {
      PagedWalk u = make_walk();
      bool ok = true;
      int J = 0;
      constexpr int kParts = k8Bit ? 1 : KC;   // boxes side by side: 64 columns of 16 bits each, or a row of codes
      // a tile's boxes are spread over the lanes; 8-row boxes of 16 bits are 32
      const int blk = lane / kParts, chunk = lane - blk * kParts;
      for (int ui = 0; ok && u.next(); ++ui) {
        const int qb = ui % p.q_bufs;
        if (ui >= p.q_bufs) ok = warp_all(mbar_wait(bars + L::kQEmpty + qb, (ui / p.q_bufs - 1) & 1, ab, kPgQEmpty));
        if (ok && lane == 0) {
          mbar_arrive_expect_tx(bars + L::kQFull + qb, KC * p.rows * 128);
          const int s = p.cu != nullptr ? s_row[u.b] + u.qt * p.per_tile : u.qt * p.per_tile;
          for (int c = 0; c < KC; ++c)
            tma_load_rows(sQ + qb * p.q_bytes + c * (p.rows_pad * 128), &tmQ, bars + L::kQFull + qb, c * 64, s, u.h * p.group, p.cu != nullptr ? 0 : u.b, p.oq);
        }
        const int* table = p.table + u.b * p.table_stride;
        auto page_at = [&](int i) {   // of this lane's box in the unit's i-th tile
          const int block = ((u.lo + u.t0 + i) * N + blk * box) >> p.page_shift;
          return blk < bpt && block < p.max_blocks ? table[block] : -1;
        };
        int page = page_at(0);
        for (int i = 0; i < u.n && ok; ++i) {
          const int jj = J + i;
          const int page_next = i + 1 < u.n ? page_at(i + 1) : -1;
          int a, e;
          u.rows_of(i, a, e);
          const bool mine = blk < bpt && blk * box < e && (blk + 1) * box > a;
          const int boxes = e > a ? (e + box - 1) / box - a / box : 0;
          const int row = ((u.lo + u.t0 + i) * N + blk * box) & ((1 << p.page_shift) - 1);
          if constexpr (k8Bit) {
            for (int kv = 0; kv < 2 && ok; ++kv) {
              const int r = 2 * jj + kv, st = r % L::kRaw;
              ok = warp_all(mbar_wait(bars + L::kRawEmpty + st, ((r / L::kRaw) & 1) ^ 1, ab, kPgRawEmpty));
              if (!ok) break;
              uint64_t* full = bars + L::kRawFull + st;
              if (lane == 0) mbar_arrive_expect_tx(full, boxes * box * D);
              __syncwarp();
              uint8_t* dst = smem + L::kOffRaw + st * L::kRawBytes + blk * box * D;
              if (mine) {
                if (kv == 0) tma_load_rows(dst, &tmK, full, 0, row, u.h, page, p.ok);
                else tma_load_rows(dst, &tmV, full, 0, row, u.h, page, p.ov);
              }
            }
          } else {
            for (int kv = 0; kv < 2 && ok; ++kv) {
              const int st = kv == 0 ? jj % L::kStagesK : jj % L::kStagesV;
              const uint32_t par = ((kv == 0 ? jj / L::kStagesK : jj / L::kStagesV) & 1) ^ 1;
              uint64_t* full = bars + (kv == 0 ? L::kKFull : L::kVFull) + st;
              ok = warp_all(mbar_wait(bars + (kv == 0 ? L::kKEmpty : L::kVEmpty) + st, par, ab, kv == 0 ? kPgKEmpty : kPgVEmpty));
              if (!ok) break;
              if (lane == 0) mbar_arrive_expect_tx(full, boxes * box * D * 2);
              __syncwarp();
              const int off = st * L::kTileBytes + chunk * kChunk + blk * box * 128;
              if (mine) {
                if (kv == 0) tma_load_rows(sK + off, &tmK, full, chunk * 64, row, u.h, page, p.ok);
                else tma_load_rows(sV + off, &tmV, full, chunk * 64, row, u.h, page, p.ov);
              }
            }
          }
          page = page_next;
        }
        J += u.n;
      }
    }
  } else if (warp == 9) {
    // ======================= issuing warp (converged, one elected lane per batch) =======================
    if (run_cta) {
      constexpr uint32_t idesc_qk = make_idesc_f16(128, N, kBf16, false, false);
      constexpr uint32_t idesc_pv = make_idesc_f16(128, D, kBf16, false, true);
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool { return warp_all(mbar_wait_poll(bar, parity, ab, site)); };
      const uint64_t k_desc0 = make_smem_desc(smem_u32(sK), 16, 1024);
      const uint64_t v_desc0 = make_smem_desc(smem_u32(sV), kChunk, 1024);
      PagedWalk uq = make_walk();
      int uq_i = -1, uq_left = 0, Jq = 0;   // unit and tile of the next scores
      auto issue_qk = [&]() -> bool {
        if (uq_left == 0) {
          uq.next();
          uq_left = uq.n;
          ++uq_i;
          if (!wait(bars + L::kQFull + uq_i % p.q_bufs, (uq_i / p.q_bufs) & 1, kPgQFull)) return false;
        }
        const int st = Jq % L::kStagesK, t = Jq & 1, qb = uq_i % p.q_bufs;
        if (!wait(bars + L::kKFull + st, (Jq / L::kStagesK) & 1, kPgKFull)) return false;
        tc_fence_after_sync();
        --uq_left;
        const uint64_t a = make_smem_desc(smem_u32(sQ + qb * p.q_bytes), 16, 1024);
        const uint64_t bk = k_desc0 + static_cast<uint64_t>(st * (L::kTileBytes >> 4));
        const uint64_t a_chunk = static_cast<uint64_t>(p.rows_pad * 128) >> 4;
        if (elect_one()) {
#pragma unroll
          for (int ch = 0; ch < KC; ++ch)
            umma_ss_x4<2, 2>(tmem_base + kColS + t * N, a + ch * a_chunk, bk + ch * (kChunk >> 4), idesc_qk, ch > 0 ? 1u : 0u);
          umma_commit(bars + L::kSFull + t);
          umma_commit(bars + L::kKEmpty + st);
          if (uq_left == 0) umma_commit(bars + L::kQEmpty + qb);
        }
        ++Jq;
        return true;
      };
      const int n_all = T1 - T0;
      bool ok = issue_qk();
      if (ok && n_all > 1) ok = issue_qk();
      PagedWalk u = make_walk();
      int J = 0;
      for (int ui = 0; ok && u.next(); ++ui) {
        for (int i = 0; i < u.n && ok; ++i, ++J) {
          const int t = J & 1, st = J % L::kStagesV;
          if (i == 0 && ui > 0) ok = wait(bars + L::kOFree, (ui - 1) & 1, kPgOFree);   // the accumulators have been read
          ok = ok && wait(bars + L::kVFull + st, (J / L::kStagesV) & 1, kPgVFull);
          if (!ok) break;
          if constexpr (!k8Bit) {
            int a, e;
            u.rows_of(i, a, e);
            if (a > 0 || e < N) {   // at most two tiles of a unit; rows of 128 bytes, whatever their swizzle
              uint8_t* tile = sV + st * L::kTileBytes;
              for (int x = lane; x < KC * N * 8; x += 32) {
                const int r = (x >> 3) & (N - 1);
                if (r < a || r >= e) *reinterpret_cast<uint4*>(tile + x * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
          }
          ok = wait(bars + L::kPReady + t, (J >> 1) & 1, kPgPReady);
          if (!ok) break;
          tc_fence_after_sync();
          const uint64_t bv = v_desc0 + static_cast<uint64_t>(st * (L::kTileBytes >> 4));
          if (elect_one()) {
#pragma unroll
            for (int g = 0; g < N / 64; ++g)
              umma_ts_x4<8, 128>(tmem_base + kColO + t * D, tmem_base + kColS + t * N + g * 32, bv + g * 512, idesc_pv,
                                 (i >= 2 || g > 0) ? 1u : 0u);
            umma_commit(bars + L::kODone + t);
            umma_commit(bars + L::kVEmpty + st);
          }
          if (Jq < n_all) ok = issue_qk();   // over the scores of tile J, behind its P.V in the pipe
        }
      }
    }
  } else if (warp < 8) {
    // ======================= softmax groups: one query row per thread, alternate tiles =======================
    if ((warp & 3) < active_warps && run_cta) {
      const int t = warp >> 2;
      const int row = (warp & 3) * 32 + lane;
      const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t tS = tmem_base + lane_base + kColS + t * N;
      const uint32_t tO = tmem_base + lane_base + kColO + t * D;
      const RowCtx ctx{0, 0, 0, 0, p.seq, 0, &p.fa};   // softmax asks for the scale only
      const int g = p.head_major ? row / p.per_tile : row % p.group;
      const int qi = p.head_major ? row % p.per_tile : row / p.group;   // position in the tile
      const float c2 = p.fa.f[0] * 1.4426950408889634f;
      PagedWalk u = make_walk();
      int J0 = 0;   // tiles of the units before this one
      for (int ui = 0; u.next(); ++ui, J0 += u.n) {
        const int tok = u.qt * p.per_tile + qi;   // the row's new token
        const bool live = row < p.rows && tok < u.fresh;
        const bool any_live = __any_sync(0xffffffffu, live);
        const int pos = u.len - u.fresh + tok;
        // keys of the row; those of a row that does not exist are not looked at
        const int key_end = live ? min(u.end, p.causal ? pos + 1 : u.len) : 0x3fffffff;
        const int key_begin = live && p.window > 0 ? pos - p.window + 1 : 0;
        float rs[2];
        F::init(rs, ctx);
        for (int J = J0 + ((J0 ^ t) & 1); J < J0 + u.n; J += 2) {
          mbar_wait_rows(bars + L::kSFull + t, (J >> 1) & 1, ab, kPgSFull);
          if (!any_live) {   // nothing of this warp's rows is kept
            mbar_arrive(bars + L::kPReady + t);
            continue;
          }
          tc_fence_after_sync();
          const int kv0 = (u.lo + u.t0 + J - J0) * N;
          const int e = key_end - kv0, a = key_begin - kv0;
          const bool edge = __any_sync(0xffffffffu, e < N || a > 0);
          float o_scale = 1.0f;
          if constexpr (!k8Bit) {
            float s[N];
#pragma unroll
            for (int c = 0; c < N / 32; ++c) tmem_ld32f(tS + c * 32, &s[c * 32]);
            tmem_wait_ld();
            if (edge) {
#pragma unroll
              for (int i = 0; i < N; ++i) s[i] = i < e && i >= a ? s[i] : -INFINITY;
            }
            o_scale = F::template tile_pieces<N, 4, false>(s, rs, ctx, [](float mx) { return mx; }, [&](int c) {
              constexpr int W = N / 4 / 2;
              uint32_t pk[W];
#pragma unroll
              for (int i = 0; i < W; ++i) pk[i] = pack2<kBf16>(s[c * 2 * W + 2 * i], s[c * 2 * W + 2 * i + 1]);
              static_assert(W == 16, "a quarter of the row per store");
              tmem_st16(tS + c * W, pk);
            });
          } else {
            // The warps that widen codes leave this thread no room for a row of 128 scores: they are read twice, a quarter at a
            // time, first for the maximum.  P goes over what has been read.
            float mx = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < N / 32; ++c) {
              float s[32];
              tmem_ld32f(tS + c * 32, s);
              tmem_wait_ld();
              if (edge) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = c * 32 + i < e && c * 32 + i >= a ? s[i] : -INFINITY;
              }
              float m0 = s[0], m1 = s[1];
#pragma unroll
              for (int i = 2; i + 4 <= 32; i += 4) {
                m0 = max3(m0, s[i], s[i + 2]);
                m1 = max3(m1, s[i + 1], s[i + 3]);
              }
              mx = max3(mx, max3(m0, s[30], s[31]), m1);
            }
            if ((mx - rs[0]) * c2 > 8.0f) {
              o_scale = fast_exp2((rs[0] - mx) * c2);
              rs[0] = mx;
              rs[1] *= o_scale;
            }
            const float neg = -rs[0] * c2;
            float a0 = 0.f, a1 = 0.f;
#pragma unroll 1
            for (int c = 0; c < N / 32; ++c) {
              float s[32];
              tmem_ld32f(tS + c * 32, s);
              tmem_wait_ld();
              if (edge) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = c * 32 + i < e && c * 32 + i >= a ? s[i] : -INFINITY;
              }
              uint32_t pk[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float x = fast_exp2(fmaf(s[2 * i], c2, neg)), y = fast_exp2(fmaf(s[2 * i + 1], c2, neg));
                a0 += x;
                a1 += y;
                pk[i] = pack2<kBf16>(x, y);
              }
              tmem_st16(tS + c * 16, pk);
            }
            rs[1] += a0 + a1;
          }
          if (J - J0 >= 2 && __any_sync(0xffffffffu, o_scale != 1.0f)) {
            mbar_wait_rows(bars + L::kODone + t, ((J >> 1) - 1) & 1, ab, kPgODone);
            tc_fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tmem_ld32f(tO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] *= o_scale;
              tmem_st32f(tO + c * 32, o);
            }
          }
          tmem_wait_st();
          tc_fence_before_sync();
          mbar_arrive(bars + L::kPReady + t);
        }
        if (t == 1) {
          if (ui > 0) mbar_wait_rows(bars + L::kOFree, (ui - 1) & 1, ab, kPgOFree);   // group 0 has read the last unit's
          s_ml[row] = make_float2(rs[0], rs[1]);
          mbar_arrive(bars + L::kStats);
          continue;
        }
        // ---- end of a unit (group 0): both accumulators of the row, weighted ----
        const int Jl = J0 + u.n - 1, l0 = (Jl & 1) == 0 ? Jl : Jl - 1, l1 = (Jl & 1) == 1 ? Jl : Jl - 1;
        const bool has0 = l0 >= J0, has1 = l1 >= J0;
        mbar_wait_rows(bars + L::kStats, ui & 1, ab, kPgStats);
        if (has0) mbar_wait_rows(bars + L::kODone, (l0 >> 1) & 1, ab, kPgODone);
        if (has1) mbar_wait_rows(bars + L::kODone + 1, (l1 >> 1) & 1, ab, kPgODone);
        if (!warp_all(!*abort_flag)) break;
        tc_fence_after_sync();
        const float2 ml1 = s_ml[row];
        const float m = fmaxf(rs[0], ml1.x);
        const float w0 = fast_exp2((rs[0] - m) * c2), w1 = fast_exp2((ml1.x - m) * c2);
        const float sum = rs[1] * w0 + ml1.y * w1;
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // no key: 0, and -inf
        const float f0 = has0 ? w0 * inv : 0.0f, f1 = has1 ? w1 * inv : 0.0f;
        const float lse = sum == 0.0f ? -INFINITY : logf(sum) + m * p.fa.f[0];
        const int head = u.h * p.group + g;
        const bool whole = u.n == u.total;
        // a partial result: the unit's first share leaves it in the second slot of its CTA, the later ones in the first
        const long long slot = (2LL * blockIdx.x + (u.t0 == 0 ? 1 : 0)) * p.rows + row;
        const long long at = p.cu != nullptr ? s_row[u.b] + tok : tok;   // row of o
        uint16_t* orow = static_cast<uint16_t*>(p.o) + (p.cu != nullptr ? 0 : u.b * p.o_sb) + at * p.o_ss + head * p.o_sh;
        if (any_live) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float a0[32], a1[32];
            tmem_ld32f(tO + c * 32, a0);
            tmem_ld32f(tO + D + c * 32, a1);
            tmem_wait_ld();
            if (has0 && has1) {   // an accumulator that the unit has not used holds anything
#pragma unroll
              for (int i = 0; i < 32; ++i) a0[i] = fmaf(a0[i], f0, a1[i] * f1);
            } else {
              const float f = has0 ? f0 : f1;
#pragma unroll
              for (int i = 0; i < 32; ++i) a0[i] = (has0 ? a0[i] : a1[i]) * f;
            }
            if (live) {
              if (whole) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  uint4 pk;
                  pk.x = pack2<kBf16>(a0[8 * v + 0], a0[8 * v + 1]);
                  pk.y = pack2<kBf16>(a0[8 * v + 2], a0[8 * v + 3]);
                  pk.z = pack2<kBf16>(a0[8 * v + 4], a0[8 * v + 5]);
                  pk.w = pack2<kBf16>(a0[8 * v + 6], a0[8 * v + 7]);
                  reinterpret_cast<uint4*>(orow + c * 32)[v] = pk;
                }
              } else {
                float4* dst = reinterpret_cast<float4*>(p.part_o + slot * D + c * 32);
#pragma unroll
                for (int v = 0; v < 8; ++v) dst[v] = make_float4(a0[4 * v], a0[4 * v + 1], a0[4 * v + 2], a0[4 * v + 3]);
              }
            }
          }
          if (live) {
            if (!whole) p.part_lse[slot] = lse;
            else if (p.lse != nullptr) p.lse[(p.cu != nullptr ? static_cast<long long>(head) : static_cast<long long>(u.b) * p.heads + head) * p.seq + at] = lse;
          }
        }
        if (row == 0 && !whole && u.t0 == 0)   // t is behind the unit's part
          p.cut[cta] = make_int4(u.b, u.h, u.qt, pg_owner(u.t - u.n + u.total - 1, shares, total));
        tc_fence_before_sync();
        mbar_arrive(bars + L::kOFree);
      }
    }
  } else if constexpr (k8Bit) {
    if (warp == 10) {
      // ======================= factors of the rows: four rows a lane, one tile ahead =======================
      if (run_cta) {
        PagedWalk u = make_walk();
        bool ok = true;
        int J = 0;
        while (ok && u.next()) {
          const int* table = p.table + u.b * p.table_stride;
          auto page_at = [&](int i) {
            const int block = ((u.lo + u.t0 + i) * N + 4 * lane) >> p.page_shift;
            const int page = i < u.n && block < p.max_blocks ? table[block] : -1;
            return page >= 0 && page < p.pages ? page : -1;
          };
          auto bytes_of = [&](int i, int page, uint32_t (&w)[2]) {   // rows that do not count: byte 256 below
            const int row = ((u.lo + u.t0 + i) * N + 4 * lane) & ((1 << p.page_shift) - 1);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
              w[kv] = 0;
              if (page < 0) continue;
              const uint8_t* s = p.scale[kv] + page * p.scale_stride[kv][0] + row * p.scale_stride[kv][1] + u.h * p.scale_stride[kv][2];
#pragma unroll
              for (int k = 0; k < 4; ++k) w[kv] |= static_cast<uint32_t>(s[k * p.scale_stride[kv][1]]) << (8 * k);
            }
          };
          int page = page_at(0), next = page_at(1);
          uint32_t w[2], w_next[2];
          bytes_of(0, page, w);
          for (int i = 0; i < u.n && ok; ++i, ++J) {
            const int after = page_at(i + 2);
            bytes_of(i + 1, next, w_next);
            const int st = J % L::kScales;
            ok = warp_all(mbar_wait(bars + L::kScaleEmpty + st, ((J / L::kScales) & 1) ^ 1, ab, kPgScaleEmpty));
            if (!ok) break;
            int a, e;
            u.rows_of(i, a, e);
            uint32_t* dst = reinterpret_cast<uint32_t*>(smem + L::kOffScale) + st * 2 * N + 4 * lane;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
              uint32_t f[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const bool in = page >= 0 && 4 * lane + k >= a && 4 * lane + k < e;
                f[k] = in ? row_factor<kBf16>((w[kv] >> (8 * k)) & 255) : kBf16 ? 0x3f800000u : 0x3c000000u;   // times 0, times 1
              }
              *reinterpret_cast<uint4*>(dst + kv * N) = make_uint4(f[0], f[1], f[2], f[3]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + L::kScaleFull + st);
            page = next;
            next = after;
            w[0] = w_next[0];
            w[1] = w_next[1];
          }
        }
      }
    } else if (run_cta) {
      // ======================= widening: codes to 16 bits, swizzled as TMA would have written them =======================
      constexpr int kUnits = D / 16, kItems = N * kUnits / (32 * kPgConvWarps);   // pieces of 16 codes of a row, of a thread
      const int ct = tid - 352;
      const int unit = ct % kUnits;
      // columns 16 unit to + 15 are two 16-byte pieces of the row's 128-byte chunk; half of the threads begin with the second,
      // so that eight neighbours write to all banks
      const int chunk = unit / 4, piece = (unit % 4) * 2, swap = (unit / 4) & 1;
      bool ok = true;
      const int n_all = T1 - T0;
      for (int J = 0; J < n_all && ok; ++J) {
        const int sc = J % L::kScales;
        ok = warp_all(mbar_wait(bars + L::kScaleFull + sc, (J / L::kScales) & 1, ab, kPgScaleFull));
        for (int kv = 0; kv < 2 && ok; ++kv) {
          const int r = 2 * J + kv, raw = r % L::kRaw, st = J % 2;
          ok = warp_all(mbar_wait(bars + (kv == 0 ? L::kKEmpty : L::kVEmpty) + st, ((J / 2) & 1) ^ 1, ab, kv == 0 ? kPgKEmpty : kPgVEmpty));
          ok = ok && warp_all(mbar_wait(bars + L::kRawFull + raw, (r / L::kRaw) & 1, ab, kPgRawFull));
          if (!ok) break;
          const uint8_t* src = smem + L::kOffRaw + raw * L::kRawBytes;
          const uint32_t* factor = reinterpret_cast<const uint32_t*>(smem + L::kOffScale) + (sc * 2 + kv) * N;
          uint8_t* dst = (kv == 0 ? sK : sV) + st * L::kTileBytes + chunk * kChunk;
#pragma unroll
          for (int it = 0; it < kItems; ++it) {
            const int row = it * (32 * kPgConvWarps / kUnits) + ct / kUnits;
            const uint4 codes = *reinterpret_cast<const uint4*>(src + row * D + unit * 16);
            const uint32_t f = factor[row];
            const uint32_t f1 = __byte_perm(f, 0, 0x1010), f2 = f >> 16;
            const uint32_t c4[4] = {codes.x, codes.y, codes.z, codes.w};
            uint32_t w[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint2 x = widen4<kBf16>(c4[k]);
              w[2 * k] = mul2<kBf16>(x.x, f1);
              w[2 * k + 1] = mul2<kBf16>(x.y, f1);
            }
            if (f2 != (kBf16 ? 0x3f80u : 0x3c00u)) {   // a factor outside the format: rows of very large or small values
              const uint32_t ff = f2 * 0x10001u;
#pragma unroll
              for (int k = 0; k < 8; ++k) w[k] = mul2<kBf16>(w[k], ff);
            }
            uint8_t* line = dst + row * 128;
            const uint4 lo = make_uint4(w[0], w[1], w[2], w[3]), hi = make_uint4(w[4], w[5], w[6], w[7]);
            const int p0 = (piece + swap) ^ (row & 7), p1 = (piece + 1 - swap) ^ (row & 7);
            *reinterpret_cast<uint4*>(line + p0 * 16) = swap ? hi : lo;
            *reinterpret_cast<uint4*>(line + p1 * 16) = swap ? lo : hi;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bars + (kv == 0 ? L::kKFull : L::kVFull) + st);
            mbar_arrive(bars + L::kRawEmpty + raw);
          }
        }
        if (ok && lane == 0) mbar_arrive(bars + L::kScaleEmpty + sc);
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// Adds up the partial rows of the units that were cut: o = sum_i exp(lse_i - lse) part_i.  Block x looks after the unit that
// begins in CTA x and goes on in others, a warp a row.
template <int D, bool kBf16>
__global__ void __launch_bounds__(128) paged_merge_kernel(const __grid_constant__ PagedParams p, int ctas) {
  pdl_launch_dependents();
  const int row = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, c_lo = blockIdx.x;
  constexpr int E = D / 32;
  pdl_wait();
  if (row >= p.rows) return;
  const int4 cut = __ldcg(p.cut + c_lo);
  if (cut.w < 0) return;
  const int g = p.head_major ? row / p.per_tile : row % p.group, qi = p.head_major ? row % p.per_tile : row / p.group;
  const int tok = cut.z * p.per_tile + qi, head = cut.y * p.group + g;
  int row0 = 0, fresh = p.seq;
  if (p.cu != nullptr) {
    row0 = min(max(p.cu[cut.x], 0), p.seq);
    fresh = min(max(p.cu[cut.x + 1], 0), p.seq) - row0;
  }
  if (tok >= fresh) return;
  const int c_hi = min(cut.w, ctas - 1);
  float mx = -INFINITY, den = 0.0f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  // four shares at a time, their statistics and rows loaded together, added up against a running maximum
#pragma unroll 1
  for (int c0 = c_lo; c0 <= c_hi; c0 += 4) {
    float l[4], x[4][E];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = c0 + k <= c_hi;
      const int c = in ? c0 + k : c_hi;
      const long long slot = (2LL * c + (c == c_lo ? 1 : 0)) * p.rows + row;
      const float* src = p.part_o + slot * D + lane * E;
      l[k] = __ldcg(p.part_lse + slot);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(src + e));
        x[k][e] = v.x;
        x[k][e + 1] = v.y;
      }
      if (!in) l[k] = -INFINITY;
    }
    // shares in which the row saw nothing count nothing; NaN passes through: the maxima ignore it, its weight does not
    const float m = fmaxf(mx, fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])));
    const float old = mx == -INFINITY ? 0.0f : __expf(mx - m);
    den *= old;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= old;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = l[k] != -INFINITY;
      const float wgt = in ? __expf(l[k] - m) : 0.0f;
      den += wgt;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = in ? fmaf(wgt, x[k][e], acc[e]) : acc[e];
    }
    mx = m;
  }
  const float inv = den == 0.0f ? 0.0f : 1.0f / den;
  const long long at = row0 + tok;
  uint16_t* orow = static_cast<uint16_t*>(p.o) + (p.cu != nullptr ? 0 : cut.x * p.o_sb) + at * p.o_ss + head * p.o_sh + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(orow + e) = pack2<kBf16>(acc[e] * inv, acc[e + 1] * inv);
  if (lane == 0 && p.lse != nullptr)
    p.lse[(p.cu != nullptr ? static_cast<long long>(head) : static_cast<long long>(cut.x) * p.heads + head) * p.seq + at] = den == 0.0f ? -INFINITY : mx + logf(den);
}

struct PagedPlan {
  int group, per_tile, rows, ctas;
  long long off_lse, off_cut, bytes;
};

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
  d->per_tile = std::min(kPgTile / d->group, a->seq);
  d->rows = d->per_tile * d->group;
  const long long most_kv = static_cast<long long>(c.max_blocks) * c.page_size;
  if (most_kv > 0x3fffffff) return ATTN_B200_E_UNSUPPORTED;
  const long long q_tiles = packed ? a->seq / d->per_tile + c.batch : static_cast<long long>(c.batch) * ((a->seq + d->per_tile - 1) / d->per_tile);
  const long long most = q_tiles * c.heads_kv * ((most_kv + kPgTile - 1) / kPgTile);
  if (most > 0x3fffffff) return ATTN_B200_E_UNSUPPORTED;
  d->ctas = static_cast<int>(std::min<long long>(sms, most));
  d->off_lse = 2LL * d->ctas * d->rows * c.head_dim * 4;
  d->off_cut = (d->off_lse + 2LL * d->ctas * d->rows * 4 + 15) / 16 * 16;
  d->bytes = (d->off_cut + 16LL * d->ctas + 255) / 256 * 256;
  return ATTN_B200_OK;
}

// Tensor map over a pool of codes [page][row][head][dim] of bytes: a box is a row of one head by `box_rows` rows of a page.
inline int encode_codes_map(CUtensorMap* tm, CoordOrder* order, const void* base, const AttnB200PagedCache& c, const int64_t stride[3], int box_rows) {
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
                         CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ATTN_B200_OK : ATTN_B200_E_UNSUPPORTED;
}

template <int D, bool kBf16, bool k8Bit>
int launch_paged(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status) {
  using L = PagedSmem<D, k8Bit>;
  const AttnB200PagedCache& c = a->cache;
  CUtensorMap tmQ, tmK, tmV;
  PagedParams p;
  std::memset(&p, 0, sizeof(p));
  const bool packed = a->cu_seqlens != nullptr;
  int rc = encode_rows_map(&tmQ, &p.oq, a->q, a->dtype, D, packed ? 1 : c.batch, a->seq, a->heads, a->q_stride, d.per_tile, d.group);
  if (rc != ATTN_B200_OK) return rc;
  const int box = std::min(c.page_size, kPgTile);
  if constexpr (k8Bit) {
    rc = encode_codes_map(&tmK, &p.ok, c.k, c, c.k_stride, box);
    if (rc == ATTN_B200_OK) rc = encode_codes_map(&tmV, &p.ov, c.v, c, c.v_stride, box);
  } else {
    rc = encode_rows_map(&tmK, &p.ok, c.k, a->dtype, D, c.num_pages, c.page_size, c.heads_kv, c.k_stride, box);
    if (rc == ATTN_B200_OK) rc = encode_rows_map(&tmV, &p.ov, c.v, a->dtype, D, c.num_pages, c.page_size, c.heads_kv, c.v_stride, box);
  }
  if (rc != ATTN_B200_OK) return rc;
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
  p.rows_pad = (d.rows + 7) / 8 * 8;
  p.q_bytes = (D / 64) * p.rows_pad * 128;
  p.q_bufs = 2 * p.q_bytes <= D * 256 ? 2 : 1;
  p.head_major = p.oq.pos_s < p.oq.pos_h ? 1 : 0;
  p.max_blocks = c.max_blocks;
  p.pages = c.num_pages;
  while ((1 << p.page_shift) < c.page_size) ++p.page_shift;
  while ((1 << p.box_shift) < box) ++p.box_shift;
  p.causal = a->causal != 0;
  p.window = a->window;
  for (int i = 0; k8Bit && i < 3; ++i) {
    const int extent[3] = {c.num_pages, c.page_size, c.heads_kv};
    p.scale[0] = c.k_scale;
    p.scale[1] = c.v_scale;
    p.scale_stride[0][i] = extent[i] > 1 ? c.k_scale_stride[i] : 0;
    p.scale_stride[1][i] = extent[i] > 1 ? c.v_scale_stride[i] : 0;
  }
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_lse = reinterpret_cast<float*>(ws + d.off_lse);
  p.cut = reinterpret_cast<int4*>(ws + d.off_cut);
  p.status = status;
  p.fa.f[0] = a->scale;
  auto kernel = paged_attention_kernel<D, kBf16, k8Bit>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess) {
    cudaGetLastError();
    return ATTN_B200_E_LAUNCH;
  }
  if (!launch_pdl(kernel, dim3(d.ctas), dim3(L::kThreads), L::kBytes, stream, tmQ, tmK, tmV, p)) return ATTN_B200_E_LAUNCH;
  if (d.ctas == 1) return ATTN_B200_OK;   // one share: nothing was cut
  const dim3 grid(d.ctas, (d.rows + 3) / 4);
  return launch_pdl(paged_merge_kernel<D, kBf16>, grid, dim3(128), 0, stream, p, d.ctas) ? ATTN_B200_OK : ATTN_B200_E_LAUNCH;
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
  const bool bf16 = a->dtype == ATTN_B200_DTYPE_BF16;
#define ATTN_B200_PAGED(DIM)                                                                                                                     \
  return codes ? (bf16 ? b200::launch_paged<DIM, true, true>(a, d, stream, status) : b200::launch_paged<DIM, false, true>(a, d, stream, status)) \
               : (bf16 ? b200::launch_paged<DIM, true, false>(a, d, stream, status) : b200::launch_paged<DIM, false, false>(a, d, stream, status))
  if (c.head_dim == 64) { ATTN_B200_PAGED(64); }
  ATTN_B200_PAGED(128);
#undef ATTN_B200_PAGED
}

}  // extern "C"
