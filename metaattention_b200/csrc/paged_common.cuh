// What the kernels of attention over a paged cache share (paged_tokens.cu, paged_chunk.cu): the list of work and its shares, the
// loads, and 8-bit rows.
//
// One list of work: a unit is a tile of query rows -- the (position, head of the group) pairs of one KV head of one
// sequence, so that K and V are read once for the group -- with the 128-row KV tiles that any of its rows sees.  The KV
// tiles of all units, in order, are cut into one equal share per SM: a long context against a single token is split over the
// chip, the units of a prompt are spread over it evenly whatever their lengths, and a share walks its units with every ring
// and barrier phase carried across them.  (Where no unit has more than four tiles, shares are whole units and there is nothing to
// merge; else a unit counts two tiles more than it has, for its beginning and end.)  A unit that lies in one share writes its rows; the others leave fp32 partial rows
// that a second small kernel adds up (paged_attention.cu).  Each CTA counts the list itself from the lengths on the device,
// so a captured call follows them.
// Pages are fetched by TMA, a box of up to 128 rows of one page, its index from the block table; boxes without a row that
// counts are not fetched.  V rows behind the last key of a unit, or in front of its window, hold anything: they are zeroed in
// shared memory (0 * NaN would reach the row), the scores there are masked.
#pragma once

#include <atomic>

#include <cuda_fp8.h>

#include "../../include/attn_b200.h"
#include "common_host.cuh"
#include "functors.cuh"
#include "parallel_launch.cuh"
#include "rotary.cuh"

namespace b200 {

constexpr int kPgTile = 128;       // KV rows of a tile
constexpr int kPgMaxBatch = 1024;  // sequences of a call

// What a unit's beginning and end cost, in tiles, where the list is cut into equal shares: 16 batches of chunks and tokens of
// all kinds took 55 us in the mean with 0, 50 with 1, 48 with 2, 48.5 with 4.
constexpr int kPgUnitCost = 2;

struct PagedParams {
  void* o;
  float* lse;
  long long o_sb, o_ss, o_sh;
  const int* cu;                 // packed rows, or null
  const int* lens;
  const int* table;
  long long table_stride;
  int batch, heads, heads_kv, group, seq;
  int per_tile;                  // query positions of a unit
  int tile_pos;                  // and of one of its tiles of query rows (paged_chunk.cu has two)
  int rows;                      // rows of a partial result: 128 to a tile, the last one's used ones
  int head_major;                // row = g * per_tile + i (1) or i * group + g (0): the order the tensor map delivers
  int max_blocks, page_shift, pages, box_shift;   // rows of a box: min(page, 128)
  int causal, window;
  int whole;                     // shares are whole units, not tiles: nothing is cut
  const uint16_t* q;             // 8-bit caches: the queries, and exponents of k and v
  long long qs[3];               // (batch, seq, head)
  const uint8_t* scale8[2];
  long long scale_stride[2][3];
  float* part_o;                 // [2 * CTAs][D / 4][rows][4]: in paged_chunk.cu a lane has a row (a row's columns in one piece: 4100 cycles a unit)
  float* part_lse;               // [2 * CTAs][rows]
  int4* cut;                     // [CTAs] sequence, KV head, query tile and last CTA of the unit that begins in a CTA and goes on, or w = -1
  int2* cut_rows;                // [CTAs] first row of that unit's sequence in packed rows (else 0), and its new tokens
  CoordOrder oq, ok, ov;
  int* status;
  float scale;
};

enum PagedWaitSite {
  kPgQFull = 101, kPgQEmpty, kPgKFull, kPgKEmpty, kPgVFull, kPgVEmpty, kPgSFull, kPgPReady, kPgODone, kPgStats, kPgOFree, kPgRawFull, kPgRawEmpty,
  kPgScales, kPgScalesEmpty, kPgSFree, kPgSmemAlign
};

// mbar_wait() whose way out of line is a call: most waits end in their first attempt, which the hardware suspends, and where
// twenty warps run seven different loops every instruction in line counts.
static __device__ __noinline__ bool paged_wait_on(uint64_t* bar, uint32_t parity, volatile int* cta_flag, int* status, int site) {
  return mbar_wait(bar, parity, AbortState{cta_flag, status}, site);
}
__device__ __forceinline__ bool paged_wait(uint64_t* bar, uint32_t parity, const AbortState& ab, int site) {
  return mbar_try_wait(bar, parity) || paged_wait_on(bar, parity, ab.cta_flag, ab.device_status, site);
}

// total * c / n, in 32 bits (a division in 64 is 100 instructions, all of them cold)
__device__ __forceinline__ int pg_share(int total, int c, int n) {
  const int q = total / n;
  return q * c + (total - q * n) * c / n;
}
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
  int t, t_end;                      // the share, in tiles of the list, kPgUnitCost of them in front of every unit's own (whole: in units)
  int b, h, qt, len, fresh;          // sequence, KV head, query tile; its length, new tokens
  int begin, end, lo, total, t0, n;  // keys and KV tiles of the unit; this share's: n from t0 on (before the first next(): the place in the unit)
  int last;                          // place of the unit's last tile in the list
  bool started = false;
  __device__ PagedWalk(const PagedParams& p_, const int* cum_, const int* lens_, const int* row0_, const int* start, int t_, int t_end_)
      : p(p_), cum(cum_), lens(lens_), row0(row0_), t(t_), t_end(t_end_) {
    if (t >= t_end) return;
    b = start[0];
    h = start[1];
    qt = start[2];
    t0 = start[3];
    sequence();
  }
  __device__ void sequence() {
    len = lens[b];
    fresh = row0[b + 1] - row0[b];
  }
  __device__ bool next() {
    if (t >= t_end) return false;
    if (started) {
      t0 = 0;
      if (++qt * p.per_tile >= fresh) {
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
    if (p.whole) {
      n = total;
      ++t;
      return true;
    }
    const int to = min(total + kPgUnitCost, t0 + t_end - t);
    last = t - t0 + total + kPgUnitCost - 1;
    t += to - t0;
    t0 = max(t0 - kPgUnitCost, 0);
    n = max(to - kPgUnitCost, 0) - t0;
    return n > 0;   // 0: the share ends in front of the unit's tiles
  }
  // rows [a, e) of the unit's i-th tile that any of its rows sees
  __device__ void rows_of(int i, int& a, int& e) const {
    const int kv0 = (lo + t0 + i) * kPgTile;
    a = max(begin - kv0, 0);
    e = max(min(end - kv0, kPgTile), 0);
  }
};

// Lengths, first rows of the new tokens and tiles in front of every sequence, by all `threads` of the CTA, and the place in the list
// where its share begins, by one warp (each role's warps looking for it themselves ran the same cold code six times over: 6500 cycles in
// front of a chunk's first unit, 3000 with this); the caller syncs behind it.
struct PagedTables {
  int *cum, *len, *row;   // [batch + 1], [batch], [batch + 1] in shared memory
  int* start;             // sequence, KV head, query tile and tile of that unit; the share [4], [5] in the list
  static constexpr int kBytes = (3 * kPgMaxBatch + 8) * 4;
  __device__ explicit PagedTables(uint8_t* at)
      : cum(reinterpret_cast<int*>(at)), len(cum + kPgMaxBatch + 1), row(len + kPgMaxBatch), start(row + kPgMaxBatch + 1) {}

  __device__ void locate(const PagedParams& p) const {   // by a warp
    const int lane = threadIdx.x & 31, total = cum[p.batch], shares = min(static_cast<int>(gridDim.x), total);
    const int cta = static_cast<int>(blockIdx.x);
    if (cta >= shares) {
      if (lane == 0) start[4] = start[5] = 0;
      return;
    }
    const int t = pg_share(total, cta, shares);
    int b = 0;   // last sequence with cum[b] <= t: it has tiles
    for (int i0 = 0; i0 < p.batch; i0 += 32) {
      const uint32_t in = __ballot_sync(0xffffffffu, i0 + lane < p.batch && cum[i0 + lane] <= t);
      if (in == 0) break;
      b = i0 + 31 - __clz(in);
    }
    const int per_head = (cum[b + 1] - cum[b]) / p.heads_kv, h = (t - cum[b]) / per_head;
    int rest = t - cum[b] - h * per_head, qt = rest;
    if (p.whole) {
      rest = 0;
    } else {
      const int fresh = row[b + 1] - row[b], tiles = (fresh + p.per_tile - 1) / p.per_tile;
      for (int q0 = 0; q0 < tiles; q0 += 32) {
        const int n = q0 + lane < tiles ? PagedSpan(p, len[b], fresh, q0 + lane).n + kPgUnitCost : 0;
        int x = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, d);
          if (lane >= d) x += y;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, x > rest);
        if (behind != 0) {
          const int at = __ffs(behind) - 1;
          qt = q0 + at;
          rest -= __shfl_sync(0xffffffffu, x - n, at);
          break;
        }
        rest -= __shfl_sync(0xffffffffu, x, 31);
      }
    }
    if (lane == 0) {
      start[0] = b;
      start[1] = h;
      start[2] = qt;
      start[3] = rest;
      start[4] = t;
      start[5] = pg_share(total, cta + 1, shares);
    }
  }

  __device__ void count(const PagedParams& p, int threads) const {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int most = p.max_blocks << p.page_shift;
    for (int b = tid; b <= p.batch; b += threads) {
      row[b] = p.cu != nullptr ? min(max(p.cu[b], 0), p.seq) : b * p.seq;
      if (b < p.batch) len[b] = min(max(p.lens[b], 0), most);
      if (p.whole) cum[b] = b * (p.heads_kv * ((p.seq + p.per_tile - 1) / p.per_tile));   // units: the same for every sequence, unless packed
    }
    __syncthreads();
    if (p.whole && p.cu == nullptr) {
      if (warp == 0) locate(p);
      return;
    }
    if (p.cu != nullptr) {   // first rows that go backwards count as their predecessors: no row is two sequences'
      if (warp == 0) {
        int run = 0;
        for (int i0 = 0; i0 <= p.batch; i0 += 32) {
          int x = i0 + lane <= p.batch ? row[i0 + lane] : 0;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x = max(x, y);
          }
          x = max(x, run);
          if (i0 + lane <= p.batch) row[i0 + lane] = x;
          run = __shfl_sync(0xffffffffu, x, 31);
        }
      }
      __syncthreads();
    }
    if (p.cu == nullptr && p.seq <= 4 * p.per_tile) {   // a few query tiles: a thread a sequence
      for (int b = tid; b < p.batch; b += threads) {
        int sum = 0;
        for (int qt = 0; qt * p.per_tile < p.seq; ++qt) sum += p.whole ? 1 : PagedSpan(p, len[b], p.seq, qt).n + kPgUnitCost;
        cum[b] = sum * p.heads_kv;
      }
    } else {
      for (int b = warp; b < p.batch; b += threads / 32) {
        const int fresh = row[b + 1] - row[b], tiles = (fresh + p.per_tile - 1) / p.per_tile;
        int sum = 0;
        for (int qt = lane; qt < tiles; qt += 32) sum += p.whole ? 1 : PagedSpan(p, len[b], fresh, qt).n + kPgUnitCost;
        if (tiles > 1) {
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        }
        if (lane == 0) cum[b] = sum * p.heads_kv;
      }
    }
    __syncthreads();
    if (warp == 0) {
      int run = 0;
      for (int i0 = 0; i0 < p.batch; i0 += 32) {
        const int tiles = i0 + lane < p.batch ? cum[i0 + lane] : 0;
        int x = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, d);
          if (lane >= d) x += y;
        }
        if (i0 + lane < p.batch) cum[i0 + lane] = run + x - tiles;
        run += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) cum[p.batch] = run;
      __syncwarp();
      locate(p);
    }
  }
};

// The share of a CTA.
struct PagedShare {
  int total, shares, t0, t1;
  __device__ PagedShare(const PagedParams& p, const PagedTables& tab) {
    total = tab.cum[p.batch];
    shares = min(static_cast<int>(gridDim.x), total);   // none is empty
    t0 = tab.start[4];
    t1 = tab.start[5];
  }
};

// A loading warp: the tiles of K or of V of a share into a ring.  A tile is kParts boxes side by side (64 columns of 16 bits
// each, chunk_bytes apart; or one of codes) of kRowBytes a row; they are spread over the lanes, at most 32 of them.
template <int kParts, int kRowBytes, int kStages, class OnUnit>
__device__ __forceinline__ void paged_load(const PagedParams& p, PagedWalk u, const CUtensorMap* tm, const CoordOrder& order, uint8_t* ring, int tile_bytes,
                                           int chunk_bytes, uint64_t* full, uint64_t* empty, const AbortState& ab, int site, OnUnit&& on_unit) {
  const int lane = threadIdx.x & 31;
  const int box = 1 << p.box_shift, bpt = kPgTile >> p.box_shift;   // rows of a box, boxes of a column of them
  const int blk = lane / kParts, chunk = lane - blk * kParts;
  int st = 0;
  uint32_t par = 1;
  for (int ui = 0; u.next(); ++ui) {
    if (!on_unit(u, ui)) return;
    const int* table = p.table + u.b * p.table_stride;
    auto page_at = [&](int i) {   // of this lane's box in the unit's i-th tile
      const int block = ((u.lo + u.t0 + i) * kPgTile + blk * box) >> p.page_shift;
      return blk < bpt && block < p.max_blocks ? table[block] : -1;
    };
    int page = page_at(0);
    for (int i = 0; i < u.n; ++i) {
      const int page_next = i + 1 < u.n ? page_at(i + 1) : -1;
      int a, e;
      u.rows_of(i, a, e);
      const bool mine = blk < bpt && blk * box < e && (blk + 1) * box > a;
      const int boxes = e > a ? (e + box - 1) / box - a / box : 0;
      const int row = ((u.lo + u.t0 + i) * kPgTile + blk * box) & ((1 << p.page_shift) - 1);
      if (!warp_all(paged_wait(empty + st, par, ab, site))) return;
      if (lane == 0) mbar_arrive_expect_tx(full + st, boxes * box * kParts * kRowBytes);
      __syncwarp();
      // a page that does not exist is out of the map's bounds: zeros
      if (mine) tma_load_rows(ring + st * tile_bytes + chunk * chunk_bytes + blk * box * kRowBytes, tm, full + st, chunk * 64, row, u.h, page, order);
      page = page_next;
      if (++st == kStages) {
        st = 0;
        par ^= 1;
      }
    }
  }
}

// Rows outside [a, e) of a 16-bit tile of V (chunks of 128-byte rows) become zeros, by one warp, for the MMAs behind it.
template <int KC>
__device__ __forceinline__ void paged_zero_rows(uint8_t* tile, int a, int e) {
  const int lane = threadIdx.x & 31;
  for (int x = lane; x < KC * kPgTile * 8; x += 32) {
    const int r = (x >> 3) & (kPgTile - 1);
    if (r < a || r >= e) *reinterpret_cast<uint4*>(tile + x * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Four e4m3 codes as 16-bit values, columns 0 and 2, then 1 and 3 (a permutation costs two instructions less than the order; who
// reads the result knows, paged_column()).  A code's bits, moved to where a wider format has its sign, exponent and mantissa,
// are the code's value times 2^-120 (bf16) or 2^-8 (fp16), subnormals among them; the row's factor takes that back.
template <bool kBf16>
__device__ __forceinline__ uint2 widen4(uint32_t codes) {
  constexpr int kShift = kBf16 ? 4 : 1;
  return make_uint2((codes & 0x007f007fu) * (256u >> kShift) + (codes & 0x00800080u) * 256u, (codes & 0x80008000u) | ((codes & 0x7f007f00u) >> kShift));
}
// The same in order: for K, whose columns meet those of Q.
template <bool kBf16>
__device__ __forceinline__ uint2 widen4_ordered(uint32_t codes) {
  constexpr int kShift = kBf16 ? 4 : 1;
  const uint32_t lo = __byte_perm(codes, 0, 0x1404), hi = __byte_perm(codes, 0, 0x3424);
  return make_uint2((lo & 0x80008000u) | ((lo & 0x7f007f00u) >> kShift), (hi & 0x80008000u) | ((hi & 0x7f007f00u) >> kShift));
}
// The column that a place of a widened row holds.
__host__ __device__ constexpr int paged_column(int place) { return (place & ~3) | ((place & 1) << 1) | ((place >> 1) & 1); }
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

// The factor of a key of an 8-bit cache, for its scores.
__device__ __forceinline__ float key_factor(int byte) {
  return __uint_as_float(byte == 255 ? 0x7fffffffu : byte == 0 ? 0x00400000u : static_cast<uint32_t>(byte) << 23);
}

// 8-bit caches: a warp that brings the rows' exponents, of K and of V, into a ring of slots [2][128]; a lane four rows of each,
// copied without waiting; who uses a factor makes it.  (Made here they were the bound of the whole kernel: 3800 to 6000 cycles a
// tile with the exponents in registers, 2100 behind copies.)  `full` counts 32 arrivals.  A page that does not exist gives zeros.
template <int kSlots>
__device__ __forceinline__ void paged_scales(const PagedParams& p, PagedWalk u, uint8_t* ring, uint64_t* full, uint64_t* empty, const AbortState& ab) {
  const int lane = threadIdx.x & 31;
  bool words = true;   // four rows are one word of memory
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
    words = words && p.scale_stride[kv][1] == 1 && ((p.scale_stride[kv][0] | p.scale_stride[kv][2]) & 3) == 0 && (reinterpret_cast<uintptr_t>(p.scale8[kv]) & 3) == 0;
  int st = 0;
  uint32_t par = 1;
  while (u.next()) {
    const int* table = p.table + u.b * p.table_stride;
    auto page_at = [&](int i) {
      const int block = ((u.lo + u.t0 + i) * kPgTile + 4 * lane) >> p.page_shift;
      return i < u.n && block < p.max_blocks ? table[block] : -1;
    };
    int page = page_at(0), next = page_at(1);
    for (int i = 0; i < u.n; ++i) {
      const int after = page_at(i + 2);
      const bool there = page >= 0 && page < p.pages;
      const int row = ((u.lo + u.t0 + i) * kPgTile + 4 * lane) & ((1 << p.page_shift) - 1);
      if (!warp_all(paged_wait(empty + st, par, ab, kPgScalesEmpty))) return;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint8_t* s = p.scale8[kv] + (there ? page * p.scale_stride[kv][0] + row * p.scale_stride[kv][1] + u.h * p.scale_stride[kv][2] : 0);
        uint8_t* dst = ring + (st * 2 + kv) * kPgTile + 4 * lane;
        if (words) {
          cp_async4(smem_u32(dst), s, there ? 4 : 0);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) dst[k] = there ? s[k * p.scale_stride[kv][1]] : 0;
        }
      }
      if (words) cp_async_arrive(full + st);
      else mbar_arrive(full + st);
      if (++st == kSlots) {
        st = 0;
        par ^= 1;
      }
      page = next;
      next = after;
    }
  }
}

// A query tile as codes, by kWarps warps (`ct` their threads from 0): a row's values times the power of two that brings them to
// 448 at most are sums of two (bf16) or three (fp16) 8-bit parts to all their bits, down to 2^-26 of the row's largest: e4m3,
// whose rounding leaves 1/16 of the value, then e5m2, which reach further down, 3 bits each.  Parts are part_bytes apart, rows
// of D bytes swizzled as operands; `factor` gets the powers that take the scaling back.
template <int D, bool kBf16, int kPieces, int kWarps>
__device__ __forceinline__ void paged_split_queries(const PagedParams& p, const PagedWalk& w, int first_row, int ct, uint8_t* tile, int part_bytes, float* factor) {
  constexpr int kUnits = D / 16, kStep = 32 * kWarps / kUnits;   // pieces of 16 columns of a row, rows at a time
  const int unit = ct % kUnits;
  for (int r0 = 0; r0 < p.rows; r0 += kStep) {
    const int r = r0 + ct / kUnits, i = r / p.group, g = r - i * p.group;
    const int tok = w.qt * p.per_tile + i;
    float x[16];
    uint32_t top = 0;
    const bool real = r < p.rows && tok < w.fresh;
    if (real) {
      const uint16_t* src = p.q + (p.cu != nullptr ? 0 : w.b * p.qs[0]) + (p.cu != nullptr ? first_row + tok : tok) * p.qs[1] + (w.h * p.group + g) * p.qs[2] + unit * 16;
      const uint4 lo = reinterpret_cast<const uint4*>(src)[0], hi = reinterpret_cast<const uint4*>(src)[1];
      const uint32_t words[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 f = unpack2<kBf16>(words[k]);
        x[2 * k] = f.x;
        x[2 * k + 1] = f.y;
        top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
      }
    }
#pragma unroll
    for (int d = 1; d < kUnits; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (r < p.rows) {
      const int e = max(code_exponent(top), -126);
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      const int piece = D == 128 ? unit ^ (r & 7) : unit ^ ((r >> 1) & 3);
      uint8_t* dst = tile + r * D + piece * 16;
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = real ? (top < 0x7f800000u ? x[k] * inv : __uint_as_float(0x7fffffffu)) : 0.0f;
#pragma unroll
      for (int part = 0; part < kPieces; ++part) {
        uint32_t c[4];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const __nv_fp8_interpretation_t format = part == 0 ? __NV_E4M3 : __NV_E5M2;
          const __nv_fp8x2_storage_t two = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * k], x[2 * k + 1]), __NV_SATFINITE, format);
          const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(two, format)));
          x[2 * k] -= back.x;   // exact
          x[2 * k + 1] -= back.y;
          c[k / 2] = k % 2 == 0 ? two : c[k / 2] | (static_cast<uint32_t>(two) << 16);
        }
        *reinterpret_cast<uint4*>(dst + part * part_bytes) = make_uint4(c[0], c[1], c[2], c[3]);
      }
      if (unit == 0) factor[r] = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// A tile of V from codes to 16 bits, by kWarps warps: chunks of 128-byte rows, swizzled as TMA would have written them.
template <int D, bool kBf16, int kWarps, bool kOrdered = false>
__device__ __forceinline__ void paged_widen(const uint8_t* src, const uint8_t* exponents, uint8_t* dst, int ct) {
  constexpr int kUnits = D / 16, kStep = 32 * kWarps / kUnits;   // pieces of 16 columns of a row, rows at a time
  const int unit = ct % kUnits;
  // columns 16 unit to + 15 are two 16-byte pieces of the row's chunk
  const int piece = (unit % 4) * 2, swap = (unit / 4) & 1;
  dst += unit / 4 * (kPgTile * 128);
  // Not unrolled: several roles share a scheduler's instruction cache, and straight code that runs once a tile comes from behind
  // it (unrolled by four 2000 cycles a tile, 40 % of all stalls on instructions).  The next piece is on its way meanwhile.
  const uint32_t at = smem_u32(src) + unit * 16, exponent_at = smem_u32(exponents);
  auto load_exponent = [&](int row) {
    uint32_t x;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(x) : "r"(exponent_at + row) : "memory");
    return x;
  };
  // half of the threads begin with the second half of their piece, so that eight neighbours write to all banks
  auto load_codes = [&](int row, int half) {
    uint2 x;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x.x), "=r"(x.y) : "r"(at + row * D + (half ^ swap) * 8) : "memory");
    return x;
  };
  int row = ct / kUnits;
  uint2 c0 = load_codes(row, 0), c1 = load_codes(row, 1);
  uint32_t byte = load_exponent(row);
  const uint32_t line = smem_u32(dst);
#pragma unroll 1
  while (row < kPgTile) {
    const int next = min(row + kStep, kPgTile - 1);
    const uint2 c0_next = load_codes(next, 0), c1_next = load_codes(next, 1);
    const uint32_t byte_next = load_exponent(next);
    const uint32_t c4[4] = {c0.x, c0.y, c1.x, c1.y};
    uint32_t w[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint2 x = kOrdered ? widen4_ordered<kBf16>(c4[k]) : widen4<kBf16>(c4[k]);
      w[2 * k] = x.x;
      w[2 * k + 1] = x.y;
    }
    // 2^(byte - 127) times what widen4() leaves out, in both halves of a word
    uint32_t factor = kBf16 ? (byte + 120u) * 0x00800080u : (byte - 104u) * 0x04000400u;
    if (kBf16 ? byte > 134u : byte - 105u > 29u) {   // not a 16-bit power of two: rows of very large or very small values
      const uint32_t f = row_factor<kBf16>(byte);
      factor = __byte_perm(f, 0, 0x1010);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = mul2<kBf16>(w[k], __byte_perm(f, 0, 0x3232));
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = mul2<kBf16>(w[k], factor);
    const uint32_t p0 = (piece + swap) ^ (row & 7);
    st_shared_v4(line + row * 128 + p0 * 16, make_uint4(w[0], w[1], w[2], w[3]));
    st_shared_v4(line + row * 128 + (p0 ^ 1) * 16, make_uint4(w[4], w[5], w[6], w[7]));
    row += kStep;
    c0 = c0_next;
    c1 = c1_next;
    byte = byte_next;
  }
  fence_proxy_async_smem();
  __syncwarp();
}

struct PagedPlan {
  int group, per_tile, tile_pos, rows, ctas;
  bool few;          // paged_tokens.cu, else paged_chunk.cu
  bool whole;        // units are not cut
  long long off_lse, off_cut, off_rows, bytes;
};

// The launches, by kernel; the tensor maps and parameters of a call are made by paged_setup().
int launch_paged_tokens(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status);
int launch_paged_chunk(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status);

// A kernel may have its shared memory: asked for once on each device.
template <class Kernel>
inline bool paged_allow(Kernel kernel, int bytes, std::atomic<uint64_t>& asked) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (asked.load(std::memory_order_relaxed) & bit) != 0) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (dev < 64) asked.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

struct PagedMaps {
  CUtensorMap q, k, v;
};
int paged_setup(const AttnB200PagedAttnArgs* a, const PagedPlan& d, int* status, PagedParams* p, PagedMaps* m);
// The merge behind a kernel whose units may have been cut.
int paged_merge(const AttnB200PagedAttnArgs* a, const PagedPlan& d, const PagedParams& p, cudaStream_t stream);

}  // namespace b200
