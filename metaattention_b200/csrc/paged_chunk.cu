// Attention over a paged cache for units of many query rows: chunks of prompts.  Bound by the tensor pipe and the exponentials.
//
// A unit is two tiles of 128 query rows of one KV head (half of the reads of K and V that one tile makes: at 128 rows to 64 KB of
// keys and values the L2 cache is the bound); each KV tile meets both.
//   softmax          16-bit caches: two threads to a query row, eight warps to a query tile.  The scores leave their buffer for
//                    registers as soon as they are there and P has columns of its own, so the next scores are computed under the
//                    exponentials.  8-bit caches: four warps to a tile (the others widen), which have no room for a row and read
//                    its scores twice, P over them; the tile's next scores wait for its P.V, the other tile's runs beside it.
//   four warps       loads of K and Q, of V; issue S = Q K^T, O += P V: with one warp for both its waits and bookkeeping stood in
//                    front of an idle pipe, 2130 cycles for a tile of 128 x 128 where the pipe needs 1024
//   eight more       8-bit caches: exponents of the rows; K and V in 16 bits (paged_common.cuh)
// P is rounded to q's type, the operand's; its sum is taken of the unrounded values, in 32 bits.  (Error of o against 64 bits, relative
// in the norm: 0.0023 in bf16 where the rounding of o alone gives 0.0017, as in the dense kernels; a P in two parts would double P V.)
// Measured: twice 1024 new tokens on 16384, 32 heads on 8 KV heads of 128: 557-568 us behind one another, at the capped clock (1.36 GHz),
// 940-955 TFLOP/s; 64 columns 384-390; 8 bits 694-700, 64 columns 550.  A step (a KV tile, both query tiles) is 3100 cycles of that
// call (670 k for 215 steps): each of the tensor pipe and the special-function unit needs 2048 of them and neither is full (63 and 67 %);
// a step of one query tile is 2100, the chain of scores, exponentials, P and product; a unit's beginning and end 4000 to 6000.
#include <cstring>

#include "paged_common.cuh"

namespace b200 {

template <int D, bool k8Bit>
struct ChunkSmem {
  static constexpr int kConvWarps = 7;                               // with them twenty warps: 96 registers a thread
  static constexpr int kRowThreads = k8Bit ? 1 : 2;                  // threads of a query row
  static constexpr int kSoftmaxWarps = 8 * kRowThreads;
  static constexpr int kThreads = (kSoftmaxWarps + 4) * 32 + (k8Bit ? 32 + 32 * kConvWarps : 0);
  static constexpr int kScores = k8Bit || D == 64 ? 2 : 1;           // score buffers: one for each query tile, or one in turn
  static constexpr int kTileBytes = kPgTile * D * 2, kRawBytes = kPgTile * D;
  static constexpr int kStagesK = D == 128 ? 2 : 4, kStagesV = D == 128 ? (k8Bit ? 1 : 2) : 4;
  static constexpr int kRawK = k8Bit ? (D == 128 ? 2 : 3) : 0, kRawV = k8Bit ? (D == 128 ? 1 : 2) : 0;   // tiles of codes
  static constexpr int kScales = k8Bit ? 4 : 0;                      // tiles of exponents
  static constexpr int kQBufs = D == 64 && !k8Bit ? 2 : 1;                     // units whose queries are there
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kOffQ + kQBufs * 2 * kTileBytes;
  static constexpr int kOffV = kOffK + kStagesK * kTileBytes;
  static constexpr int kOffRawK = kOffV + kStagesV * kTileBytes;
  static constexpr int kOffRawV = kOffRawK + kRawK * kRawBytes;
  static constexpr int kOffScales = kOffRawV + kRawV * kRawBytes;    // uint8 [kScales][2][128]
  static constexpr int kOffBar = kOffScales + kScales * 2 * kPgTile;
  static constexpr int kQFull = 0, kQEmpty = 2, kSFull = 4, kPReady = 6, kODone = 8, kOFree = 10, kKFull = 12, kKEmpty = kKFull + kStagesK;
  static constexpr int kVFull = kKEmpty + kStagesK, kVEmpty = kVFull + kStagesV, kRawKFull = kVEmpty + kStagesV, kRawKEmpty = kRawKFull + kRawK;
  static constexpr int kRawVFull = kRawKEmpty + kRawK, kRawVEmpty = kRawVFull + kRawV, kScFull = kRawVEmpty + kRawV, kScEmpty = kScFull + kScales;
  static constexpr int kSFree = kScEmpty + kScales, kNumBars = kSFree + 2;   // the scores of a buffer are in registers
  static constexpr int kOffMisc = kOffBar + 8 * kNumBars;
  static constexpr int kOffExchange = kOffMisc + 16;                 // float [2][2][2][128]: by step, tile and half, the row's
  static constexpr int kOffTables = kOffExchange + (k8Bit ? 0 : 8 * kPgTile * 4);
  static constexpr int kBytes = kOffTables + PagedTables::kBytes;    // the dynamic shared memory is declared 1024-byte aligned
  static_assert(kBytes <= 232448, "shared memory layout exceeds an SM");
};

template <int D, bool kBf16, bool k8Bit>
__global__ void __launch_bounds__(ChunkSmem<D, k8Bit>::kThreads, 1)
paged_chunk_kernel(const __grid_constant__ PagedMaps maps, const __grid_constant__ PagedParams p) {
  using L = ChunkSmem<D, k8Bit>;
  using F = SoftmaxFunctor;
  constexpr int N = kPgTile, KC = D / 64, kChunk = N * 128;
  constexpr int kKWarp = L::kSoftmaxWarps, kVWarp = kKWarp + 1, kQkWarp = kKWarp + 2, kPvWarp = kKWarp + 3;
  // accumulators; P, or P over the scores; scores
  constexpr uint32_t kTmemCols = 512, kColO = 0, kColS = 512 - L::kScores * N, kColP = k8Bit ? kColS : 2 * D, kPStep = k8Bit ? N : N / 2;
  static_assert(kColP + (k8Bit ? 0 : N) <= kColS && 2 * D <= kColS, "tensor memory layout");

  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem + L::kOffQ;
  uint8_t* sK = smem + L::kOffK;
  uint8_t* sV = smem + L::kOffV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 8);
  const PagedTables tab(smem + L::kOffTables);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = static_cast<int>(blockIdx.x);
  const AbortState ab{abort_flag, p.status};

  // The merge kernel may be made ready ahead of this kernel's own tensor memory: shared memory keeps every other kernel with
  // tensor memory off the SM.
  static_assert(L::kBytes + 65536 > 233472, "a CTA with tensor memory could share the SM");
  pdl_launch_dependents();

  if (warp == kQkWarp) {
    for (int i = lane; i < L::kNumBars; i += 32) {
      int count = 1;
      if ((i >= L::kPReady && i < L::kODone) || (i >= L::kOFree && i < L::kKFull) || i >= L::kSFree) count = 4 * L::kRowThreads;
      if constexpr (k8Bit) {   // written, or read, by the warps that widen
        if ((i >= L::kKFull && i < L::kKEmpty) || (i >= L::kVFull && i < L::kVEmpty) || (i >= L::kRawKEmpty && i < L::kRawVFull) || (i >= L::kRawVEmpty && i < L::kScFull))
          count = L::kConvWarps;
        if (i >= L::kScFull && i < L::kSFree) count = i < L::kScEmpty ? 32 : L::kConvWarps;
      }
      mbar_init(bars + i, count);
    }
    fence_barrier_init();
    __syncwarp();
    if (lane == 0) {
      tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
    }
  }
  if (warp == kPvWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // head of the group, and position in the tile, of a softmax thread's row
  const int row_of_tile = (warp & 3) * 32 + lane, by = p.head_major ? p.tile_pos : p.group, high = row_of_tile / by, low = row_of_tile - high * by;
  const int g = p.head_major ? high : low, qi = p.head_major ? low : high;
  pdl_wait();
  if (tid == 0) {
    *abort_flag = (*reinterpret_cast<volatile int*>(p.status) != 0) ? 1 : 0;
    if ((smem_u32(smem) & 1023u) != 0) {   // the swizzles' patterns repeat every 1024 bytes of the shared window
      *abort_flag = 1;
      atomicCAS(p.status, 0, kStatusTimeoutBase + kPgSmemAlign);
    }
    p.cut[cta].w = -1;   // this thread writes the real one, too
  }
  tab.count(p, L::kThreads);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const PagedShare share(p, tab);
  const bool run_cta = warp_all(share.t1 > share.t0 && !*abort_flag);
  auto make_walk = [&]() { return PagedWalk(p, tab.cum, tab.len, tab.row, tab.start, share.t0, share.t1); };
  // keys [begin, end) that any row of the unit's query tile t sees
  auto keys_of = [&](const PagedWalk& u, int t, int& begin, int& end) {
    const int tok = u.qt * p.per_tile + t * p.tile_pos, n = min(p.tile_pos, u.fresh - tok);   // the tile's tokens
    const int first = u.len - u.fresh + tok, last = first + n - 1;
    end = n <= 0 || (t == 1 && p.per_tile <= p.tile_pos) ? 0 : p.causal ? min(u.len, last + 1) : u.len;
    begin = p.window > 0 ? max(0, first - p.window + 1) : 0;
  };

  if (!run_cta) {
  } else if (warp == kKWarp) {
    // ======================= loads of keys and queries =======================
    paged_load<k8Bit ? 1 : KC, k8Bit ? D : 128, k8Bit ? L::kRawK : L::kStagesK>(
        p, make_walk(), &maps.k, p.ok, k8Bit ? smem + L::kOffRawK : sK, k8Bit ? L::kRawBytes : L::kTileBytes, kChunk, bars + (k8Bit ? L::kRawKFull : L::kKFull),
        bars + (k8Bit ? L::kRawKEmpty : L::kKEmpty), ab, kPgKEmpty, [&](const PagedWalk& u, int ui) -> bool {
          const int qb = ui % L::kQBufs;
          if (ui >= L::kQBufs && !warp_all(paged_wait(bars + L::kQEmpty + qb, (ui / L::kQBufs - 1) & 1, ab, kPgQEmpty))) return false;
          if (lane == 0) {
            const int tiles = p.per_tile > p.tile_pos ? 2 : 1;
            mbar_arrive_expect_tx(bars + L::kQFull + qb, tiles * KC * p.tile_pos * p.group * 128);
            const int s = (p.cu != nullptr ? tab.row[u.b] : 0) + u.qt * p.per_tile;
            for (int t = 0; t < tiles; ++t)
              for (int c = 0; c < KC; ++c)
                tma_load_rows(sQ + (qb * 2 + t) * L::kTileBytes + c * kChunk, &maps.q, bars + L::kQFull + qb, c * 64, s + t * p.tile_pos, u.h * p.group, p.cu != nullptr ? 0 : u.b, p.oq);
          }
          return true;
        });
  } else if (warp == kVWarp) {
    // ======================= loads of values =======================
    paged_load<k8Bit ? 1 : KC, k8Bit ? D : 128, k8Bit ? L::kRawV : L::kStagesV>(
        p, make_walk(), &maps.v, p.ov, k8Bit ? smem + L::kOffRawV : sV, k8Bit ? L::kRawBytes : L::kTileBytes, kChunk, bars + (k8Bit ? L::kRawVFull : L::kVFull),
        bars + (k8Bit ? L::kRawVEmpty : L::kVEmpty), ab, kPgVEmpty, [](const PagedWalk&, int) { return true; });
  } else if (warp == kQkWarp || warp == kPvWarp) {
    // ======================= issue S = Q K^T and O += P V (converged, one elected lane a batch) =======================
    auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool { return warp_all(paged_wait(bar, parity, ab, site)); };
    PagedWalk u = make_walk();
    bool ok = true;
    int st = 0, own[2] = {0, 0}, all = 0;   // scores, or products, so far of each query tile, and of both
    uint32_t par = 0;
    if (warp == kQkWarp) {
      constexpr uint32_t idesc = make_idesc_f16(128, N, kBf16, false, false);
      const uint64_t q_desc0 = make_smem_desc(smem_u32(sQ), 16, 1024), k_desc0 = make_smem_desc(smem_u32(sK), 16, 1024);
      for (int ui = 0; ok && u.next(); ++ui) {
        int begin[2], end[2];
        keys_of(u, 0, begin[0], end[0]);
        keys_of(u, 1, begin[1], end[1]);
        const int qb = ui % L::kQBufs;
        ok = wait(bars + L::kQFull + qb, (ui / L::kQBufs) & 1, kPgQFull);
        for (int i = 0; i < u.n && ok; ++i) {
          const int kv0 = (u.lo + u.t0 + i) * N;
          ok = wait(bars + L::kKFull + st, par, kPgKFull);
          const uint64_t bk = k_desc0 + static_cast<uint64_t>(st * (L::kTileBytes >> 4));
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || kv0 >= end[t] || kv0 + N <= begin[t]) continue;
            const int buf = L::kScores == 2 ? t : 0, use = L::kScores == 2 ? own[t] : all;
            if (k8Bit) {
              if (own[t] > 0) ok = wait(bars + L::kODone + t, (own[t] - 1) & 1, kPgODone);   // the P in these columns has been read
            } else if (use > 0) {
              ok = wait(bars + L::kSFree + buf, (use - 1) & 1, kPgSFree);
            }
            if (!ok) continue;
            tc_fence_after_sync();
            const uint64_t a = q_desc0 + static_cast<uint64_t>((qb * 2 + t) * (L::kTileBytes >> 4));
            if (elect_one()) {
#pragma unroll
              for (int ch = 0; ch < KC; ++ch)
                umma_ss_x4<2, 2>(tmem_base + kColS + buf * N, a + ch * (kChunk >> 4), bk + ch * (kChunk >> 4), idesc, ch > 0 ? 1u : 0u);
              umma_commit(bars + L::kSFull + t);
            }
            ++own[t];
            ++all;
          }
          if (ok && elect_one()) {   // behind the tile's scores, if any
            umma_commit(bars + L::kKEmpty + st);
            if (i == u.n - 1) umma_commit(bars + L::kQEmpty + qb);
          }
          __syncwarp();
          if (++st == L::kStagesK) {
            st = 0;
            par ^= 1;
          }
        }
      }
    } else {
      constexpr uint32_t idesc = make_idesc_f16(128, D, kBf16, false, true);
      const uint64_t v_desc0 = make_smem_desc(smem_u32(sV), kChunk, 1024);
      for (int ui = 0; ok && u.next(); ++ui) {
        int begin[2], end[2];
        keys_of(u, 0, begin[0], end[0]);
        keys_of(u, 1, begin[1], end[1]);
        bool begun[2] = {false, false};
        for (int i = 0; i < u.n && ok; ++i) {
          const int kv0 = (u.lo + u.t0 + i) * N;
          ok = wait(bars + L::kVFull + st, par, kPgVFull);
          if (!ok) break;
          int a, e;
          u.rows_of(i, a, e);
          if (a > 0 || e < N) paged_zero_rows<KC>(sV + st * L::kTileBytes, a, e);
          const uint64_t bv = v_desc0 + static_cast<uint64_t>(st * (L::kTileBytes >> 4));
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || kv0 >= end[t] || kv0 + N <= begin[t]) continue;
            if (!begun[t] && ui > 0) ok = wait(bars + L::kOFree + t, (ui - 1) & 1, kPgOFree);   // the last unit's rows have been read
            ok = ok && wait(bars + L::kPReady + t, own[t] & 1, kPgPReady);
            if (!ok) continue;
            tc_fence_after_sync();
            if (elect_one()) {
#pragma unroll
              for (int g = 0; g < N / 64; ++g)
                umma_ts_x4<8, 128>(tmem_base + kColO + t * D, tmem_base + kColP + t * kPStep + g * 32, bv + g * 512, idesc, (begun[t] || g > 0) ? 1u : 0u);
              umma_commit(bars + L::kODone + t);
            }
            begun[t] = true;
            ++own[t];
          }
          if (ok && elect_one()) umma_commit(bars + L::kVEmpty + st);
          __syncwarp();
          if (++st == L::kStagesV) {
            st = 0;
            par ^= 1;
          }
        }
      }
    }
  } else if (warp < L::kSoftmaxWarps) {
    // ======================= softmax =======================
    constexpr int RT = L::kRowThreads, TC = N / RT, OC = D / RT;   // threads of a row; columns of a thread, of scores and of o
    const int t = warp / (4 * RT), half = RT == 1 ? 0 : (warp >> 2) & 1;
    const int row = row_of_tile;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_base + lane_base + kColS + (L::kScores == 2 ? t * N : 0) + half * TC;
    const uint32_t tP = tmem_base + lane_base + kColP + t * kPStep + half * (TC / 2);
    const uint32_t tO = tmem_base + lane_base + kColO + t * D + half * OC;
    const int pair_bar = 1 + t * 4 + (warp & 3);   // of the two warps that share rows
    float* xch = reinterpret_cast<float*>(smem + L::kOffExchange) + t * 2 * N + row;
    int exchanges = 0;   // two buffers in turn: the partner may still read the last one's
    auto exchange = [&](float mine) -> float {
      float* x = xch + (exchanges++ & 1) * (4 * N);
      x[half * N] = mine;
      named_sync(pair_bar, 64);
      return x[(half ^ 1) * N];
    };
    const FunctorArgs fa{{p.scale}};
    const RowCtx ctx{0, 0, 0, 0, p.seq, 0, &fa};   // softmax asks for the scale only
    const float c2 = p.scale * 1.4426950408889634f;
    PagedWalk u = make_walk();
    int own = 0;   // tiles so far
    for (int ui = 0; u.next(); ++ui) {
      int begin, end;
      keys_of(u, t, begin, end);
      const int tok = u.qt * p.per_tile + t * p.tile_pos + qi;   // the row's new token
      const bool live = row < p.tile_pos * p.group && tok < u.fresh && t * p.tile_pos < p.per_tile;
      const bool any_live = __any_sync(0xffffffffu, live);
      const int pos = u.len - u.fresh + tok;
      // keys of the row; those of a row that does not exist are not looked at
      const int key_end = live ? min(u.end, p.causal ? pos + 1 : u.len) : 0x3fffffff;
      const int key_begin = live && p.window > 0 ? pos - p.window + 1 : 0;
      float rs[2];
      F::init(rs, ctx);
      bool begun = false;
      // the walk waits in memory: its registers belong to the row's scores
      const int kv_first = (u.lo + u.t0) * N, kv_last = kv_first + u.n * N;
      asm volatile("" ::"l"(&u) : "memory");
#pragma unroll 1
      for (int kv0 = kv_first; kv0 < kv_last; kv0 += N) {
        if (kv0 >= end || kv0 + N <= begin) continue;
        paged_wait(bars + L::kSFull + t, own & 1, ab, kPgSFull);
        ++own;
        if (!any_live) {   // nothing of this warp's rows is kept
          // (its arrivals keep in step: one for the next P before the last P.V would count for that)
          if (!k8Bit && begun) paged_wait(bars + L::kODone + t, own & 1, ab, kPgODone);
          begun = true;
          __syncwarp();
          if (lane == 0) {
            if (!k8Bit) mbar_arrive(bars + L::kSFree + (L::kScores == 2 ? t : 0));
            mbar_arrive(bars + L::kPReady + t);
          }
          continue;
        }
        tc_fence_after_sync();
        const int e = key_end - kv0, a = key_begin - kv0;
        const bool edge = __any_sync(0xffffffffu, e < N || a > 0);
        float o_scale = 1.0f;
        if constexpr (!k8Bit) {
          float s[TC];
#pragma unroll
          for (int c = 0; c < TC / 32; ++c) tmem_ld32f(tS + c * 32, &s[c * 32]);
          tmem_wait_ld();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + L::kSFree + (L::kScores == 2 ? t : 0));
          if (edge) {   // mostly on one side
            const int e1 = e - half * TC, a1 = a - half * TC;
            if (__any_sync(0xffffffffu, e1 < TC)) {
#pragma unroll
              for (int k = 0; k < TC; ++k) s[k] = k < e1 ? s[k] : -INFINITY;
            }
            if (__any_sync(0xffffffffu, a1 > 0)) {
#pragma unroll
              for (int k = 0; k < TC; ++k) s[k] = k >= a1 ? s[k] : -INFINITY;
            }
          }
          o_scale = F::template tile_pieces<TC, TC / 32>(s, rs, ctx, [&](float mx) { return fmaxf(mx, exchange(mx)); }, [&](int c) {
            if (c == 0 && begun) {   // P's columns are free, and the accumulator is, behind the tile's last P.V
              mbar_wait_rows(bars + L::kODone + t, own & 1, ab, kPgODone);   // (in line: a call would cost the row's registers)
              tc_fence_after_sync();
            }
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) pk[k] = pack2<kBf16>(s[c * 32 + 2 * k], s[c * 32 + 2 * k + 1]);
            tmem_st16(tP + c * 16, pk);
          });
        } else {
          // twice, 32 columns at a time: for the maximum, then for P, over what has been read
          auto scores = [&](float (&s)[32], int c) {
            if (edge) {
#pragma unroll
              for (int k = 0; k < 32; ++k) s[k] = c + k < e && c + k >= a ? s[k] : -INFINITY;
            }
          };
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < N; c += 32) {
            float s[32];
            tmem_ld32f(tS + c, s);
            tmem_wait_ld();
            scores(s, c);
            float m0 = s[0], m1 = s[1];
#pragma unroll
            for (int k = 2; k + 4 <= 32; k += 4) {
              m0 = max3(m0, s[k], s[k + 2]);
              m1 = max3(m1, s[k + 1], s[k + 3]);
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
          for (int c = 0; c < N; c += 32) {
            float s[32];
            tmem_ld32f(tS + c, s);
            tmem_wait_ld();
            scores(s, c);
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              fma_x2(s[2 * k], s[2 * k + 1], c2, c2, neg, neg);
              s[2 * k] = fast_exp2(s[2 * k]);
              s[2 * k + 1] = fast_exp2(s[2 * k + 1]);
              add_x2(a0, a1, s[2 * k], s[2 * k + 1]);
              pk[k] = pack2<kBf16>(s[2 * k], s[2 * k + 1]);
            }
            tmem_st16(tP + c / 2, pk);
          }
          rs[1] += a0 + a1;
        }
        if (begun && __any_sync(0xffffffffu, o_scale != 1.0f)) {   // (8 bits: these scores were issued behind the last P.V)
#pragma unroll 1
          for (int c = 0; c < OC / 32; ++c) {
            float o[32];
            tmem_ld32f(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= o_scale;
            tmem_st32f(tO + c * 32, o);
          }
        }
        begun = true;
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + L::kPReady + t);
      }
      // ---- end of a unit ----
      if (begun) paged_wait(bars + L::kODone + t, (own - 1) & 1, ab, kPgODone);
      if constexpr (RT == 2) {
        rs[1] += exchange(rs[1]);
        if (!named_sync_and(pair_bar, 64, !*abort_flag)) break;
      } else {
        if (!warp_all(!*abort_flag)) break;
      }
      tc_fence_after_sync();
      const float sum = rs[1], inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // no key: 0, and -inf
      const float lse = sum == 0.0f ? -INFINITY : logf(sum) + rs[0] * p.scale;
      const int head = u.h * p.group + g;
      const bool whole = u.n == u.total;
      // a partial result: the unit's first share leaves it in the second slot of its CTA, the later ones in the first
      const long long slot = (2LL * cta + (u.t0 == 0 ? 1 : 0)) * p.rows;
      const long long at = p.cu != nullptr ? tab.row[u.b] + tok : tok;   // row of o
      uint16_t* orow = static_cast<uint16_t*>(p.o) + (p.cu != nullptr ? 0 : u.b * p.o_sb) + at * p.o_ss + head * p.o_sh + half * OC;
      if (any_live) {
#pragma unroll 1
        for (int c = 0; c < OC / 32; ++c) {
          float o[32];
          tmem_ld32f(tO + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = begun ? o[k] * inv : 0.0f;
          if constexpr (k8Bit) {   // columns in their order
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              const float x = o[k + 1];
              o[k + 1] = o[k + 2];
              o[k + 2] = x;
            }
          }
          if (live) {
            if (whole) {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                uint4 pk;
                pk.x = pack2<kBf16>(o[8 * v + 0], o[8 * v + 1]);
                pk.y = pack2<kBf16>(o[8 * v + 2], o[8 * v + 3]);
                pk.z = pack2<kBf16>(o[8 * v + 4], o[8 * v + 5]);
                pk.w = pack2<kBf16>(o[8 * v + 6], o[8 * v + 7]);
                reinterpret_cast<uint4*>(orow + c * 32)[v] = pk;
              }
            } else {
              float4* dst = reinterpret_cast<float4*>(p.part_o + slot * D) + (half * (OC / 4) + c * 8) * p.rows + t * N + row;
#pragma unroll
              for (int v = 0; v < 8; ++v) dst[v * p.rows] = make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
            }
          }
        }
        if (live && half == 0) {
          if (!whole) p.part_lse[slot + t * N + row] = lse;
          else if (p.lse != nullptr) p.lse[(p.cu != nullptr ? static_cast<long long>(head) : static_cast<long long>(u.b) * p.heads + head) * p.seq + at] = lse;
        }
      }
      if (tid == 0 && !whole && u.t0 == 0) {
        p.cut[cta] = make_int4(u.b, u.h, u.qt, pg_owner(u.last, share.shares, share.total));
        p.cut_rows[cta] = make_int2(p.cu != nullptr ? tab.row[u.b] : 0, u.fresh);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + L::kOFree + t);
    }
  } else if constexpr (k8Bit) {
    if (warp == 12) {
      paged_scales<L::kScales>(p, make_walk(), smem + L::kOffScales, bars + L::kScFull, bars + L::kScEmpty, ab);
    } else {
      // ======================= K and V in 16 bits, K a tile ahead =======================
      const int ct = tid - 416;
      int n = 0;   // tiles of the share
      for (PagedWalk u = make_walk(); u.next();) n += u.n;
      bool ok = true;
      for (int j = 0; j <= n && ok; ++j) {
        if (j < n) {
          const int sc = j % L::kScales, raw = j % L::kRawK, st = j % L::kStagesK;
          ok = warp_all(paged_wait(bars + L::kScFull + sc, (j / L::kScales) & 1, ab, kPgScales));
          ok = ok && warp_all(paged_wait(bars + L::kRawKFull + raw, (j / L::kRawK) & 1, ab, kPgRawFull));
          ok = ok && warp_all(paged_wait(bars + L::kKEmpty + st, ((j / L::kStagesK) & 1) ^ 1, ab, kPgKEmpty));
          if (!ok) break;
          paged_widen<D, kBf16, L::kConvWarps, true>(smem + L::kOffRawK + raw * L::kRawBytes, smem + L::kOffScales + sc * 2 * N, sK + st * L::kTileBytes, ct);
          if (lane == 0) {
            mbar_arrive(bars + L::kKFull + st);
            mbar_arrive(bars + L::kRawKEmpty + raw);
          }
        }
        if (j > 0) {
          const int v = j - 1, sc = v % L::kScales, raw = v % L::kRawV, st = v % L::kStagesV;
          ok = warp_all(paged_wait(bars + L::kRawVFull + raw, (v / L::kRawV) & 1, ab, kPgRawFull));
          ok = ok && warp_all(paged_wait(bars + L::kVEmpty + st, ((v / L::kStagesV) & 1) ^ 1, ab, kPgVEmpty));
          if (!ok) break;
          paged_widen<D, kBf16, L::kConvWarps, false>(smem + L::kOffRawV + raw * L::kRawBytes, smem + L::kOffScales + (sc * 2 + 1) * N, sV + st * L::kTileBytes, ct);
          if (lane == 0) {
            mbar_arrive(bars + L::kVFull + st);
            mbar_arrive(bars + L::kRawVEmpty + raw);
            mbar_arrive(bars + L::kScEmpty + sc);
          }
        }
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == kPvWarp) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int D, bool kBf16, bool k8Bit>
int launch_chunk(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status) {
  using L = ChunkSmem<D, k8Bit>;
  PagedParams p;
  PagedMaps maps;
  const int rc = paged_setup(a, d, status, &p, &maps);
  if (rc != ATTN_B200_OK) return rc;
  auto kernel = paged_chunk_kernel<D, kBf16, k8Bit>;
  static std::atomic<uint64_t> asked{0};
  if (!paged_allow(kernel, L::kBytes, asked)) return ATTN_B200_E_LAUNCH;
  return launch_pdl(kernel, dim3(d.ctas), dim3(L::kThreads), L::kBytes, stream, maps, p) ? paged_merge(a, d, p, stream) : ATTN_B200_E_LAUNCH;
}

int launch_paged_chunk(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status) {
  const bool bf16 = a->dtype == ATTN_B200_DTYPE_BF16, codes = a->cache.dtype == ATTN_B200_DTYPE_E4M3;
  if (a->cache.head_dim == 64)
    return codes ? (bf16 ? launch_chunk<64, true, true>(a, d, stream, status) : launch_chunk<64, false, true>(a, d, stream, status))
                 : (bf16 ? launch_chunk<64, true, false>(a, d, stream, status) : launch_chunk<64, false, false>(a, d, stream, status));
  return codes ? (bf16 ? launch_chunk<128, true, true>(a, d, stream, status) : launch_chunk<128, false, true>(a, d, stream, status))
               : (bf16 ? launch_chunk<128, true, false>(a, d, stream, status) : launch_chunk<128, false, false>(a, d, stream, status));
}

}  // namespace b200
