// Attention over a paged cache for units of more rows than paged_tokens.cu takes: chunks of prompts.
#include <cstring>

#include "paged_common.cuh"

namespace b200 {

constexpr int kPgConvWarps = 4;    // 8-bit caches: warps that widen codes

template <int D, bool kBf16, bool k8Bit>
struct PagedSmem {
  static constexpr int kThreads = 352 + (k8Bit ? 32 + 32 * kPgConvWarps : 0);
  static constexpr int kPieces = kBf16 ? 2 : 3;                     // 8-bit caches: parts of a query value
  static constexpr int kTileBytes = kPgTile * D * 2;                // 128 rows in 16 bits
  static constexpr int kRawBytes = kPgTile * D;                     // and as codes
  static constexpr int kKBytes = k8Bit ? kRawBytes : kTileBytes;
  static constexpr int kStagesK = k8Bit ? (D == 128 ? 4 : 8) : D == 128 ? 3 : 6, kStagesV = k8Bit ? 2 : D == 128 ? 2 : 5;
  static constexpr int kRaw = k8Bit ? (D == 128 ? (kBf16 ? 3 : 2) : 6) : 0;   // tiles of codes of V
  static constexpr int kScales = k8Bit ? 4 : 0;                      // tiles of exponents
  // query tiles; an MMA reads 128 rows from a tile's start whatever its rows, so what follows must be shared memory too
  static constexpr int kQRegion = k8Bit ? kPieces * kRawBytes : D * 256;
  static constexpr int kOffK = kQRegion;
  static constexpr int kOffV = kOffK + kStagesK * kKBytes;
  static constexpr int kOffRaw = kOffV + kStagesV * kTileBytes;
  static constexpr int kOffScales = kOffRaw + kRaw * kRawBytes;     // uint8 [kScales][2][128]
  static constexpr int kOffQs = kOffScales + kScales * 2 * kPgTile;   // float [4][128]: factors of the query rows, by unit
  static constexpr int kOffBar = kOffQs + (k8Bit ? 4 * kPgTile * 4 : 0);
  static constexpr int kQFull = 0, kQEmpty = 2, kSFull = 4, kPReady = 6, kODone = 8, kStats = 10, kOFree = 11, kKFull = 12;
  static constexpr int kKEmpty = kKFull + kStagesK, kVFull = kKEmpty + kStagesK, kVEmpty = kVFull + kStagesV;
  static constexpr int kRawFull = kVEmpty + kStagesV, kRawEmpty = kRawFull + kRaw, kScFull = kRawEmpty + kRaw, kScEmpty = kScFull + kScales;
  static constexpr int kNumBars = kScEmpty + kScales;
  static constexpr int kOffMisc = kOffBar + 8 * kNumBars;
  static constexpr int kOffMl = (kOffMisc + 16 + 15) / 16 * 16;     // float2 [128]: group 1's (reference maximum, sum) of a row
  static constexpr int kOffCum = kOffMl + 128 * 8;                  // int [batch + 1] tiles in front, [batch] lengths, [batch + 1] first rows
  static constexpr int kBytes = kOffCum + PagedTables::kBytes;   // the dynamic shared memory is declared 1024-byte aligned
  static_assert(kBytes <= 232448, "shared memory layout exceeds an SM");
};

template <int D, bool kBf16, bool k8Bit>
__global__ void __launch_bounds__(PagedSmem<D, kBf16, k8Bit>::kThreads, 1)
paged_chunk_kernel(const __grid_constant__ PagedMaps maps, const __grid_constant__ PagedParams p) {
  using L = PagedSmem<D, kBf16, k8Bit>;
  using F = SoftmaxFunctor;
  constexpr int N = kPgTile, KC = D / 64, kChunk = N * 128, kThreads = L::kThreads;
  constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256;

  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::kOffK;
  uint8_t* sV = smem + L::kOffV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBar);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 8);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::kOffMl);
  const PagedTables tab(smem + L::kOffCum);
  const FunctorArgs fa{{p.scale}};

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
      if constexpr (k8Bit) {
        if (i == L::kQFull || i == L::kQFull + 1 || (i >= L::kVFull && i < L::kVEmpty) || (i >= L::kRawEmpty && i < L::kScFull))
          count = kPgConvWarps;   // written, or read, by the warps that widen
        if (i >= L::kScFull) count = i < L::kScEmpty ? 32 : active_warps + kPgConvWarps;
      }
      mbar_init(bars + i, count);
    }
    fence_barrier_init();
    __syncwarp();
    if (lane == 0) {
      if (!k8Bit) tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
    }
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  if (tid == 0) {
    *abort_flag = (*reinterpret_cast<volatile int*>(p.status) != 0) ? 1 : 0;
    if ((smem_u32(smem) & 1023u) != 0) {   // the swizzles' patterns repeat every 1024 bytes of the shared window
      *abort_flag = 1;
      atomicCAS(p.status, 0, kStatusTimeoutBase + kPgSmemAlign);
    }
    p.cut[cta].w = -1;   // this thread writes the real one, too
  }
  tab.count(p, kThreads);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const PagedShare share(p, tab);
  const int T0 = share.t0, T1 = share.t1;
  const bool run_cta = warp_all(T1 > T0 && !*abort_flag);
  auto make_walk = [&]() { return PagedWalk(p, tab.cum, tab.len, tab.row, T0, T1); };

  if (warp == 8) {
    // ======================= loads of keys, and of queries in 16 bits =======================
    if (run_cta) {
      paged_load<k8Bit ? 1 : KC, k8Bit ? D : 128, L::kStagesK>(p, make_walk(), &maps.k, p.ok, sK, L::kKBytes, kChunk, bars + L::kKFull, bars + L::kKEmpty, ab, kPgKEmpty,
                                                             [&](const PagedWalk& u, int ui) -> bool {
        if constexpr (!k8Bit) {
          const int qb = ui % p.q_bufs;
          if (ui >= p.q_bufs && !warp_all(mbar_wait(bars + L::kQEmpty + qb, (ui / p.q_bufs - 1) & 1, ab, kPgQEmpty))) return false;
          if (lane == 0) {
            mbar_arrive_expect_tx(bars + L::kQFull + qb, KC * p.rows * 128);
            const int s = p.cu != nullptr ? tab.row[u.b] + u.qt * p.per_tile : u.qt * p.per_tile;
            for (int c = 0; c < KC; ++c)
              tma_load_rows(sQ + qb * p.q_bytes + c * (p.rows_pad * 128), &maps.q, bars + L::kQFull + qb, c * 64, s, u.h * p.group, p.cu != nullptr ? 0 : u.b, p.oq);
          }
        }
        return true;
      });
    }
  } else if (warp == 10) {
    // ======================= loads of values =======================
    if (run_cta) {
      if constexpr (k8Bit)
        paged_load<1, D, L::kRaw>(p, make_walk(), &maps.v, p.ov, smem + L::kOffRaw, L::kRawBytes, 0, bars + L::kRawFull, bars + L::kRawEmpty, ab, kPgRawEmpty,
                                  [](const PagedWalk&, int) { return true; });
      else
        paged_load<KC, 128, L::kStagesV>(p, make_walk(), &maps.v, p.ov, sV, L::kTileBytes, kChunk, bars + L::kVFull, bars + L::kVEmpty, ab, kPgVEmpty,
                                         [](const PagedWalk&, int) { return true; });
    }
  } else if (warp == 9) {
    // ======================= issuing warp (converged, one elected lane per batch) =======================
    if (run_cta) {
      constexpr uint32_t idesc_qk = make_idesc_f16(128, N, kBf16, false, false);
      constexpr uint32_t idesc_pv = make_idesc_f16(128, D, kBf16, false, true);
      auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool { return warp_all(mbar_wait_poll(bar, parity, ab, site)); };
      auto operand = [](uint32_t at) { return k8Bit && D == 64 ? make_smem_desc_64b(at) : make_smem_desc(at, 16, 1024); };
      constexpr int kQRow = k8Bit ? D : 128;   // bytes of a row of a part, or of 64 columns
      const uint64_t k_desc0 = operand(smem_u32(sK));
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
        const uint64_t a = operand(smem_u32(sQ + qb * p.q_bytes));
        const uint64_t bk = k_desc0 + static_cast<uint64_t>(st * (L::kKBytes >> 4));
        const uint64_t a_part = static_cast<uint64_t>(p.rows_pad * kQRow) >> 4;
        if (elect_one()) {
          if constexpr (k8Bit) {   // the parts of the queries against the codes as they are
#pragma unroll
            for (int part = 0; part < L::kPieces; ++part)
              umma_f8_ss<D / 32>(tmem_base + kColS + t * N, a + part * a_part, bk, make_idesc_f8(128, N, part == 0 ? 0 : 1, 0), part > 0 ? 1u : 0u);
          } else {
#pragma unroll
            for (int ch = 0; ch < KC; ++ch)
              umma_ss_x4<2, 2>(tmem_base + kColS + t * N, a + ch * a_part, bk + ch * (kChunk >> 4), idesc_qk, ch > 0 ? 1u : 0u);
          }
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
          int a, e;
          u.rows_of(i, a, e);
          if (a > 0 || e < N) paged_zero_rows<KC>(sV + st * L::kTileBytes, a, e);
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
      const RowCtx ctx{0, 0, 0, 0, p.seq, 0, &fa};   // softmax asks for the scale only
      const int g = p.head_major ? row / p.per_tile : row % p.group;
      const int qi = p.head_major ? row % p.per_tile : row / p.group;   // position in the tile
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
        // scale * log2(e) of the scores as they come: 8-bit caches leave the factor of the query row to it
        float c2 = p.scale * 1.4426950408889634f, q_factor = 1.0f;
        bool first = true;
        for (int J = J0 + ((J0 ^ t) & 1); J < J0 + u.n; J += 2) {
          mbar_wait_rows(bars + L::kSFull + t, (J >> 1) & 1, ab, kPgSFull);
          if (!any_live) {   // nothing of this warp's rows is kept
            if constexpr (k8Bit) {
              if (lane == 0) mbar_arrive(bars + L::kScEmpty + J % L::kScales);
            }
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
            // time with the next on its way, first for the maximum.  Each is times its key's factor.  P goes over what has been read.
            const int slot = J % L::kScales;
            if (first) {   // the queries of the unit are there: so are their factors
              q_factor = reinterpret_cast<const float*>(smem + L::kOffQs)[(ui & 3) * N + row];
              c2 *= q_factor;
              first = false;
            }
            mbar_wait_rows(bars + L::kScFull + slot, (J / L::kScales) & 1, ab, kPgScales);
            const uint32_t* kf = reinterpret_cast<const uint32_t*>(smem + L::kOffScales + slot * 2 * N);
            auto scores = [&](float (&s)[32], int c) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const uint32_t f = kf[c * 8 + i / 4];
                mul_x2(s[i], s[i + 1], key_factor(f & 255), key_factor((f >> 8) & 255));
                mul_x2(s[i + 2], s[i + 3], key_factor((f >> 16) & 255), key_factor(f >> 24));
              }
              if (edge) {
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = c * 32 + i < e && c * 32 + i >= a ? s[i] : -INFINITY;
              }
            };
            float mx = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < N / 32; c += 2) {
              float x[2][32];
              tmem_ld32f(tS + c * 32, x[0]);
              tmem_ld32f(tS + c * 32 + 32, x[1]);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                scores(x[k], c + k);
                float m0 = x[k][0], m1 = x[k][1];
#pragma unroll
                for (int i = 2; i + 4 <= 32; i += 4) {
                  m0 = max3(m0, x[k][i], x[k][i + 2]);
                  m1 = max3(m1, x[k][i + 1], x[k][i + 3]);
                }
                mx = max3(mx, max3(m0, x[k][30], x[k][31]), m1);
              }
            }
            if ((mx - rs[0]) * c2 > 8.0f) {
              o_scale = fast_exp2((rs[0] - mx) * c2);
              rs[0] = mx;
              rs[1] *= o_scale;
            }
            const float neg = -rs[0] * c2;
            float a0 = 0.f, a1 = 0.f;
#pragma unroll 1
            for (int c = 0; c < N / 32; c += 2) {
              float x[2][32];
              tmem_ld32f(tS + c * 32, x[0]);
              tmem_ld32f(tS + c * 32 + 32, x[1]);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                scores(x[k], c + k);
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  fma_x2(x[k][2 * i], x[k][2 * i + 1], c2, c2, neg, neg);
                  x[k][2 * i] = fast_exp2(x[k][2 * i]);
                  x[k][2 * i + 1] = fast_exp2(x[k][2 * i + 1]);
                  add_x2(a0, a1, x[k][2 * i], x[k][2 * i + 1]);
                  pk[i] = pack2<kBf16>(x[k][2 * i], x[k][2 * i + 1]);
                }
                tmem_st16(tS + (c + k) * 16, pk);
              }
            }
            rs[1] += a0 + a1;
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + L::kScEmpty + slot);
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
        const float lse = sum == 0.0f ? -INFINITY : logf(sum) + m * (p.scale * q_factor);
        const int head = u.h * p.group + g;
        const bool whole = u.n == u.total;
        // a partial result: the unit's first share leaves it in the second slot of its CTA, the later ones in the first
        const long long slot = (2LL * blockIdx.x + (u.t0 == 0 ? 1 : 0)) * p.rows + row;
        const long long at = p.cu != nullptr ? tab.row[u.b] + tok : tok;   // row of o
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
            if constexpr (k8Bit) {   // columns in their order
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float x = a0[i + 1];
                a0[i + 1] = a0[i + 2];
                a0[i + 2] = x;
              }
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
          p.cut[cta] = make_int4(u.b, u.h, u.qt, pg_owner(u.t - u.n + u.total - 1, share.shares, share.total));
        tc_fence_before_sync();
        mbar_arrive(bars + L::kOFree);
      }
    }
  } else if constexpr (k8Bit) {
    if (warp == 11) {
      if (run_cta)
        paged_scales<L::kScales>(p, make_walk(), smem + L::kOffScales, bars + L::kScFull, bars + L::kScEmpty, ab);
    } else if (run_cta) {
      // ======================= queries in parts, and V in 16 bits =======================
      const int ct = tid - 384;
      PagedWalk u = make_walk(), ahead = make_walk();
      auto split = [&](int ui) -> bool {
        const int qb = ui % p.q_bufs;
        if (ui >= p.q_bufs && !warp_all(mbar_wait(bars + L::kQEmpty + qb, (ui / p.q_bufs - 1) & 1, ab, kPgQEmpty))) return false;
        paged_split_queries<D, kBf16, L::kPieces, kPgConvWarps>(p, ahead, tab.row[ahead.b], ct, sQ + qb * p.q_bytes, p.rows_pad * D,
                                                               reinterpret_cast<float*>(smem + L::kOffQs) + (ui & 3) * N);
        if (lane == 0) mbar_arrive(bars + L::kQFull + qb);
        return true;
      };
      ahead.next();
      bool ok = split(0);
      int J = 0;
      for (int ui = 0; ok && u.next(); ++ui) {
        const bool more = ahead.next();
        if (more && p.q_bufs == 2) ok = split(ui + 1);   // else when the unit's last scores are under way
        for (int i = 0; i < u.n && ok; ++i, ++J) {
          const int sc = J % L::kScales, raw = J % L::kRaw, st = J % L::kStagesV;
          ok = warp_all(paged_wait(bars + L::kScFull + sc, (J / L::kScales) & 1, ab, kPgScales));
          ok = ok && warp_all(paged_wait(bars + L::kRawFull + raw, (J / L::kRaw) & 1, ab, kPgRawFull));
          ok = ok && warp_all(paged_wait(bars + L::kVEmpty + st, ((J / L::kStagesV) & 1) ^ 1, ab, kPgVEmpty));
          if (!ok) break;
          paged_widen<D, kBf16, kPgConvWarps>(smem + L::kOffRaw + raw * L::kRawBytes, smem + L::kOffScales + (sc * 2 + 1) * N, sV + st * L::kTileBytes, ct);
          if (lane == 0) {
            mbar_arrive(bars + L::kVFull + st);
            mbar_arrive(bars + L::kRawEmpty + raw);
            mbar_arrive(bars + L::kScEmpty + sc);
          }
        }
        if (more && ok && p.q_bufs == 1) ok = split(ui + 1);
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

template <int D, bool kBf16, bool k8Bit>
int launch_chunk(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status) {
  using L = PagedSmem<D, kBf16, k8Bit>;
  PagedParams p;
  PagedMaps maps;
  const int rc = paged_setup(a, d, status, &p, &maps);
  if (rc != ATTN_B200_OK) return rc;
  p.q_bytes = k8Bit ? L::kPieces * p.rows_pad * D : (D / 64) * p.rows_pad * 128;
  p.q_bufs = 2 * p.q_bytes <= L::kQRegion ? 2 : 1;
  auto kernel = paged_chunk_kernel<D, kBf16, k8Bit>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes) != cudaSuccess) {
    cudaGetLastError();
    return ATTN_B200_E_LAUNCH;
  }
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
