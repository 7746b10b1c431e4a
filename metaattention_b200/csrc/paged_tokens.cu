// Attention over a paged cache for units of up to 32 query rows: single tokens, and a few of them, against long contexts.
// Bound by the bytes of the cache.
//
// The keys are the rows of the score tile: S^T = K Q^T (128 keys x R query rows, R = 16 or 32), P^T, O^T = V^T P (D x R).  With
// the query rows as its rows a tile of 128 x 128 has four used rows of a token with four heads to a KV head, and the one warp that
// holds them makes 128 exponentials a lane where this form makes R in each of four warps: 2200 ns a tile of an 8-bit
// cache against 1140 for its bytes (in 16 bits the bytes, 1480, hid it).  A thread has a key, so the factor of an 8-bit key is one register.
//   warps 0-7    scores from tensor memory, probabilities to shared memory as P.V's operand, alternate tiles to each of two
//                groups with accumulators and maxima of their own; the unit's rows at its end
//   8, 9         loads of K (and of Q in 16 bits), of V
//   10, 11       issue S^T = K Q^T, O^T += V^T P
//   12, 13-19    8-bit caches: exponents of the rows; queries in parts and V in 16 bits (paged_common.cuh)
// The running maximum of a row is one value for a group, in the logarithm's scale; a tile is looked at for scores more than
// 2^8 above it, by a barrier's reduction, and only then are maxima taken and the accumulator rescaled.  The sum of a row stays in
// parts, one a thread, until the unit ends.
// P is rounded to q's type, the operand's; its sum is taken of the unrounded values, in 32 bits.  (Error of o against 64 bits, relative
// in the norm: 0.0023 in bf16 where the rounding of o alone gives 0.0017, as in the dense kernels.)
// Measured: 64 sequences of up to 8192 tokens, 32 heads on 8 KV heads of 128: 209-212 us, 6.4 TB/s of the cache's bytes, 97 % of the rate
// of a copy.  8 bits, 16 sequences of up to 32768: 178-184 us, 4.1 TB/s: per tile of 128 rows the widening of V and the softmax take
// turns at the issue slots of twenty warps (54 % of them used, DRAM at 64 %); a single sequence of 333 tokens 8.2 us, start, three
// tiles and end.
// Units of 17 to 32 rows in 8 bits (32 rows of scores and sums in 96 registers, 208 bytes of spills a thread; 16 rows 12): 16 sequences of
// 16384 tokens 163 us with 20 rows, 211-220 with 32, where 16 rows take 141, and 32 in 16 bits 172.
#include <cstring>

#include "paged_common.cuh"

namespace b200 {

template <int D, int R, bool kBf16, bool k8Bit>
struct TokensSmem {
  static constexpr int kConvWarps = 7;                               // with them twenty warps: 96 registers a thread
  static constexpr int kThreads = 384 + (k8Bit ? 32 + 32 * kConvWarps : 0);
  static constexpr int kPieces = kBf16 ? 2 : 3;
  static constexpr int kScores = 4;                                  // score buffers in tensor memory
  static constexpr int kTileBytes = kPgTile * D * 2, kRawBytes = kPgTile * D;
  static constexpr int kKBytes = k8Bit ? kRawBytes : kTileBytes;
  // As much of the cache on its way as shared memory holds: 128 to 192 KB; latency times bandwidth is about 50
  static constexpr int kStagesK = k8Bit ? (D == 128 ? (R == 16 && kBf16 ? 5 : 4) : 8) : D == 128 ? 3 : 6;
  static constexpr int kStagesV = k8Bit ? 2 : D == 128 ? (R == 16 ? 3 : 2) : 5;
  static constexpr int kRaw = k8Bit ? (D == 128 ? (R == 32 && !kBf16 ? 2 : 3) : 6) : 0;
  static constexpr int kScales = k8Bit ? 8 : 0;                      // tiles of exponents
  static constexpr int kQBytes = k8Bit ? kPieces * R * D : R * D * 2;
  static constexpr int kPBytes = R * 256;
  static constexpr int kOffQ = 0;
  static constexpr int kOffP = kOffQ + 2 * kQBytes;
  static constexpr int kOffK = (kOffP + 2 * kPBytes + 1023) / 1024 * 1024;
  static constexpr int kOffV = kOffK + kStagesK * kKBytes;
  static constexpr int kOffRaw = kOffV + kStagesV * kTileBytes;
  static constexpr int kOffScales = kOffRaw + kRaw * kRawBytes;      // uint8 [kScales][2][128]
  static constexpr int kOffQs = kOffScales + kScales * 2 * kPgTile;   // float [4][R]: factors of the query rows, by unit
  // float [2][2][R] by unit and group: reference maxima, and sums; float [2][R] by group: rescales; int [2][R]: position in the
  // tile and head of the group of each row
  static constexpr int kOffRow = kOffQs + (k8Bit ? 4 * R * 4 : 0);
  static constexpr int kOffWarp = kOffRow + 12 * R * 4;              // float [8][R]: a value of each warp
  static constexpr int kOffBar = kOffWarp + 8 * R * 4;
  static constexpr int kQFull = 0, kQEmpty = 2, kPReady = 4, kODone = 6, kOFree = 8, kSFull = 10, kSFree = kSFull + kScores, kKFull = kSFree + kScores;
  static constexpr int kKEmpty = kKFull + kStagesK, kVFull = kKEmpty + kStagesK, kVEmpty = kVFull + kStagesV;
  static constexpr int kRawFull = kVEmpty + kStagesV, kRawEmpty = kRawFull + kRaw, kScFull = kRawEmpty + kRaw, kScEmpty = kScFull + kScales;
  static constexpr int kNumBars = kScEmpty + kScales;
  static constexpr int kOffMisc = kOffBar + 8 * kNumBars;
  static constexpr int kOffTables = kOffMisc + 16;
  static constexpr int kBytes = kOffTables + PagedTables::kBytes;    // the dynamic shared memory is declared 1024-byte aligned
  static_assert(kBytes <= 232448, "shared memory layout exceeds an SM");
};

// Sums over a warp's lanes of R values each, a row to every lane (to 32 / R neighbours): at each step half of the rows go to the
// partner, the other half come from it.
template <int kRows, int d>
__device__ __forceinline__ void sum_rows(float* acc, int lane) {
  if constexpr (kRows > 1) {
    constexpr int w = kRows / 2;
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int r = 0; r < w; ++r) {
      const float give = upper ? acc[r] : acc[r + w], keep = upper ? acc[r + w] : acc[r];
      acc[r] = keep + __shfl_xor_sync(0xffffffffu, give, d);
    }
    if constexpr (d > 1) sum_rows<w, d / 2>(acc, lane);
  } else {
    acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], d);
    if constexpr (d > 1) sum_rows<1, d / 2>(acc, lane);
  }
}

template <int D, int R, bool kBf16, bool k8Bit>
__global__ void __launch_bounds__(TokensSmem<D, R, kBf16, k8Bit>::kThreads, 1)
paged_tokens_kernel(const __grid_constant__ PagedMaps maps, const __grid_constant__ PagedParams p) {
  using L = TokensSmem<D, R, kBf16, k8Bit>;
  constexpr int N = kPgTile, KC = D / 64, kChunk = N * 128;
  constexpr uint32_t kTmemCols = 256, kColS = 0, kColO = L::kScores * R;
  static_assert(kColO + 4 * R <= kTmemCols, "tensor memory layout");   // accumulators by unit and group

  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem + L::kOffQ;
  uint8_t* sP = smem + L::kOffP;
  uint8_t* sK = smem + L::kOffK;
  uint8_t* sV = smem + L::kOffV;
  float* s_refs = reinterpret_cast<float*>(smem + L::kOffRow);
  float* s_sums = s_refs + 4 * R;
  float* s_rescales = s_sums + 4 * R;
  int* s_pos = reinterpret_cast<int*>(s_rescales + 2 * R);
  float* s_warps = reinterpret_cast<float*>(smem + L::kOffWarp);
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

  if (warp == 10) {
    for (int i = lane; i < L::kNumBars; i += 32) {
      int count = 1;
      if (i == L::kPReady || i == L::kPReady + 1 || (i >= L::kSFree && i < L::kKFull)) count = 4;
      if (i == L::kOFree || i == L::kOFree + 1) count = 8;
      if constexpr (k8Bit) {
        if (i == L::kQFull || i == L::kQFull + 1 || (i >= L::kVFull && i < L::kVEmpty) || (i >= L::kRawEmpty && i < L::kScFull)) count = L::kConvWarps;
        if (i >= L::kScFull) count = i < L::kScEmpty ? 32 : 4 + L::kConvWarps;
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
  if (warp == 11) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  if (p.rows < R) {   // rows of the operand that no query has
    for (int i = tid; i < 2 * L::kQBytes / 16; i += L::kThreads) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  if (tid < R) {
    s_pos[tid] = p.head_major ? tid % p.per_tile : tid / p.group;
    if (!k8Bit) s_pos[R + tid] = p.head_major ? tid / p.per_tile : tid % p.group;
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
  tab.count(p, L::kThreads);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const PagedShare share(p, tab);
  const bool run_cta = warp_all(share.t1 > share.t0 && !*abort_flag);
  auto make_walk = [&]() { return PagedWalk(p, tab.cum, tab.len, tab.row, tab.start, share.t0, share.t1); };

  if (!run_cta) {
  } else if (warp == 8) {
    // ======================= loads of keys, and of queries in 16 bits =======================
    paged_load<k8Bit ? 1 : KC, k8Bit ? D : 128, L::kStagesK>(p, make_walk(), &maps.k, p.ok, sK, L::kKBytes, kChunk, bars + L::kKFull, bars + L::kKEmpty, ab, kPgKEmpty,
                                                           [&](const PagedWalk& u, int ui) -> bool {
      if constexpr (!k8Bit) {
        const int qb = ui & 1;
        if (ui >= 2 && !warp_all(paged_wait(bars + L::kQEmpty + qb, ((ui >> 1) - 1) & 1, ab, kPgQEmpty))) return false;
        if (lane == 0) {
          mbar_arrive_expect_tx(bars + L::kQFull + qb, KC * p.rows * 128);
          const int s = p.cu != nullptr ? tab.row[u.b] + u.qt * p.per_tile : u.qt * p.per_tile;
          for (int c = 0; c < KC; ++c)
            tma_load_rows(sQ + qb * L::kQBytes + c * (R * 128), &maps.q, bars + L::kQFull + qb, c * 64, s, u.h * p.group, p.cu != nullptr ? 0 : u.b, p.oq);
        }
      }
      return true;
    });
  } else if (warp == 9) {
    // ======================= loads of values =======================
    if constexpr (k8Bit)
      paged_load<1, D, L::kRaw>(p, make_walk(), &maps.v, p.ov, smem + L::kOffRaw, L::kRawBytes, 0, bars + L::kRawFull, bars + L::kRawEmpty, ab, kPgRawEmpty,
                                [](const PagedWalk&, int) { return true; });
    else
      paged_load<KC, 128, L::kStagesV>(p, make_walk(), &maps.v, p.ov, sV, L::kTileBytes, kChunk, bars + L::kVFull, bars + L::kVEmpty, ab, kPgVEmpty,
                                       [](const PagedWalk&, int) { return true; });
  } else if (warp == 10) {
    // ======================= issues S^T = K Q^T (converged, one elected lane a batch) =======================
    auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool { return warp_all(k8Bit ? paged_wait(bar, parity, ab, site) : mbar_wait_poll(bar, parity, ab, site)); };
    auto operand = [](uint32_t at) { return k8Bit && D == 64 ? make_smem_desc_64b(at) : make_smem_desc(at, 16, 1024); };
    const uint64_t k_desc0 = operand(smem_u32(sK)), q_desc0 = operand(smem_u32(sQ));
    PagedWalk u = make_walk();
    bool ok = true;
    int J = 0, st = 0;
    uint32_t par = 0;
    for (int ui = 0; ok && u.next(); ++ui) {
      const int qb = ui & 1;
      ok = wait(bars + L::kQFull + qb, (ui >> 1) & 1, kPgQFull);
      const uint64_t bq = q_desc0 + static_cast<uint64_t>(qb * (L::kQBytes >> 4));
      for (int i = 0; i < u.n && ok; ++i, ++J) {
        const int sb = J % L::kScores;
        ok = wait(bars + L::kKFull + st, par, kPgKFull);
        if (ok && J >= L::kScores) ok = wait(bars + L::kSFree + sb, (J / L::kScores - 1) & 1, kPgSFree);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t ak = k_desc0 + static_cast<uint64_t>(st * (L::kKBytes >> 4));
        if (elect_one()) {
          if constexpr (k8Bit) {   // the codes as they are against the parts of the queries
#pragma unroll
            for (int part = 0; part < L::kPieces; ++part)
              umma_f8_ss<D / 32>(tmem_base + kColS + sb * R, ak, bq + part * ((R * D) >> 4), make_idesc_f8(128, R, 0, part == 0 ? 0 : 1), part > 0 ? 1u : 0u);
          } else {
#pragma unroll
            for (int ch = 0; ch < KC; ++ch)
              umma_ss_x4<2, 2>(tmem_base + kColS + sb * R, ak + ch * (kChunk >> 4), bq + ch * ((R * 128) >> 4), make_idesc_f16(128, R, kBf16, false, false), ch > 0 ? 1u : 0u);
          }
          umma_commit(bars + L::kSFull + sb);
          umma_commit(bars + L::kKEmpty + st);
          if (i == u.n - 1) umma_commit(bars + L::kQEmpty + qb);
        }
        if (++st == L::kStagesK) {
          st = 0;
          par ^= 1;
        }
      }
    }
  } else if (warp == 11) {
    // ======================= issues O^T += V^T P =======================
    auto wait = [&](uint64_t* bar, uint32_t parity, int site) -> bool { return warp_all(k8Bit ? paged_wait(bar, parity, ab, site) : mbar_wait_poll(bar, parity, ab, site)); };
    // V [key][column] is V^T with the columns as rows, M-major; 64 columns are given twice (the same chunk again), their second
    // results are not looked at
    const uint64_t v_desc0 = make_smem_desc(smem_u32(sV), D == 128 ? kChunk : 0, 1024);
    const uint64_t p_desc0 = make_smem_desc(smem_u32(sP), 16, 1024);
    constexpr uint32_t idesc = make_idesc_f16(128, R, kBf16, true, false);
    PagedWalk u = make_walk();
    bool ok = true;
    int J = 0, st = 0;
    uint32_t par = 0;
    for (int ui = 0; ok && u.next(); ++ui) {
      if (ui >= 2) ok = wait(bars + L::kOFree + (ui & 1), ((ui >> 1) - 1) & 1, kPgOFree);   // the accumulator has been read
      for (int i = 0; i < u.n && ok; ++i, ++J) {
        ok = wait(bars + L::kVFull + st, par, kPgVFull);
        if (!ok) break;
        int a, e;
        u.rows_of(i, a, e);
        if (a > 0 || e < N) paged_zero_rows<KC>(sV + st * L::kTileBytes, a, e);
        ok = wait(bars + L::kPReady + (J & 1), (J >> 1) & 1, kPgPReady);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t av = v_desc0 + static_cast<uint64_t>(st * (L::kTileBytes >> 4));
        const uint64_t bp = p_desc0 + static_cast<uint64_t>((J & 1) * (L::kPBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int g = 0; g < N / 64; ++g)   // 16 keys a step: 2048 bytes of V, 32 of P
            umma_ss_x4<128, 2>(tmem_base + kColO + ((ui & 1) * 2 + (J & 1)) * R, av + g * 512, bp + g * ((R * 128) >> 4), idesc, (i >= 2 || g > 0) ? 1u : 0u);
          umma_commit(bars + L::kODone + (J & 1));
          umma_commit(bars + L::kVEmpty + st);
        }
        if (++st == L::kStagesV) {
          st = 0;
          par ^= 1;
        }
      }
    }
  } else if (warp < 8) {
    // ======================= scores and probabilities: a key a thread, alternate tiles to each of two groups of four warps;
    // the unit's rows at its end: a column of o a thread, alternate rows =======================
    const int group = warp >> 2, key0 = tid & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_base + lane_base + kColS, tO = tmem_base + lane_base + kColO;
    const float c2 = p.scale * 1.4426950408889634f;
    // P [row][key], 64 keys to a 128-byte row of a chunk; a buffer for each group
    const uint32_t line = smem_u32(sP) + group * L::kPBytes + (key0 >> 6) * (R * 128) + (key0 & 7) * 2, p_piece = (key0 >> 3) & 7;
    float *s_rescale = s_rescales + group * R, *s_warp = s_warps + group * 4 * R;
    auto sync = [&]() { named_sync(1 + group, 128); };
    auto head_of = [&](const PagedWalk& u, int r) -> int {   // 8 bits: divided, since the table's registers make the loop spill (240 us for 179: 16 sequences, up to 32768 keys)
      return u.h * p.group + (!k8Bit ? s_pos[R + r] : p.head_major ? r / p.per_tile : r - s_pos[r] * p.group);
    };
    auto load_rows = [&](uint32_t at, float (&x)[R]) {
      if constexpr (R == 16) tmem_ld16f(at, x);
      else tmem_ld32f(at, x);
    };
    PagedWalk u = make_walk();
    int J0 = 0;   // tiles of the units before this one
    for (int ui = 0; u.next(); ++ui, J0 += u.n) {
      const int first = u.len - u.fresh + u.qt * p.per_tile, last = first + min(p.per_tile, u.fresh - u.qt * p.per_tile) - 1;   // positions
      // keys that every row of the unit sees
      const int all_end = p.causal ? min(u.end, first + 1) : u.end, all_begin = p.window > 0 ? max(0, last - p.window + 1) : 0;
      float *s_ref = s_refs + ((ui & 1) * 2 + group) * R, *s_sum = s_sums + ((ui & 1) * 2 + group) * R;
      const uint32_t tOg = tO + ((ui & 1) * 2 + group) * R;
      if (key0 < R) s_ref[key0] = -1.0e30f;   // stands for -inf
      sync();
      float acc[R];
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r] = 0.0f;
      const int n = u.n, kv_first = (u.lo + u.t0) * N, end = u.end;
      if constexpr (k8Bit) asm volatile("" ::"l"(&u) : "memory");   // the walk waits in memory
#pragma unroll 1
      for (int i = (J0 ^ group) & 1; i < n; i += 2) {
        const int J = J0 + i, sb = J % L::kScores;
        paged_wait(bars + L::kSFull + sb, (J / L::kScores) & 1, ab, kPgSFull);
        tc_fence_after_sync();
        float s[R];
        load_rows(tS + sb * R, s);
        tmem_wait_ld();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + L::kSFree + sb);
        if constexpr (k8Bit) {
          const int slot = J % L::kScales;
          mbar_wait_rows(bars + L::kScFull + slot, (J / L::kScales) & 1, ab, kPgScales);
          const float f = key_factor(smem[L::kOffScales + slot * 2 * N + key0]) * c2;
          const float4* qs = reinterpret_cast<const float4*>(smem + L::kOffQs) + (ui & 3) * (R / 4);
#pragma unroll
          for (int r = 0; r < R; r += 4) {
            if (r >= p.rows) break;
            const float4 q = qs[r / 4];
            s[r] *= f * q.x;
            s[r + 1] *= f * q.y;
            s[r + 2] *= f * q.z;
            s[r + 3] *= f * q.w;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bars + L::kScEmpty + slot);
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (r % 4 == 0 && r >= p.rows) break;
            s[r] *= c2;
          }
        }
        const int kv0 = kv_first + i * N, key = kv0 + key0;
        if (kv0 < all_begin || kv0 + N > all_end) {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (r % 4 == 0 && r >= p.rows) break;
            const int pos = first + s_pos[r];
            const bool in = key < end && (!p.causal || key <= pos) && (p.window == 0 || key > pos - p.window);
            s[r] = in ? s[r] : -INFINITY;
          }
        }
        // 16 rows in 8 bits hold their reference maxima and rescales (173 us for 182, 16 sequences of up to 32768); else they are read
        // again where they are used: 32 rows in 8 bits spilled more with them (298 us for 218, 16 sequences of 16384, 32 rows; 208 bytes
        // a thread are left)
        constexpr bool kHold = k8Bit && R == 16;
        float ref[kHold ? R : 1], over = -INFINITY;
        auto hold = [&](int r, const float4& m) {
          if constexpr (kHold) {
            ref[r] = m.x;
            ref[r + 1] = m.y;
            ref[r + 2] = m.z;
            ref[r + 3] = m.w;
          }
        };
#pragma unroll
        for (int r = 0; r < R; r += 4) {
          if (r >= p.rows) break;
          const float4 m = reinterpret_cast<const float4*>(s_ref)[r / 4];
          hold(r, m);
          over = max3(over, s[r] - m.x, s[r + 1] - m.y);
          over = max3(over, s[r + 2] - m.z, s[r + 3] - m.w);
        }
        if (named_sync_or(1 + group, 128, over > 8.0f)) {
          // some row has grown: its maximum of this tile is the new reference
          float mine = 0.0f;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            if (r % 4 == 0 && r >= p.rows) break;
            const float m = warp_max(s[r]);
            if (lane == r) mine = m;
          }
          if (lane < R) s_warp[(warp & 3) * R + lane] = mine;
          sync();
          if (key0 < R) {
            const float m = fmaxf(fmaxf(s_warp[key0], s_warp[R + key0]), fmaxf(s_warp[2 * R + key0], s_warp[3 * R + key0])), old = s_ref[key0];
            const bool grown = m - old > 8.0f;
            s_rescale[key0] = grown ? fast_exp2(old - m) : 1.0f;
            if (grown) s_ref[key0] = m;
          }
          sync();
          float scale[kHold ? R : 1];
#pragma unroll
          for (int r = 0; r < R; r += 4) {
            if (r >= p.rows) break;
            const float4 x = reinterpret_cast<const float4*>(s_rescale)[r / 4];
            if constexpr (kHold) {
              hold(r, reinterpret_cast<const float4*>(s_ref)[r / 4]);
              scale[r] = x.x; scale[r + 1] = x.y; scale[r + 2] = x.z; scale[r + 3] = x.w;
            } else {
              acc[r] *= x.x;
              acc[r + 1] *= x.y;
              acc[r + 2] *= x.z;
              acc[r + 3] *= x.w;
            }
          }
          if constexpr (kHold) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
              if (r % 4 == 0 && r >= p.rows) break;
              acc[r] *= scale[r];
            }
          }
          if (i >= 2) {   // behind the group's last P.V
            mbar_wait_rows(bars + L::kODone + group, ((J >> 1) - 1) & 1, ab, kPgODone);
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < R; c += 16) {
              float o[16];
              tmem_ld16f(tOg + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int r = 0; r < 16; ++r) o[r] *= kHold ? scale[kHold ? c + r : 0] : s_rescale[c + r];
              tmem_st16f(tOg + c, o);
            }
            tmem_wait_st();
          }
        }
        // the operand's buffer is free behind the group's last P.V
        if (J >= 2) mbar_wait_rows(bars + L::kODone + group, ((J >> 1) - 1) & 1, ab, kPgODone);
        float4 m;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r % 4 == 0) {   // four rows at a time, those that there are
            if (r >= p.rows) break;
            if (!kHold) m = reinterpret_cast<const float4*>(s_ref)[r / 4];
          }
          const float x = fast_exp2(s[r] - (kHold ? ref[kHold ? r : 0] : r % 4 == 0 ? m.x : r % 4 == 1 ? m.y : r % 4 == 2 ? m.z : m.w));
          acc[r] += x;
          const uint32_t two = pack2<kBf16>(x, 0.0f);
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(line + r * 128 + ((p_piece ^ (r & 7)) << 4)), "h"(static_cast<uint16_t>(two)) : "memory");
        }
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars + L::kPReady + group);
      }
      // ---- end of the unit: sums over the keys, a row to every lane by halves ----
      sum_rows<R, 16>(acc, lane);
      const int my_row = lane * R / 32;   // R = 16: two lanes a row
      s_warp[(warp & 3) * R + my_row] = acc[0];
      sync();
      if (key0 < R) s_sum[key0] = (s_warp[key0] + s_warp[R + key0]) + (s_warp[2 * R + key0] + s_warp[3 * R + key0]);
      const int Jl = J0 + u.n - 1, mine = (Jl & 1) == group ? Jl : Jl - 1;   // the group's last tile
      if (mine >= J0) paged_wait(bars + L::kODone + group, (mine >> 1) & 1, ab, kPgODone);
      if (named_sync_or(3, 256, *abort_flag != 0)) break;   // both groups; all warps together
      tc_fence_after_sync();
      const bool has0 = ((Jl & 1) == 0 ? Jl : Jl - 1) >= J0, has1 = ((Jl & 1) == 1 ? Jl : Jl - 1) >= J0;
      const bool whole = u.n == u.total;
      // a partial result: the unit's first share leaves it in the second slot of its CTA, the later ones in the first
      const long long slot = (2LL * cta + (u.t0 == 0 ? 1 : 0)) * p.rows;
      const int row0 = p.cu != nullptr ? tab.row[u.b] : 0;
      const float *ref0 = s_refs + (ui & 1) * 2 * R, *sum0 = s_sums + (ui & 1) * 2 * R;   // group 1's R further
      const uint32_t tO0 = tO + (ui & 1) * 2 * R;
      const int column = k8Bit ? paged_column(key0) : key0;
      uint16_t* o = static_cast<uint16_t*>(p.o) + (p.cu != nullptr ? 0 : u.b * p.o_sb) + column;
#pragma unroll 1
      for (int c = group * 8; c < p.rows; c += 16) {
        float x[8], y[8];
        tmem_ld8f(tO0 + c, x);
        tmem_ld8f(tO0 + R + c, y);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = c + k, tok = u.qt * p.per_tile + s_pos[min(r, R - 1)];
          if (r >= p.rows || tok >= u.fresh || key0 >= D) continue;
          const float m = fmaxf(ref0[r], ref0[R + r]), w0 = fast_exp2(ref0[r] - m), w1 = fast_exp2(ref0[R + r] - m);
          const float sum = sum0[r] * w0 + sum0[R + r] * w1, inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // no key: 0, and -inf
          // an accumulator that the unit has not used holds anything
          const float v = ((has0 ? x[k] * w0 : 0.0f) + (has1 ? y[k] * w1 : 0.0f)) * inv;
          const int head = head_of(u, r);
          if (whole) {
            const uint32_t two = pack2<kBf16>(v, 0.0f);
            o[(row0 + tok) * p.o_ss + head * p.o_sh] = static_cast<uint16_t>(two);
          } else {
            p.part_o[slot * D + ((column >> 2) * p.rows + r) * 4 + (column & 3)] = v;
          }
        }
      }
      if (tid < p.rows) {
        const int tok = u.qt * p.per_tile + s_pos[tid];
        if (tok < u.fresh) {
          const float m = fmaxf(ref0[tid], ref0[R + tid]);
          const float sum = sum0[tid] * fast_exp2(ref0[tid] - m) + sum0[R + tid] * fast_exp2(ref0[R + tid] - m);
          const float lse = sum == 0.0f ? -INFINITY : logf(sum) + m * 0.6931471805599453f;
          const int head = head_of(u, tid);
          if (!whole) p.part_lse[slot + tid] = lse;
          else if (p.lse != nullptr) p.lse[(p.cu != nullptr ? static_cast<long long>(head) : static_cast<long long>(u.b) * p.heads + head) * p.seq + row0 + tok] = lse;
        }
      }
      if (tid == 0 && !whole && u.t0 == 0) {
        p.cut[cta] = make_int4(u.b, u.h, u.qt, pg_owner(u.last, share.shares, share.total));
        p.cut_rows[cta] = make_int2(p.cu != nullptr ? tab.row[u.b] : 0, u.fresh);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + L::kOFree + (ui & 1));
    }
  } else if constexpr (k8Bit) {
    if (warp == 12) {
      paged_scales<L::kScales>(p, make_walk(), smem + L::kOffScales, bars + L::kScFull, bars + L::kScEmpty, ab);
    } else {
      // ======================= queries in parts, a unit ahead, and V in 16 bits =======================
      const int ct = tid - 416;
      PagedWalk u = make_walk(), ahead = make_walk();
      auto split = [&](int ui) -> bool {
        const int qb = ui & 1;
        if (ui >= 2 && !warp_all(paged_wait(bars + L::kQEmpty + qb, ((ui >> 1) - 1) & 1, ab, kPgQEmpty))) return false;
        paged_split_queries<D, kBf16, L::kPieces, L::kConvWarps>(p, ahead, tab.row[ahead.b], ct, sQ + qb * L::kQBytes, R * D, reinterpret_cast<float*>(smem + L::kOffQs) + (ui & 3) * R);
        if (lane == 0) mbar_arrive(bars + L::kQFull + qb);
        return true;
      };
      ahead.next();
      bool ok = split(0);
      int J = 0;
      for (int ui = 0; ok && u.next(); ++ui) {
        if (ahead.next()) ok = split(ui + 1);
        for (int i = 0; i < u.n && ok; ++i, ++J) {
          const int sc = J % L::kScales, raw = J % L::kRaw, st = J % L::kStagesV;
          ok = warp_all(paged_wait(bars + L::kScFull + sc, (J / L::kScales) & 1, ab, kPgScales));
          ok = ok && warp_all(paged_wait(bars + L::kRawFull + raw, (J / L::kRaw) & 1, ab, kPgRawFull));
          ok = ok && warp_all(paged_wait(bars + L::kVEmpty + st, ((J / L::kStagesV) & 1) ^ 1, ab, kPgVEmpty));
          if (!ok) break;
          paged_widen<D, kBf16, L::kConvWarps>(smem + L::kOffRaw + raw * L::kRawBytes, smem + L::kOffScales + (sc * 2 + 1) * N, sV + st * L::kTileBytes, ct);
          if (lane == 0) {
            mbar_arrive(bars + L::kVFull + st);
            mbar_arrive(bars + L::kRawEmpty + raw);
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
  if (warp == 11) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

template <int D, int R, bool kBf16, bool k8Bit>
int launch_tokens(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status) {
  using L = TokensSmem<D, R, kBf16, k8Bit>;
  PagedParams p;
  PagedMaps maps;
  const int rc = paged_setup(a, d, status, &p, &maps);
  if (rc != ATTN_B200_OK) return rc;
  auto kernel = paged_tokens_kernel<D, R, kBf16, k8Bit>;
  static std::atomic<uint64_t> asked{0};
  if (!paged_allow(kernel, L::kBytes, asked)) return ATTN_B200_E_LAUNCH;
  return launch_pdl(kernel, dim3(d.ctas), dim3(L::kThreads), L::kBytes, stream, maps, p) ? paged_merge(a, d, p, stream) : ATTN_B200_E_LAUNCH;
}

template <int D, int R>
int tokens_of(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status) {
  const bool bf16 = a->dtype == ATTN_B200_DTYPE_BF16;
  if (a->cache.dtype == ATTN_B200_DTYPE_E4M3) return bf16 ? launch_tokens<D, R, true, true>(a, d, stream, status) : launch_tokens<D, R, false, true>(a, d, stream, status);
  return bf16 ? launch_tokens<D, R, true, false>(a, d, stream, status) : launch_tokens<D, R, false, false>(a, d, stream, status);
}

int launch_paged_tokens(const AttnB200PagedAttnArgs* a, const PagedPlan& d, cudaStream_t stream, int* status) {
  if (a->cache.head_dim == 64) return d.rows <= 16 ? tokens_of<64, 16>(a, d, stream, status) : tokens_of<64, 32>(a, d, stream, status);
  return d.rows <= 16 ? tokens_of<128, 16>(a, d, stream, status) : tokens_of<128, 32>(a, d, stream, status);
}

}  // namespace b200
