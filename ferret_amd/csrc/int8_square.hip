// int8 product of many tokens (math and contract: int8_gemm.hip): tiles of BN weight rows
// by BM tokens, both operands copied straight into LDS and multiplied by
// v_mfma_i32_32x32x32_i8.
//
// Work-group: WR x WT waves, a wave takes BN / WR weight rows by BM / WT tokens as NI x
// MI blocks of 32 x 32 (weight rows are the A side, so a lane holds four outputs in a
// row of one token).  Stages of KS bytes of every row go through two rings, NW slots of
// weight rows and NT of tokens, by asynchronous loads of a base in scalar registers and
// one offset per lane, fixed for the whole product.
//
// Schedule.  A substep is 32 bytes of K, NI * MI MFMAs; the fragments of the next one are
// read among the first of them, into the other of two register sets.  With the last
// substep of stage s in registers the wave waits for its own loads of stage s + 1 and
// meets the others, once per stage: the slots just read are refilled, one load every few
// MFMAs until the next barrier (all at once, they hold up the waves that issue them: 117.6
// us at M = N = 4096, K = 7168 where this takes 98), and the next stage's first fragments
// are read.
//
// What bounds it: power.  M = N = 4096, K = 7168, 256 x 256 tiles, one per CU: 98 us, 2.45
// POP/s, with random codes; 71 us with zeros, at a clock of 2.4 GHz where the matrix
// units alone take 48, the launch, the first loads and the last stores about 10; without the loads
// 88 and 64, without loads and fragment reads 83 and 64.
#include "attention.hpp"
#include "int8_epilogue.hpp"

namespace ferret {
namespace i8 {
namespace {

typedef int i32x16 __attribute__((ext_vector_type(16)));

// D(32x32 i32) += A(32x32 i8) B(32x32 i8).  Lane l: A row / B column l % 32, bytes 16 (l /
// 32) .. +16 of the 32; D column l % 32, rows 8 (i / 4) + 4 (l / 32) + i % 4 for element i.
__device__ __forceinline__ i32x16 mfma32(u32x4 a, u32x4 b, i32x16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

template <int BN, int BM, int KS, int NW, int NT, int WR, int WT>
struct Sq {
  static constexpr int kWaves = WR * WT, kThreads = 64 * kWaves;
  static constexpr int kNI = BN / WR / 32, kMI = BM / WT / 32, kU = KS / 32, kMF = kNI * kMI;
  static constexpr int kW = BN * KS, kT = BM * KS;                             // bytes of a stage
  static constexpr int kLW = kW / 1024 / kWaves, kLT = kT / 1024 / kWaves;     // 1-KB loads of a wave per stage
  static constexpr int kLoads = kLW + kLT;
  static constexpr int kAway = (NW > NT ? kLW : 0) + (NT - 2) * kLoads;        // in flight at a barrier
  static constexpr int kRing = NW * kW + NT * kT;
  static constexpr int kPitch = BN / WR * 2 + 16;                              // bytes of a token row of the epilogue
  static constexpr int kEpi = kWaves * (BM / WT) * kPitch;
  static constexpr int kLds = kRing > kEpi ? kRing : kEpi;
  static_assert(kW % (1024 * kWaves) == 0 && kT % (1024 * kWaves) == 0 && kLds <= 160 * 1024, "LDS budget");
  static_assert(NT >= 2 && (NW == NT || NW == NT + 1) && kAway + kLoads < 63, "rings");
  static_assert(BN % (32 * WR) == 0 && BM % (32 * WT) == 0 && kU % 2 == 0, "tile");
  // The MFMA of the period from barrier to barrier that load j is issued behind.
  static constexpr int slot(int j) { return j * (kU * kMF) / kLoads; }
};

// Slot of 16-byte chunk c of a stage row: the lanes that LDS serves together (rows 0 - 3, 12
// - 15 and 20 - 27 of 32, or the others) fall on distinct banks.
template <int KS>
__device__ __forceinline__ int sq_swz(int row, int c) {
  static_assert(KS == 128 || KS == 256, "bytes of a stage row");
  return KS == 256 ? c ^ (row & 15) : c ^ ((row >> 1) & 7);
}

template <int BN, int BM, int KS, int NW, int NT, int WR, int WT>
__global__ __launch_bounds__(64 * WR * WT, WR * WT == 8 ? 2 : 1) void int8_square_kernel(Args p) {
  using S = Sq<BN, BM, KS, NW, NT, WR, WT>;
  constexpr int NI = S::kNI, MI = S::kMI, U = S::kU, MF = S::kMF;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int c32 = lane & 31, h = lane >> 5;
  const int wr = wave % WR, wt = wave / WR;

  // Work-groups are dealt to the 8 XCDs in turn: each takes a contiguous range of tiles, in
  // groups of 4 token tiles, so that its 32 CUs share panels through their L2.
  const int split = blockIdx.x % p.splits;
  int tile = blockIdx.x / p.splits;
  const int tiles = gridDim.x / p.splits, row_tiles = tiles / p.tok_tiles;
  if (p.splits == 1 && tiles % 8 == 0) tile = (tile & 7) * (tiles >> 3) + (tile >> 3);
  constexpr int GM = 4;
  const int first = tile / (GM * row_tiles) * GM, in_group = tile % (GM * row_tiles);
  const int size = min(p.tok_tiles - first, GM);
  const int tok0 = (first + in_group % size) * BM, row0 = in_group / size * BN;

  const int K = p.K, nks = (K + KS - 1) / KS;
  const int k0 = (int)((long long)split * nks / p.splits), k1 = (int)((long long)(split + 1) * nks / p.splits);

  // ---- loads: load j of a stage, tokens first, is 1 KB of rows; a wave has kLT + kLW of them
  const uint8_t* const base_w = p.b + (size_t)row0 * K;
  const uint8_t* const base_t = p.a + (size_t)tok0 * K;
  int off[S::kLoads];
  constexpr int LR = KS / 16, IR = 1024 / KS;  // lanes of a row, rows of a load
  const auto row_of = [&](int j) { return (j < S::kLT ? wave * S::kLT + j : wave * S::kLW + j - S::kLT) * IR + lane / LR; };
#pragma unroll
  for (int j = 0; j < S::kLoads; ++j) {
    const int lr = row_of(j), row = min(lr, j < S::kLT ? p.M - 1 - tok0 : p.N - 1 - row0);
    off[j] = row * K + sq_swz<KS>(lr & 31, lane % LR) * 16;
  }
  // Load j of its operand's stage s; WHOLE: K does not end inside it.
  const auto load = [&](auto wholec, auto jc, int s) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(wholec)::value;
    constexpr int j = decltype(jc)::value;
    constexpr bool T = j < S::kLT;
    int o = off[j];
    if constexpr (!WHOLE) {
      if (s >= k1) return;
      if ((s + 1) * KS > K)  // chunks past K: the row's last one again
        o -= max(sq_swz<KS>(row_of(j) & 31, lane % LR) * 16 + 16 - (K - s * KS), 0);
    }
    const int at = T ? NW * S::kW + (s - k0) % NT * S::kT + (wave * S::kLT + j) * 1024
                     : (s - k0) % NW * S::kW + (wave * S::kLW + j - S::kLT) * 1024;
    dma_16((T ? base_t : base_w) + (size_t)s * KS, o, uniform(lds_address(lds) + at));
  };
  // The loads that go out behind MFMA `m` of the period that starts with stage s's barrier.
  const auto loads_at = [&](auto wholec, auto mc, int s) __attribute__((always_inline)) {
    constexpr int m = decltype(mc)::value;
    static_for<0, S::kLoads>([&](auto j) {
      if constexpr (S::slot(decltype(j)::value) == m) load(wholec, j, s + (decltype(j)::value < S::kLT ? NT : NW));
    });
  };

  // ---- fragments, in the order of their use
  u32x4 wf[2][NI], tf[2][MI];
  const auto read = [&](int s, int u, int set, auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value, both = 2 * (NI < MI ? NI : MI);
    constexpr bool T = i < both ? i % 2 == 0 : MI > NI;
    constexpr int n = i < both ? i / 2 : i - both / 2;
    const uint8_t* st = T ? lds + NW * S::kW + (s - k0) % NT * S::kT + (wt * MI + n) * 32 * KS
                          : lds + (s - k0) % NW * S::kW + (wr * NI + n) * 32 * KS;
    const u32x4 v = ld_u32x4(st + c32 * KS + (sq_swz<KS>(c32, 2 * u + h) << 4));
    if constexpr (T) tf[set][n] = v;
    else wf[set][n] = v;
  };

  i32x16 acc[NI][MI];
#pragma unroll
  for (int ni = 0; ni < NI; ++ni)
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) acc[ni][mi] = i32x16{};

  // Stage s.  NEXT: there is a stage s + 1; WHOLE: every load that goes out is of a whole
  // stage before the last one.
  const auto stage = [&](auto nextc, auto wholec, int s) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(nextc)::value, WHOLE = decltype(wholec)::value;
    static_for<0, U>([&](auto uc) {
      constexpr int u = decltype(uc)::value, set = u & 1, other = set ^ 1;
      constexpr bool last = u == U - 1;
      if constexpr (!NEXT) {
        if ((2 * u + h) * 16 >= K - s * KS)
#pragma unroll
          for (int mi = 0; mi < MI; ++mi) tf[set][mi] = u32x4{0u, 0u, 0u, 0u};
      }
      static_for<0, MF>([&](auto tc) {
        constexpr int t = decltype(tc)::value, ni = t / MI, mi = t % MI;
        acc[ni][mi] = mfma32(wf[set][ni], tf[set][mi], acc[ni][mi]);
        if constexpr (last && NEXT && t == 0) {
          // The slots have been read; stage s + 1 has landed.
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (WHOLE || s - 1 + NW < k1) wait_vmcnt<S::kAway>();
          else wait_vmcnt<0>();
          __builtin_amdgcn_sched_barrier(0);
          __builtin_amdgcn_s_barrier();
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!last || NEXT)
          static_for<2 * t, 2 * t + 2 + (t == MF - 1 ? NI + MI : 0)>([&](auto i) {
            if constexpr (decltype(i)::value < NI + MI) read(last ? s + 1 : s, last ? 0 : u + 1, other, i);
          });
        if constexpr (NEXT) {
          if constexpr (last) loads_at(wholec, tc, s);
          else loads_at(wholec, IntC<(u + 1) * MF + t>{}, s - 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  };

  // The first stages' loads in the order in which they are waited for, and those of the
  // period before stage k0's barrier that its MFMAs do not issue.
#pragma unroll
  for (int s = 0; s < NW - 1; ++s)
    static_for<0, S::kLoads>([&](auto j) {
      if (decltype(j)::value >= S::kLT || s < NT - 1) load(IntC<false>{}, j, k0 + s);
    });
  static_for<0, MF>([&](auto m) { loads_at(IntC<false>{}, m, k0 - 1); });
  wait_vmcnt<0>();
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  static_for<0, NI + MI>([&](auto i) { read(k0, 0, 0, i); });
  int s = k0;
  for (; s + NW < k1 - 1; ++s) stage(IntC<true>{}, IntC<true>{}, s);
  for (; s + 1 < k1; ++s) stage(IntC<true>{}, IntC<false>{}, s);
  stage(IntC<false>{}, IntC<false>{}, k1 - 1);

  // ---- epilogue
  const int wrow0 = row0 + wr * NI * 32, wtok0 = tok0 + wt * MI * 32;
  if (p.splits > 1) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const int m = wtok0 + 32 * mi + c32, n = wrow0 + 32 * ni + 8 * g4 + 4 * h;
          const i32x16& a = acc[ni][mi];
          if (m < p.M && n < p.N)
            *reinterpret_cast<i32x4*>(p.partial + ((size_t)split * p.M + m) * p.N + n) =
                i32x4{a[4 * g4], a[4 * g4 + 1], a[4 * g4 + 2], a[4 * g4 + 3]};
        }
    return;
  }
  // Through LDS, so that a store writes whole runs of a token's row.
  __syncthreads();
  uint8_t* const stg = lds + wave * (MI * 32) * S::kPitch;
#pragma unroll
  for (int mi = 0; mi < MI; ++mi) {
    const int m = min(wtok0 + 32 * mi + c32, p.M - 1);
    const float sa = p.sa[m];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
        const int at = 32 * ni + 8 * g4 + 4 * h, n = min(wrow0 + at, p.N - 4);
        const i32x16& a = acc[ni][mi];
        *reinterpret_cast<u32x2*>(stg + (32 * mi + c32) * S::kPitch + at * 2) =
            four_outputs(p, m, n, sa, i32x4{a[4 * g4], a[4 * g4 + 1], a[4 * g4 + 2], a[4 * g4 + 3]});
      }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own rows are written
  constexpr int RC = NI * 4;  // 16-byte chunks of a wave's token row
#pragma unroll
  for (int i = 0; i < MI * 32 * RC / 64; ++i) {
    const int r = (i * 64 + lane) / RC, c = (i * 64 + lane) % RC;
    const int m = wtok0 + r, n = wrow0 + c * 8;
    if (m < p.M && n < p.N)
      *reinterpret_cast<u32x4*>(p.out + (size_t)m * p.N + n) = *reinterpret_cast<const u32x4*>(stg + r * S::kPitch + c * 16);
  }
}

template <int BN, int BM, int KS, int NW, int NT, int WR, int WT>
int launch_square(const Args& p, hipStream_t st) {
  using S = Sq<BN, BM, KS, NW, NT, WR, WT>;
  FERRET_HIP_CHECK((set_lds_limit_once<int8_square_kernel<BN, BM, KS, NW, NT, WR, WT>>(S::kLds)));
  hipLaunchKernelGGL((int8_square_kernel<BN, BM, KS, NW, NT, WR, WT>),
                     dim3((unsigned)(cdiv(p.N, BN) * p.tok_tiles * p.splits)), dim3(S::kThreads), S::kLds, st, p);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace i8
}  // namespace ferret

// The kernels of kTiles from kFirstSquare on.
int ferret_int8_square(int tile, const ferret::i8::Args& p, hipStream_t st) {
  using namespace ferret::i8;
  switch (tile) {
    case 5: return launch_square<64, 32, 256, 3, 3, 2, 1>(p, st);
    case 6: return launch_square<64, 64, 128, 4, 4, 2, 2>(p, st);
    case 7: return launch_square<64, 128, 128, 3, 3, 2, 2>(p, st);
    case 8: return launch_square<128, 128, 128, 4, 4, 2, 4>(p, st);
    case 9: return launch_square<128, 128, 128, 3, 2, 2, 2>(p, st);
    case 10: return launch_square<256, 128, 128, 3, 3, 4, 2>(p, st);
    case 11: return launch_square<256, 256, 128, 3, 2, 2, 4>(p, st);
  }
  return FERRET_ERR_SHAPE;
}
