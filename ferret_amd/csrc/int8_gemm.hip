// int8 product with a scale per token and per output channel for gfx950:
//   y[m, n] = bf16_RNE(float(sum_k a[m,k] b[n,k]) * sa[m] * sb[n] (+ residual[m, n]))
// The sum is whole and exact in 32 bits (K <= 65536), so the result depends on
// neither tile, split nor order: bit for bit the same from every variant.
//
// Here: the kernel for few tokens, the sum over K splits, and the entry points;
// int8_square.hip: the kernel for more.  int8_plan.hpp chooses.
//
// Few tokens: the bytes of the weights bound it.  A work-group of four or eight waves takes
// RT x 16 weight rows by all TT x 16 tokens over one K split; both operands go global ->
// LDS in stages of KS bytes of each row through a ring of NS stages, one barrier per
// stage.  The waves split the K of a stage as well as the tile (WK); the parts meet in
// LDS once.  Rows past N or M repeat the last one (never stored), 16-byte chunks past K the
// last one of their row, with the tokens' as zeros.  v_mfma_i32_16x16x64_i8: weight rows
// are the A side, tokens the B side, so a lane holds four outputs in a row of one token.
// Tiles of 16 rows and 512 bytes let 4096 rows fill the CUs in one launch: 4096 x 12288 at
// 16 tokens 11.3 to 11.7 us, 12.6 in tiles of 32 rows and 13.0 of 64, with splits of K (two launches);
// 4096 x 4096 at 1 6.2, 7.5 and 8.7.  24576 x 4096 at 1 token, 96 rows, 17.0 to 17.6 us, 5.7 TB/s or more.
//
// Every work-group starts at another K step (row tile index modulo its steps) and wraps
// around: in lockstep, all of them read the same columns of rows a power of two
// apart, which sit on few of the memory channels.
#include "int8_epilogue.hpp"
#include "ranges.hpp"

namespace ferret {
namespace i8 {
namespace {

// D(16x16 i32) += A(16x64 i8) B(64x16 i8). Lane l: A row / B column l % 16, bytes 16 (l /
// 16) .. +16 of the 64; D rows 4 (l / 16) + i, column l % 16.
__device__ __forceinline__ i32x4 mfma_i8(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// Waves: WR along the rows, WT along the tokens, WK along the K of a stage.
template <int RT, int TT, int KS, int NS, int WR, int WT, int WK>
struct Cfg {
  static constexpr int kRows = 16 * RT, kToks = 16 * TT;
  static constexpr int kStage = (RT + TT) * 16 * KS;
  static constexpr int kInstr = kStage / 1024;                 // 1-KB loads of a stage: weights, then tokens
  static constexpr int kWInstr = RT * 16 * KS / 1024;
  static constexpr int kIRows = 1024 / KS;                     // rows of a load
  static constexpr int kWaves = WR * WT * WK, kThreads = 64 * kWaves;
  static constexpr int kLd = (kInstr + kWaves - 1) / kWaves;   // loads per wave (past kInstr: the last one again)
  static constexpr int kRB = RT / WR, kTB = TT / WT, kKB = KS / 64 / WK;  // row and token blocks, MFMAs deep, per wave
  static constexpr int kPitch = kRows + 4;                     // words of a token row of the epilogue
  static constexpr int kRing = NS * kStage;
  static constexpr int kEpi = WK * kToks * kPitch * 4;
  static constexpr int kLds = kRing > kEpi ? kRing : kEpi;
  static constexpr int kQuads = kRows / 4;                     // groups of four outputs of a token
  static_assert(kThreads <= 1024 && RT % WR == 0 && TT % WT == 0 && (KS / 64) % WK == 0, "waves");
  static_assert(KS >= 256 && kStage % 1024 == 0 && kLds <= 160 * 1024, "LDS budget");  // 16 chunks to a row: swz
  static_assert(NS >= 2 && (NS - 2) * kLd < 63, "vmcnt range");
};

// Slot of 16-byte chunk c of stage row `row`: the lanes of a fragment that LDS serves
// together (rows 0 - 3 and 12 - 15 of one chunk with 4 - 11 of the next) fall on distinct
// banks.
__device__ __forceinline__ int swz(int row, int c) { return c ^ row; }

// Wait until at most min(n, N) stages of L loads are in flight.
template <int L, int N>
__device__ __forceinline__ void wait_younger(int n) {
  if constexpr (N == 0) {
    wait_vmcnt<0>();
  } else {
    if (n >= N) wait_vmcnt<N * L>();
    else wait_younger<L, N - 1>(n);
  }
}

__device__ __forceinline__ void put_four(const Args& p, int m, int n, i32x4 sum) {
  *reinterpret_cast<u32x2*>(p.out + (size_t)m * p.N + n) = four_outputs(p, m, n, p.sa[m], sum);
}

template <int RT, int TT, int KS, int NS, int WR, int WT, int WK>
__global__ __launch_bounds__(64 * WR * WT * WK) void int8_tiled_kernel(Args p) {
  using C = Cfg<RT, TT, KS, NS, WR, WT, WK>;
  extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int wr = wave % WR, wt = (wave / WR) % WT, wk = wave / (WR * WT);

  const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
  const int tt = tile % p.tok_tiles, rt = tile / p.tok_tiles;
  const int row0 = rt * C::kRows, tok0 = tt * C::kToks;
  const int nks = (p.K + KS - 1) / KS, chunks = p.K / 16;
  const int k0 = (int)((long long)split * nks / p.splits), k1 = (int)((long long)(split + 1) * nks / p.splits);
  const int nsteps = k1 - k0, rot = nsteps > 0 ? rt % nsteps : 0;

  const uint8_t* src[C::kLd];  // the row
  int chunk[C::kLd];           // its 16-byte chunk of a stage
#pragma unroll
  for (int i = 0; i < C::kLd; ++i) {
    const int j = min(wave * C::kLd + i, C::kInstr - 1);
    constexpr int LR = 64 / C::kIRows;         // lanes of a row
    const int lr = C::kIRows * j + lane / LR;  // stage row
    chunk[i] = swz(lr & 15, lane % LR);
    const size_t row = j < C::kWInstr ? min(row0 + lr, p.N - 1) : min(tok0 + lr - C::kRows, p.M - 1);
    src[i] = (j < C::kWInstr ? p.b : p.a) + row * p.K;
  }
  const auto step_at = [&](int step) { return k0 + (step + rot < nsteps ? step + rot : step + rot - nsteps); };
  const auto issue = [&](int step) __attribute__((always_inline)) {
    uint8_t* st = lds + (step % NS) * C::kStage;
    const int c0 = step_at(step) * (KS / 16);
#pragma unroll
    for (int i = 0; i < C::kLd; ++i) {
      const int j = min(wave * C::kLd + i, C::kInstr - 1);
      const uint8_t* from = src[i] + (size_t)min(c0 + chunk[i], chunks - 1) * 16;
      if (p.nt && j < C::kWInstr) g2l_16_nt(from, st + j * 1024);
      else g2l_16(from, st + j * 1024);
    }
  };

  i32x4 acc[C::kRB][C::kTB];
#pragma unroll
  for (int x = 0; x < C::kRB; ++x)
#pragma unroll
    for (int y = 0; y < C::kTB; ++y) acc[x][y] = i32x4{0, 0, 0, 0};

#pragma unroll
  for (int s = 0; s < NS - 1; ++s)
    if (s < nsteps) issue(s);
  for (int step = 0; step < nsteps; ++step) {
    // This stage has landed for every wave, and the slot of the stage before
    // (the one refilled below) has been read by every wave.
    wait_younger<C::kLd, NS - 2>(nsteps - 1 - step);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (step + NS - 1 < nsteps) issue(step + NS - 1);
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t* st = lds + (step % NS) * C::kStage;
    const int left = chunks - step_at(step) * (KS / 16);  // chunks of the stage below K
#pragma unroll
    for (int k = 0; k < C::kKB; ++k) {
      const int ch = 4 * (wk * C::kKB + k) + g, c = swz(r, ch) << 4;
      u32x4 wf[C::kRB], xf[C::kTB];
#pragma unroll
      for (int x = 0; x < C::kRB; ++x)
        wf[x] = *reinterpret_cast<const u32x4*>(st + ((wr * C::kRB + x) * 16 + r) * KS + c);
#pragma unroll
      for (int y = 0; y < C::kTB; ++y) {
        xf[y] = *reinterpret_cast<const u32x4*>(st + (C::kRows + (wt * C::kTB + y) * 16 + r) * KS + c);
        if (ch >= left) xf[y] = u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int x = 0; x < C::kRB; ++x)
#pragma unroll
        for (int y = 0; y < C::kTB; ++y) acc[x][y] = mfma_i8(wf[x], xf[y], acc[x][y]);
    }
  }

  // Epilogue through the idle ring: [K part][token][row], then four outputs of a token
  // per thread.
  __builtin_amdgcn_sched_barrier(0);
  __syncthreads();
  int32_t* red = reinterpret_cast<int32_t*>(lds);
#pragma unroll
  for (int x = 0; x < C::kRB; ++x)
#pragma unroll
    for (int y = 0; y < C::kTB; ++y)
      *reinterpret_cast<i32x4*>(red + (wk * C::kToks + (wt * C::kTB + y) * 16 + r) * C::kPitch +
                                (wr * C::kRB + x) * 16 + 4 * g) = acc[x][y];
  __syncthreads();
  for (int i = threadIdx.x; i < C::kToks * C::kQuads; i += C::kThreads) {
    const int t = i / C::kQuads, q = i % C::kQuads, n = row0 + 4 * q;
    if (tok0 + t >= p.M || n >= p.N) continue;
    const int32_t* part = red + t * C::kPitch + 4 * q;
    i32x4 v = *reinterpret_cast<const i32x4*>(part);
#pragma unroll
    for (int k = 1; k < WK; ++k) v += *reinterpret_cast<const i32x4*>(part + k * C::kToks * C::kPitch);
    if (p.splits > 1) *reinterpret_cast<i32x4*>(p.partial + ((size_t)split * p.M + tok0 + t) * p.N + n) = v;
    else put_four(p, tok0 + t, n, v);
  }
}

// The sum over S K splits, four outputs per thread, all loads before the first sum.
template <int S>
__global__ __launch_bounds__(256) void int8_reduce_kernel(Args p) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x, quads = p.N / 4;
  if (i >= p.M * quads) return;
  const int m = (int)(i / quads), n = (int)(i % quads) * 4;
  i32x4 v[S];
#pragma unroll
  for (int s = 0; s < S; ++s) v[s] = *reinterpret_cast<const i32x4*>(p.partial + ((size_t)s * p.M + m) * p.N + n);
#pragma unroll
  for (int s = 1; s < S; ++s) v[0] += v[s];
  put_four(p, m, n, v[0]);
}

template <int S>
int launch_reduce(const Args& p, hipStream_t st) {
  const long long quads = (long long)p.M * (p.N / 4);
  hipLaunchKernelGGL(int8_reduce_kernel<S>, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, p);
  return (int)hipGetLastError();
}

template <int RT, int TT, int KS, int NS, int WR, int WT, int WK>
int launch(const Args& p, hipStream_t st) {
  using C = Cfg<RT, TT, KS, NS, WR, WT, WK>;
  FERRET_HIP_CHECK((set_lds_limit_once<int8_tiled_kernel<RT, TT, KS, NS, WR, WT, WK>>(C::kLds)));
  hipLaunchKernelGGL((int8_tiled_kernel<RT, TT, KS, NS, WR, WT, WK>),
                     dim3((unsigned)(cdiv(p.N, C::kRows) * p.tok_tiles * p.splits)), dim3(C::kThreads), C::kLds, st, p);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace i8
}  // namespace ferret

int ferret_int8_square(int tile, const ferret::i8::Args& p, hipStream_t st);

// The product by one plan.
int ferret_int8_run(const ferret::i8::Plan& plan, ferret::i8::Args p, hipStream_t st) {
  using namespace ferret::i8;
  p.splits = plan.splits;
  p.tok_tiles = plan.tok_tiles;
  p.nt = plan.tok_tiles == 1;
  static_assert(kFirstSquare == 5 && kNumTiles == 12, "one case per tile");
  int rc = FERRET_ERR_SHAPE;
  switch (plan.tile) {
    case 0: rc = launch<1, 1, 512, 4, 1, 1, 8>(p, st); break;
    case 1: rc = launch<2, 1, 256, 6, 1, 1, 4>(p, st); break;
    case 2: rc = launch<6, 1, 256, 5, 2, 1, 4>(p, st); break;
    case 3: rc = launch<2, 2, 512, 4, 1, 1, 8>(p, st); break;
    case 4: rc = launch<6, 4, 256, 4, 2, 2, 2>(p, st); break;
    default: rc = ferret_int8_square(plan.tile, p, st); break;
  }
  if (rc != FERRET_OK || p.splits == 1) return rc;
  switch (p.splits) {
    case 2: return launch_reduce<2>(p, st);
    case 3: return launch_reduce<3>(p, st);
    case 4: return launch_reduce<4>(p, st);
    case 6: return launch_reduce<6>(p, st);
    case 8: return launch_reduce<8>(p, st);
  }
  return FERRET_ERR_SHAPE;
}

using namespace ferret;

// False where the shape is refused.
static bool int8_plan(int M, int N, int K, i8::Plan* plan) {
  if (M < 1 || M >= 1 << 22 || N < 8 || N >= 1 << 22 || N % 8 != 0 || K < 16 || K > 65536 || K % 16 != 0) return false;
  *plan = i8::plan(M, N, K);
  // a launch holds less than 2^32 threads, 512 at most to a work-group
  return i8::cdiv(N, i8::kTiles[plan->tile].rows) * plan->tok_tiles * plan->splits < 1 << 23;
}

extern "C" size_t ferret_int8_gemm_workspace(int M, int N, int K) {
  i8::Plan plan;
  return int8_plan(M, N, K, &plan) ? i8::workspace(plan, M, N) : 0;
}

extern "C" int ferret_int8_gemm(const void* a, const float* sa, const void* b, const float* sb, const void* residual,
                                void* y, int M, int N, int K, void* ws, size_t ws_bytes, void* stream) {
  FERRET_REQUIRE(a && sa && b && sb && y, FERRET_ERR_NULL);
  i8::Plan plan;
  FERRET_REQUIRE(int8_plan(M, N, K, &plan), FERRET_ERR_SHAPE);
  const auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  FERRET_REQUIRE(((bits(a) | bits(b) | bits(sb) | bits(residual) | bits(y)) & 15) == 0 && (bits(sa) & 3) == 0,
                 FERRET_ERR_ALIGN);
  const size_t need = i8::workspace(plan, M, N);
  FERRET_REQUIRE(need == 0 || (ws != nullptr && ws_bytes >= need && (bits(ws) & 15) == 0), FERRET_ERR_WORKSPACE);
  const uint64_t m = M, n = N, k = K;
  FERRET_REQUIRE(!clash({Range{y, m * n * 2}, Range{need != 0 ? ws : nullptr, need}},
                        {Range{a, m * k}, Range{sa, m * 4}, Range{b, n * k}, Range{sb, n * 4},
                         Range{residual == y ? nullptr : residual, m * n * 2}}),
                 FERRET_ERR_SHAPE);
  i8::Args p{};
  p.a = static_cast<const uint8_t*>(a);
  p.sa = sa;
  p.b = static_cast<const uint8_t*>(b);
  p.sb = sb;
  p.residual = static_cast<const uint16_t*>(residual);
  p.out = static_cast<uint16_t*>(y);
  p.partial = static_cast<int32_t*>(ws);
  p.M = M;
  p.N = N;
  p.K = K;
  return ferret_int8_run(plan, p, (hipStream_t)stream);
}
