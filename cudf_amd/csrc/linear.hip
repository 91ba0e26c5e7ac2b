// The matrix product of a layer with bias, activation and residual, and its gradients.
#include "encoder.cuh"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------------ activations
// gelu needs the normal distribution's integral: for a >= 0, 1 - Phi(a) = 2^P(a) with a polynomial of degree 8 in place of its
// logarithm, fitted here on 0..6 with the error of Phi levelled: 1.1e-7 of it evaluated in 32 bits, and from where 1 - Phi is below
// 1e-3 on 8e-5 of that; behind 6 P goes on falling (-5140 at 20), so the result goes to 0.  14 instructions, one of them
// transcendental; erff has 50, with which a product of 32768 x 1024 x 4096 took 75 us longer.  The other two activations are z times a logistic function.
__device__ __forceinline__ float normal_integral(float z)
{
  float const a = fabsf(z);
  float p       = -5.755030656473537e-07f;
  p             = fmaf(p, a, 1.026782047119923e-05f);
  p             = fmaf(p, a, -3.916913556167856e-05f);
  p             = fmaf(p, a, -5.069178878329694e-04f);
  p             = fmaf(p, a, 7.554566487669945e-03f);
  p             = fmaf(p, a, -5.283220857381821e-02f);
  p             = fmaf(p, a, -4.591012299060822e-01f);
  p             = fmaf(p, a, -1.151117563247681f);
  p             = fmaf(p, a, -9.999997615814209e-01f);
  float const q = __builtin_amdgcn_exp2f(p);
  return z < 0.f ? q : 1.f - q;
}

__device__ __forceinline__ float logistic(float u) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * u)); }

constexpr float kTwoRootTwoOverPi = 1.5957691216057308f;  // (1 + tanh u) / 2 is logistic(2 u)

template <int ACTIVATION>
__device__ __forceinline__ float activate(float z)
{
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_GELU) return z * normal_integral(z);
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_GELU_TANH) return z * logistic(kTwoRootTwoOverPi * fmaf(0.044715f * z * z, z, z));
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_SILU) return z * logistic(z);
  return z;
}

template <int ACTIVATION>
__device__ __forceinline__ float slope(float z)
{
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_GELU) {
    float const density = 0.39894228040143268f * __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
    return fmaf(z, density, normal_integral(z));
  }
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_GELU_TANH) {
    float const s = logistic(kTwoRootTwoOverPi * fmaf(0.044715f * z * z, z, z));
    float const c = fminf(fmaxf(z, -30.f), 30.f);  // (s is 0 or 1 long before, and z^2 must not become infinite beside it)
    return fmaf(c * (s - s * s), kTwoRootTwoOverPi * fmaf(0.134145f * c, c, 1.f), s);
  }
  if constexpr (ACTIVATION == NVTEXT_AMD_ACTIVATION_SILU) {
    float const s = logistic(z);
    return fmaf(z, s - s * s, s);
  }
  return 1.f;
}

// calls f with the activation as a constant
template <typename F>
__device__ __forceinline__ void with_activation(int activation, F&& f)
{
  switch (activation) {
    case NVTEXT_AMD_ACTIVATION_RELU: f(std::integral_constant<int, NVTEXT_AMD_ACTIVATION_RELU>{}); break;
    case NVTEXT_AMD_ACTIVATION_GELU: f(std::integral_constant<int, NVTEXT_AMD_ACTIVATION_GELU>{}); break;
    case NVTEXT_AMD_ACTIVATION_GELU_TANH: f(std::integral_constant<int, NVTEXT_AMD_ACTIVATION_GELU_TANH>{}); break;
    case NVTEXT_AMD_ACTIVATION_SILU: f(std::integral_constant<int, NVTEXT_AMD_ACTIVATION_SILU>{}); break;
    default: break;
  }
}

// What becomes of eight sums over k.
template <typename T>
struct Epilogue {
  Rows<const T> bias, residual;
  Rows<T> out, preactivation;
  int activation;

  struct Columns {
    float bias[8];
    __device__ __forceinline__ Columns(Epilogue const& e, int64_t j, int64_t n)
    {
      if (e.bias)
        load8(bias, e.bias.data + j, n - j);
      else
#pragma unroll
        for (int k = 0; k < 8; ++k) bias[k] = 0.f;
    }
  };
  // PAST: the results are stored past the caches (of a large product: 342 us instead of 367 for 32768 x 1024 x 4096 with two results)
  template <bool PAST = false>
  __device__ __forceinline__ void finish(float (&z)[8], Columns const& columns, int64_t i, int64_t j, int64_t n) const
  {
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] += columns.bias[k];
    if (preactivation) store8<PAST>(preactivation.row(i) + j, z, n - j);
    with_activation(activation, [&](auto which) {
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k] = activate<decltype(which)::value>(z[k]);
    });
    if (residual) {
      float r[8];
      load8(r, residual.row(i) + j, n - j);
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k] += r[k];
    }
    store8<PAST>(out.row(i) + j, z, n - j);
  }
};

// ------------------------------------------------------------------ products of 16-bit types
// out (i, j) = sum over k of a (i, k) * b (j, k) on the matrix cores.  An operand lies either with its k next to each other
// (K_NEXT: value (i, k) at i * stride + k) or with its rows next to each other (k * stride + i); both come into LDS as they lie,
// 64 values of k a stage, by loads that write LDS without a register in between.
//
// LDS image of a stage of EXT rows, EXT * 128 bytes, of which a wavefront's load fills 1 KB from one 16-byte piece a lane:
//   K_NEXT: row i has 128 bytes (whole cache lines: with 64 L2 answered as many requests for half the bytes), its piece c (8 values
//           of k) lies at c ^ (i & 7): the rows that a fragment reads at one c are spread over all banks.
//   else:   value k has EXT * 2 bytes, its units of 16 rows (32 bytes) lie at u ^ (k & 3 | (k >> 3 & 1) << 2), for the same reason;
//           a fragment is read by the transposing load, four values of k at a time.
// What lies outside the operands is read as zeros: its offset lies beyond the buffer's range, which is at most 2^31 bytes: the lines
// of a tile (K_NEXT) or of a stage, so lines of more values than most_line() allows are not for these loads (product_kernel has 64 bits).
constexpr int kStageK     = 64;
constexpr uint32_t kFar   = 0x80000000u;  // an offset outside every buffer, whatever is added for a row of the tile
constexpr int64_t most_line(int64_t lines) { return (int64_t{1} << 31) / (2 * lines); }  // values, of `lines` lines at a time

typedef float f32x4_t __attribute__((ext_vector_type(4)));
template <typename T>
using Fragment = T __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
using LdsBytes = __attribute__((address_space(3))) char*;

__device__ __forceinline__ f32x4_t multiply(Fragment<bf16_t> a, Fragment<bf16_t> b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4_t multiply(Fragment<half_t> a, Fragment<half_t> b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// (16 x 16 x 4 at a time: that value e of every lane goes into product e is as good an order of k as another)
__device__ __forceinline__ f32x4_t multiply(Fragment<float> a, Fragment<float> b, f32x4_t c)
{
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// An operand: a multiple of 8 values next to each other in each line, lines at multiples of 16 bytes.
struct Side {
  const void* data;
  int64_t stride;  // in values
};

// The same in every lane, and known to be.
__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

// 16 bytes a lane from base + offset to 16 bytes a lane from `to` on; zeros where the offset is not less than `range`.  Written out: the
// compiler would wait for loads that it knows to write LDS before every transposing read of LDS (a product of which one operand
// is read that way took 153 us instead of 118).  It has no register as a result, so it is waited for by stage_barrier alone.
__device__ __forceinline__ void load_to_lds(const char* base, uint32_t range, LdsBytes to, uint32_t offset)
{
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  uint64_t const address = reinterpret_cast<uint64_t>(base);
  // a buffer: address, no stride, length, plain 32-bit data
  u32x4 const buffer = {static_cast<uint32_t>(address), static_cast<uint32_t>(address >> 32) & 0xffffu, range, 0x00027000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to))), "v"(offset), "s"(buffer)
               : "memory");  // (m0 is set wherever the compiler uses it itself)
}

// What a wavefront loads of an operand for a stage: kPieces loads.  Lines behind the last, rows or values of k, lie behind the
// buffer's range; the other direction is looked at lane by lane.
template <bool K_NEXT, int EXT, int WAVES>
struct Loader {
  static constexpr int kPieces = EXT / 8 / WAVES;
  static constexpr int kLine   = EXT / 8;  // (not K_NEXT) lanes that a value of k takes
  const char* base;  // of the tile's first value of the next stage
  uint32_t line;     // bytes from a line to the next
  uint32_t rows;     // (K_NEXT) bytes of the rows that are there
  uint32_t offset[K_NEXT ? 1 : kPieces];
  int k_first;       // (K_NEXT) of the lane's pieces, in the stage

  // at the tile of rows from i0 on, and at value k0 of k
  __device__ __forceinline__ void aim(Side const& side, int64_t i0, int64_t extent, int64_t k0, int wave, int lane)
  {
    base = static_cast<const char*>(side.data) + 2 * (K_NEXT ? i0 * side.stride + k0 : k0 * side.stride + i0);
    line = static_cast<uint32_t>(side.stride * 2);
    if constexpr (K_NEXT) {
      rows            = static_cast<uint32_t>(extent - i0 < EXT ? extent - i0 : EXT) * line;
      int const row   = wave * kPieces * 8 + lane / 8;
      int const piece = (lane % 8) ^ (lane / 8);
      k_first         = piece * 8;
      offset[0]       = row * line + piece * 16;
    } else {
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        int const k = (wave * kPieces + p) * (kWave / kLine) + lane / kLine, at = lane % kLine;
        int const piece = ((at >> 1) ^ ((k & 3) | (k >> 3 & 1) << 2)) * 2 + (at & 1);
        offset[p] = i0 + piece * 8 < extent ? k * line + piece * 16 : kFar;
      }
    }
  }
  // Piece `p` of the next stage, of whose 64 values of k `here` are there, into `to`.
  __device__ __forceinline__ void load(LdsBytes to, int here, int wave, int p) const
  {
    LdsBytes const place = to + (wave * kPieces + p) * 1024;
    if constexpr (K_NEXT)
      load_to_lds(base, rows, place, (k_first < here ? offset[0] : kFar) + p * 8 * line);
    else
      load_to_lds(base, here * line, place, offset[p]);
  }
  __device__ __forceinline__ void next() { base += K_NEXT ? 2 * kStageK : static_cast<int64_t>(kStageK) * line; }
};

// Where a lane finds the fragments of 16 rows each, the first beginning at row `first` of the tile.
template <typename T, bool K_NEXT, int EXT>
struct Reader {
  uint32_t at;
  __device__ __forceinline__ Reader(int first, int lane)
  {
    int const i = lane % 16, g = lane / 16;
    if constexpr (K_NEXT)
      at = (first + i) * 128 + ((g ^ (i & 7)) * 16);
    else  // value k = 8 g + i / 4, and four further on
      at = (g * 8 + i / 4) * EXT * 2 + (((first / 16) ^ ((i >> 2) | (g & 1) << 2)) * 32) + i % 4 * 8;
  }
  // fragment `number` of the first or second 32 values of k
  __device__ __forceinline__ Fragment<T> read(LdsBytes stage, int half, int number) const
  {
    if constexpr (K_NEXT) {
      return *reinterpret_cast<__attribute__((address_space(3))) Fragment<T>*>(stage + (at ^ half * 64) + number * 2048);
    } else {
      LdsBytes const p   = stage + (at ^ number * 32) + half * 64 * EXT;
      s16x4_t const low  = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(p));
      s16x4_t const high = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(p + 4 * EXT * 2));
      s16x8_t const both = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(Fragment<T>, both);
    }
  }
};

// All wavefronts have come here, their reads of LDS are done, and of the loads of each all but the last N.  (Written out: a fence in
// front of the barrier would wait for all loads, because they write LDS.)
template <int N>
__device__ __forceinline__ void stage_barrier()
{
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);
  asm volatile("s_barrier" ::: "memory");
}

// f(0), ... f(N - 1) with the numbers as constants, so that arrays that they index stay in registers.
template <typename F, int... I>
__device__ __forceinline__ void for_each(std::integer_sequence<int, I...>, F&& f)
{
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void for_each(F&& f)
{
  for_each(std::make_integer_sequence<int, N>{}, f);
}

// A product: out (m x n) of operands a and b, with `depth` values of k in `parts` parts of `part` values; of several parts the sums go
// to sums [part][m][n] and are finished by join_kernel.
template <typename T>
struct Problem {
  Side a, b;
  int64_t m, n, depth, part;
  int32_t parts;
  float* sums;
  Epilogue<T> end;
};

// Where an item of work, a tile of the result and a part of the values of k, begins.
struct Item {
  int64_t i0, j0;
  int32_t part;
};

// A workgroup takes items of BM x BN one after the other.  WAVES_M x WAVES_N wavefronts, each with MI x NI fragments of 16 x 16.
// The loads are a stream of stages that goes on from an item into the next: the first two stages of an item come while the
// one before is finished and written, for which the wavefronts have LDS of their own (waiting for them anew at every item
// made 32768 x 1024 x 4096 a ninth longer).
template <typename T, bool A_NEXT, bool B_NEXT, int BM, int BN, int WAVES_M, int WAVES_N>
struct TileProduct {
  static constexpr int kWaves = WAVES_M * WAVES_N, MI = BM / WAVES_M / 16, NI = BN / WAVES_N / 16;
  static constexpr int kCols = NI * 16, kRowLanes = kCols / 8;  // of a wavefront's tile: columns, lanes that a row takes in the end
  static constexpr int kStage = (BM + BN) * 128, kLoads = (BM + BN) / 8 / kWaves;
  static constexpr int kLds = 2 * kStage + kWaves * 16 * kCols * 4;
  // as workgroup `block` of `blocks`
  static __device__ __forceinline__ void run(Problem<T> const& problem, LdsBytes stages, int32_t block, int32_t blocks);
};

template <typename T, bool A_NEXT, bool B_NEXT, int BM, int BN, int WAVES_M, int WAVES_N>
__device__ __forceinline__ void TileProduct<T, A_NEXT, B_NEXT, BM, BN, WAVES_M, WAVES_N>::run(Problem<T> const& problem, LdsBytes stages, int32_t block, int32_t blocks)
{
  Side const a = problem.a, b = problem.b;
  int64_t const m = problem.m, n = problem.n, depth = problem.depth, part = problem.part;
  int32_t const parts    = problem.parts;
  float* const sums      = problem.sums;
  Epilogue<T> const& end = problem.end;

  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  int const wm = wave / WAVES_N, wn = wave % WAVES_N;

  // Workgroups go to the eight XCDs in turn: each takes a run of items, within which eight tiles of rows share their columns.
  int32_t const tiles_m = uniform(static_cast<int32_t>((m + BM - 1) / BM)), tiles_n = uniform(static_cast<int32_t>((n + BN - 1) / BN)), tiles = tiles_m * tiles_n;
  int32_t const items = tiles * parts;
  constexpr int kXcds = 8, kGroup = 8;
  int32_t const xcd = block % kXcds, per_xcd = items / kXcds, more = items % kXcds;
  int32_t const begin = xcd * per_xcd + (xcd < more ? xcd : more), last = begin + per_xcd + (xcd < more ? 1 : 0);
  int32_t const stride = blocks / kXcds + (xcd < blocks % kXcds ? 1 : 0);  // workgroups of this XCD
  auto const place = [&](int32_t item) {
    int32_t const p = uniform(item / tiles), tile = item - p * tiles, group = uniform(tile / (kGroup * tiles_n)), in_group = tile - group * kGroup * tiles_n;
    int32_t const rows_here = tiles_m - group * kGroup < kGroup ? tiles_m - group * kGroup : kGroup;
    int32_t const column    = uniform(in_group / rows_here);
    return Item{static_cast<int64_t>(group * kGroup + in_group - column * rows_here) * BM, static_cast<int64_t>(column) * BN, p};
  };
  // (in 32 bits: a comparison of 64 is a vector one, whose operand was kept in memory and waited for at every item, with all loads)
  int32_t const depth32 = static_cast<int32_t>(depth), part32 = static_cast<int32_t>(part);
  auto const values_of  = [&](Item const& at) {
    int32_t const rest = depth32 - at.part * part32;
    return rest < part32 ? rest : part32;
  };

  Loader<A_NEXT, BM, kWaves> load_a;
  Loader<B_NEXT, BN, kWaves> load_b;
  Reader<T, A_NEXT, BM> const read_a(wm * MI * 16, lane);
  Reader<T, B_NEXT, BN> const read_b(wn * NI * 16, lane);
  int32_t const first = begin + block / kXcds;
  int32_t loaded      = first;  // the item whose stages are loaded
  int32_t left        = 0;      // values of k of it that are still to be loaded
  auto const aim = [&] {
    Item const at = place(loaded);
    load_a.aim(a, at.i0, m, at.part * part, wave, lane);
    load_b.aim(b, at.j0, n, at.part * part, wave, lane);
    left = values_of(at);
  };
  if (loaded >= last) return;
  aim();
  // Two stages are in LDS.  Load number `p` of the next one, into place `slot`; behind the last stage of all, zeros.
  auto const before_stage = [&] {
    if (left <= 0 && depth32 > 0 && loaded + stride < last) {
      loaded += stride;
      aim();
    }
  };
  auto const load = [&](int slot, int p) {
    LdsBytes const to = stages + slot * kStage;
    int const here    = uniform(left < 0 ? 0 : left < kStageK ? left : kStageK);
    if (p < BM / 8 / kWaves)
      load_a.load(to, here, wave, p);
    else
      load_b.load(to + BM * 128, here, wave, p - BM / 8 / kWaves);
    if (p == kLoads - 1) {
      load_a.next();
      load_b.next();
      left -= kStageK;
    }
  };
  f32x4_t sum[MI][NI];
  struct Fragments {
    Fragment<T> a[MI], b[NI];
  };
  Fragments f[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    before_stage();
#pragma unroll
    for (int p = 0; p < kLoads; ++p) load(s, p);
  }
  stage_barrier<kLoads>();
  // (in the order of the reads in the loop: what the compiler waits for there follows from both)
#pragma unroll
  for (int r = 0; r < MI + NI; ++r) {
    if (r == 0 || r > NI)
      f[0].a[r == 0 ? 0 : r - NI] = read_a.read(stages, 0, r == 0 ? 0 : r - NI);
    else
      f[0].b[r - 1] = read_b.read(stages + BM * 128, 0, r - 1);
    __builtin_amdgcn_sched_barrier(0);
  }
  // Multiplies the fragments of one half of a stage, reads those of the next and asks for stages to come: after each product, which
  // keeps the matrix core busy for 16 cycles, at most one read or load, in this order (left to itself, the compiler puts the
  // products together).  SECOND: the next half is the first of the other stage, for which everybody waits after a row of
  // products; this stage has been read then and makes room for the one after that.
  auto const step = [&](Fragments const& now, Fragments& next, int slot, auto second) {
    constexpr bool kSecond = decltype(second)::value;
    LdsBytes const from    = stages + (kSecond ? slot ^ 1 : slot) * kStage;
    if constexpr (kSecond) before_stage();
    // read number r: a fragment of a, all of b, the others of a
    auto const read = [&](int r) {
      if (r == 0 || r > NI)
        next.a[r == 0 ? 0 : r - NI] = read_a.read(from, kSecond ? 0 : 1, r == 0 ? 0 : r - NI);
      else
        next.b[r - 1] = read_b.read(from + BM * 128, kSecond ? 0 : 1, r - 1);
    };
    constexpr int kReads = MI + NI, kOps = kReads + (kSecond ? kLoads : 0), kFrom = kSecond ? NI : 0, kSlots = MI * NI - kFrom - 2;
    for_each<MI * NI>([&](auto slot_of) {
      constexpr int q = decltype(slot_of)::value, i = q / NI, j = q % NI;
      if constexpr (kSecond && q == NI) stage_barrier<0>();
      sum[i][j] = multiply(now.b[j], now.a[i], sum[i][j]);  // (the transposed tile: a lane has four values of a row)
      for_each<kOps>([&](auto op) {
        constexpr int o = decltype(op)::value;
        if constexpr (kFrom + o * kSlots / kOps == q) {
          // reads and loads in turn, as far as there are both
          constexpr int kBoth = kSecond ? (kReads < kLoads ? kReads : kLoads) : 0;
          if constexpr (o < 2 * kBoth) {
            if constexpr (o % 2 == 0)
              read(o / 2);
            else
              load(slot, o / 2);
          } else if constexpr (kReads > kBoth) {
            read(o - kBoth);
          } else {
            load(slot, o - kBoth);
          }
        }
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  int slot = 0;  // of the stage that is multiplied
  for (int32_t item = first; item < last; item += stride) {
    Item const at   = place(item);
    int const steps = (values_of(at) + kStageK - 1) / kStageK;
    for_each<MI * NI>([&](auto q) { sum[decltype(q)::value / NI][decltype(q)::value % NI] = f32x4_t{0.f, 0.f, 0.f, 0.f}; });
    for (int t = 0; t < steps; ++t) {
      step(f[0], f[1], slot, std::false_type{});
      step(f[1], f[0], slot, std::true_type{});
      slot ^= 1;
    }
    // Every wavefront turns its tile round in its own part of LDS, 16 rows at a time, and goes on with eight values of a row a lane.
    // (A row's units of four values lie at unit ^ row, within the row.)
    constexpr int kUnits = kCols / 4 < 16 ? kCols / 4 - 1 : 15;
    LdsBytes const mine = stages + 2 * kStage + wave * (16 * kCols * 4);
    int64_t const j     = at.j0 + wn * kCols + lane % kRowLanes * 8;
    typename Epilogue<T>::Columns const columns(end, j, n);
#pragma nounroll
    for (int rows = 0; rows < MI; ++rows) {
      for_each<MI * NI>([&](auto q) {
        constexpr int i = decltype(q)::value / NI, c = decltype(q)::value % NI;
        if (i == rows)
          *reinterpret_cast<__attribute__((address_space(3))) f32x4_t*>(mine + lane % 16 * kCols * 4 + ((c * 4 + lane / 16) ^ (lane % 16 & kUnits)) * 16) = sum[i][c];
      });
      wave_lds_fence();
#pragma nounroll
      for (int row = lane / kRowLanes; row < 16; row += kWave / kRowLanes) {
        auto const unit = [&](int u) { return *reinterpret_cast<__attribute__((address_space(3))) f32x4_t*>(mine + row * kCols * 4 + (u ^ (row & kUnits)) * 16); };
        f32x4_t const x = unit(lane % kRowLanes * 2), y = unit(lane % kRowLanes * 2 + 1);
        float z[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        int64_t const i = at.i0 + (wm * MI + rows) * 16 + row;
        if (i < m && j < n) {
          if (sums)
            store8(sums + (at.part * m + i) * n + j, z, n - j);
          else
            end.template finish<true>(z, columns, i, j, n);
        }
      }
      wave_lds_fence();
    }
  }
  stage_barrier<0>();  // (the loads behind the last stage write LDS as well, which is not to be given away before)
}

template <typename T, bool A_NEXT, bool B_NEXT, int BM, int BN, int WAVES_M, int WAVES_N>
__global__ void __launch_bounds__(WAVES_M * WAVES_N * kWave, 2) tile_product_kernel(Problem<T> problem)
{
  using Tiles = TileProduct<T, A_NEXT, B_NEXT, BM, BN, WAVES_M, WAVES_N>;
  __shared__ __attribute__((aligned(1024))) char lds[Tiles::kLds];
  Tiles::run(problem, (LdsBytes)lds, blockIdx.x, gridDim.x);
}

// ------------------------------------------------------------------ products of few rows
// A call for one token, or a few: nothing but the reading of the weights, which no workgroup shares.  A workgroup takes 16 outputs
// and all values of k, its wavefronts a run of k each; the weights go from memory into the fragments of the matrix
// instructions, kDeep loads of 16 bytes a lane on their way at a time, as do up to 16 * MI rows of x, which the caches hold; the
// wavefronts' sums are added up in order in LDS.  One launch and no temporaries.  Rows may lie anyhow.
template <typename T, int MI, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave) few_rows_kernel(Rows<const T> x, Rows<const T> weight, int64_t m, int64_t n, int64_t depth, Epilogue<T> end)
{
  constexpr int kDeep = sizeof(T) == 4 ? (MI == 1 && WAVES < 16 ? 4 : 2) : MI == 4 ? 4 : WAVES == 16 ? 6 : 8;  // (as many as the registers hold)
  __shared__ __attribute__((aligned(16))) float lds[WAVES][MI][16][20];  // (16 outputs a row, and room against conflicts)
  int const wave = threadIdx.x / kWave, lane = lane_id();
  int64_t const j0 = block_number() * 16;
  if (j0 >= n) return;
  const T* const w = weight.row(j0 + lane % 16 < n ? j0 + lane % 16 : n - 1);  // (outputs and rows behind the last: the last once more, not written)
  const T* rows[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) rows[i] = x.row(i * 16 + lane % 16 < m ? i * 16 + lane % 16 : m - 1);
  f32x4_t sum[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) sum[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  int64_t const steps = (depth + 31) / 32, each = (steps + WAVES - 1) / WAVES;
  int64_t const first = wave * each, last = first + each < steps ? first + each : steps;
  for (int64_t t = first; t < last; t += kDeep) {
    typename Eight<T>::type vw[kDeep], vx[kDeep][MI];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      int64_t const k = (t + u) * 32 + lane / 16 * 8, left = t + u < last ? depth - k : 0;
      vw[u]           = load_raw8<T>(w + k, left);
#pragma unroll
      for (int i = 0; i < MI; ++i) vx[u][i] = load_raw8<T>(rows[i] + k, left);
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
#pragma unroll
      for (int i = 0; i < MI; ++i) sum[i] = multiply(__builtin_bit_cast(Fragment<T>, vw[u]), __builtin_bit_cast(Fragment<T>, vx[u][i]), sum[i]);
  }
  // a lane has outputs lane / 16 * 4 .. + 3 of row lane % 16
#pragma unroll
  for (int i = 0; i < MI; ++i) *reinterpret_cast<f32x4_t*>(&lds[wave][i][lane % 16][lane / 16 * 4]) = sum[i];
  __syncthreads();
  int const i = threadIdx.x / 2, j = threadIdx.x % 2 * 8;
  if (i >= MI * 16 || i >= m || j0 + j >= n) return;
  float z[8] = {};
#pragma unroll
  for (int v = 0; v < WAVES; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] += lds[v][i / 16][i % 16][j + k];
  end.finish(z, typename Epilogue<T>::Columns(end, j0 + j, n), i, j0 + j, n);
}

// The gradients of a call of up to 16 * MI rows, in one launch or, where many outputs are cut into parts, two.  A workgroup takes 64
// inputs and a part of the outputs, 64 of them at a time: it makes d for them (which every workgroup of the part does anew: it
// is small), stages it and the 64 x 64 weights in LDS through registers, one stage ahead, and has of both the sums that x's gradient
// needs, which it keeps, and the weights' gradient, which is complete after one stage.  A wavefront has 16 of the inputs.
// Rows may lie anyhow.  d is rounded to the matrices' type, which is what the matrix instructions take: where there is an activation, the
// products' gradients are off by two roundings instead of one (0.0023 of a value in bfloat16 instead of 0.0017).  The bias'
// gradient adds d up before that.  Bound by launches and, of many weights, by memory: with gelu 7 x 64 x 64 4.5 us (11.1 in three
// launches with tiles), 34 x 924 x 4928 26 (35).
template <typename T>
struct FewRowsBackward {
  Rows<const T> grad, z, x, weight;
  Rows<T> x_grad, weight_grad;
  T* bias_grad;
  int activation;
  int64_t m, n, depth;
  int64_t part;  // outputs a part, a multiple of 64
  int32_t parts;
  float* sums;   // [part][m][depth], of several parts
};

constexpr int kFewEdge = 64, kFewPitch = kFewEdge + 8;

// eight values of k for each of 16 columns from `at` on, k along the rows
template <typename T>
__device__ __forceinline__ Fragment<T> read_turned(const T* at, int lane)
{
  int const i = lane % 16, g = lane / 16;
  auto const p       = (LdsBytes)(at + (g * 8 + i / 4) * kFewPitch + i % 4 * 4);
  s16x4_t const low  = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(p));
  s16x4_t const high = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(p + 4 * kFewPitch * 2));
  return __builtin_bit_cast(Fragment<T>, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
}

// four of a row's values from p on, of which n are there
template <typename T>
__device__ __forceinline__ void store4(T* p, f32x4_t const& f, int64_t n)
{
  typedef T V __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (n >= 4) {
    *reinterpret_cast<V*>(p) = V{static_cast<T>(f[0]), static_cast<T>(f[1]), static_cast<T>(f[2]), static_cast<T>(f[3])};
  } else {
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (k < n) p[k] = static_cast<T>(f[k]);
  }
}

template <typename T, int MI>
__global__ void __launch_bounds__(kThreads, 2) few_rows_backward_kernel(FewRowsBackward<T> w)
{
  // (MI = 1: 32 values of k all the same, the second half zeros)
  constexpr int kRows = MI == 1 ? 32 : MI * 16, KI = kRows / 32, kEach = kRows * 8 / kThreads;  // pieces of eight of d (and x) a thread
  static_assert(kEach >= 1 && kThreads == 4 * kWave);
  __shared__ __attribute__((aligned(16))) T ld[2][kRows][kFewPitch], lw[2][kFewEdge][kFewPitch], lx[kRows][kFewPitch];
  __shared__ float added[kThreads / 8][kFewEdge];
  using Raw = typename Eight<T>::type;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
  int const row = threadIdx.x / 8, piece = threadIdx.x % 8 * 8;  // of the first of a thread's pieces; the others lie 32 rows on
  int64_t const blocks = (w.depth + kFewEdge - 1) / kFewEdge, c0 = block_number() % blocks * kFewEdge, part = block_number() / blocks;
  if (part >= w.parts) return;
  int64_t const first = part * w.part, last = first + w.part < w.n ? first + w.part : w.n;
  bool const sum_bias = w.bias_grad && c0 == 0;

  // a piece of row i of `rows`, at column j of `cols`: zeros outside
  auto const load = [](Rows<const T> const& from, int64_t i, int64_t rows, int64_t j, int64_t cols) {
    Raw v{};
    if (i < rows && j < cols) {
      v = load_row8<T>(from.row(i), j, cols);
      settle_row8<T>(v, j, cols);
    }
    return v;
  };
  Raw vg[kEach], vz[kEach], vw[2];
  auto const ask = [&](int64_t r0) {
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      vg[u] = load(w.grad, row + u * 32, w.m, r0 + piece, w.n);
      if (w.z) vz[u] = load(w.z, row + u * 32, w.m, r0 + piece, w.n);
    }
    if (w.x_grad) {
#pragma unroll
      for (int u = 0; u < 2; ++u) vw[u] = load(w.weight, r0 + row + u * 32, w.n, c0 + piece, w.depth);
    }
  };
  ask(first);
#pragma unroll
  for (int u = 0; u < kEach; ++u) *reinterpret_cast<Raw*>(&lx[row + u * 32][piece]) = load(w.x, row + u * 32, w.m, c0 + piece, w.depth);
  f32x4_t sum[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) sum[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  Fragment<T> fx[KI];
  int64_t const j = c0 + wave * 16 + lane / 16 * 4;  // the lane's four inputs
  int buffer      = 0;
  for (int64_t r0 = first; r0 < last; r0 += kFewEdge, buffer ^= 1) {
    float bias[8] = {};
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      float g[8];
      widen<T>(g, vg[u]);
      if (w.z) {
        float v[8];
        widen<T>(v, vz[u]);
        with_activation(w.activation, [&](auto which) {
#pragma unroll
          for (int k = 0; k < 8; ++k) g[k] *= slope<decltype(which)::value>(v[k]);
        });
      }
      Raw d;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        d[k] = static_cast<T>(g[k]);
        bias[k] += g[k];
      }
      *reinterpret_cast<Raw*>(&ld[buffer][row + u * 32][piece]) = d;
    }
    if (w.x_grad) {
#pragma unroll
      for (int u = 0; u < 2; ++u) *reinterpret_cast<Raw*>(&lw[buffer][row + u * 32][piece]) = vw[u];
    }
    if (sum_bias) {
      if (r0 > first) __syncthreads();  // (what was added before has been read)
#pragma unroll
      for (int k = 0; k < 8; ++k) added[row][piece + k] = bias[k];
    }
    __syncthreads();
    if (r0 == first) {
#pragma unroll
      for (int k = 0; k < KI; ++k) fx[k] = read_turned<T>(&lx[k * 32][wave * 16], lane);
    }
    ask(r0 + kFewEdge);  // (behind the last: zeros)
    if (sum_bias && threadIdx.x < kFewEdge && r0 + threadIdx.x < w.n) {
      float all = 0.f;
      for (int q = 0; q < kThreads / 8; ++q) all += added[q][threadIdx.x];
      w.bias_grad[r0 + threadIdx.x] = static_cast<T>(all);
    }
    if (w.x_grad) {
#pragma unroll
      for (int k = 0; k < kFewEdge / 32; ++k) {
        Fragment<T> const fw = read_turned<T>(&lw[buffer][k * 32][wave * 16], lane);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          Fragment<T> const fd = *reinterpret_cast<const Fragment<T>*>(&ld[buffer][i * 16 + lane % 16][k * 32 + lane / 16 * 8]);
          sum[i]               = multiply(fw, fd, sum[i]);  // (a lane has four inputs of a row)
        }
      }
    }
    if (w.weight_grad) {
#pragma unroll
      for (int r = 0; r < kFewEdge / 16; ++r) {
        f32x4_t of_weight = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KI; ++k) of_weight = multiply(fx[k], read_turned<T>(&ld[buffer][k * 32][r * 16], lane), of_weight);
        int64_t const o = r0 + r * 16 + lane % 16;
        if (o < w.n && j < w.depth) store4(w.weight_grad.row(o) + j, of_weight, w.depth - j);
      }
    }
  }
  if (!w.x_grad || j >= w.depth) return;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    int64_t const of = i * 16 + lane % 16;
    if (of >= w.m) continue;
    if (w.sums)
      store4(w.sums + (part * w.m + of) * w.depth + j, sum[i], w.depth - j);
    else
      store4(w.x_grad.row(of) + j, sum[i], w.depth - j);
  }
}

// ------------------------------------------------------------------ before and after
// The parts of a product that was cut along k, eight of them asked for at a time.  Where there are many results a thread has eight of
// them, else (`spread`) a workgroup has 64 times eight, and each of its wavefronts a run of the parts.  (4 parts of 4096 x 1024
// 19 us, spread 26; many parts of a small result 55 -> 39 us for the whole of a gradient of 34 x 924 x 4928.)
template <typename T>
struct Join {
  const float* sums;
  int64_t parts, m, n;
  Epilogue<T> end;
  bool spread;
  // workgroups
  int64_t blocks() const { return spread ? (m * ((n + 7) / 8) + kWave - 1) / kWave : (m * ((n + 7) / 8) + kThreads - 1) / kThreads; }
  __device__ __forceinline__ void add(float (&z)[8], int64_t i, int64_t j, int64_t first, int64_t last) const
  {
#pragma unroll 8
    for (int64_t p = first; p < last; ++p) {
      float more[8];
      load8(more, sums + (p * m + i) * n + j, n - j);
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k] += more[k];
    }
  }
  __device__ __forceinline__ void run(int64_t block) const
  {
    constexpr int kWaves = kThreads / kWave;
    __shared__ float lds[kWaves][8][kWave];
    int const wave = threadIdx.x / kWave, lane = lane_id();
    int64_t const blocks = (n + 7) / 8, at = spread ? block * kWave + lane : block * kThreads + threadIdx.x;
    int64_t const i = m * blocks <= UINT32_MAX ? static_cast<uint32_t>(at) / static_cast<uint32_t>(blocks) : at / blocks, j = (at - i * blocks) * 8;
    bool const here = at < m * blocks;
    float z[8]      = {};
    if (!spread) {
      if (!here) return;
      add(z, i, j, 0, parts);
    } else {
      int64_t const each = (parts + kWaves - 1) / kWaves, first = wave * each, last = first + each < parts ? first + each : parts;
      if (here) add(z, i, j, first, last);
#pragma unroll
      for (int k = 0; k < 8; ++k) lds[wave][k][lane] = z[k];
      __syncthreads();
      if (wave != 0 || !here) return;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int w = 1; w < kWaves; ++w) z[k] += lds[w][k][lane];
    }
    end.finish(z, typename Epilogue<T>::Columns(end, j, n), i, j, n);
  }
};

template <typename T>
Join<T> join_of(const float* sums, int64_t parts, int64_t m, int64_t n, Epilogue<T> const& end)
{
  return Join<T>{sums, parts, m, n, end, m * ((n + 7) / 8) < 256 * static_cast<int64_t>(device_cus())};
}

// The parts of the sums of columns: a workgroup 64 columns, a wavefront a run of parts.
template <typename T>
struct JoinColumns {
  const float* sums;
  int64_t parts, n;
  T* out;
  __device__ __forceinline__ void run(int64_t block) const
  {
    constexpr int kWaves = kThreads / kWave;
    __shared__ float lds[kWaves][kWave];
    int const wave = threadIdx.x / kWave, lane = lane_id();
    int64_t const j = block * kWave + lane, each = (parts + kWaves - 1) / kWaves, first = wave * each, last = first + each < parts ? first + each : parts;
    float sum = 0.f;
    if (j < n) {
#pragma unroll 8
      for (int64_t p = first; p < last; ++p) sum += sums[p * n + j];
    }
    lds[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || j >= n) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += lds[w][lane];
    out[j] = static_cast<T>(sum);
  }
};

// What is left after the products, in one launch: `first` workgroups, `second` workgroups, and the columns'.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_kernel(Join<T> a, int64_t first, Join<T> b, int64_t second, JoinColumns<T> columns)
{
  int64_t const block = block_number();
  if (block < first)
    a.run(block);
  else if (block < first + second)
    b.run(block - first);
  else
    columns.run(block - first - second);
}

// From a line of a copy to the next: a multiple of 8 values, or of 64, whole cache lines, where these are few more (a stage's 128
// bytes lie in one of them then: 1777 x 2051 x 1003 33 us instead of 38).
inline int64_t copy_stride(int64_t cols) { return cols >= 512 ? (cols + 63) / 64 * 64 : (cols + 7) / 8 * 8; }

// Lines of `cols` values, aligned anyhow, into lines of a multiple of 8 values, zeros behind the last.
template <typename T>
struct Align {
  Rows<const T> in;
  int64_t rows, cols;
  Rows<T> out;
  __device__ __forceinline__ void run(int64_t block) const
  {
    int64_t const blocks = (cols + 7) / 8, at = block * kThreads + threadIdx.x;
    if (at >= rows * blocks) return;
    // (32 bits where they do: a division of 64 takes as long as the rest)
    int64_t const i = rows * blocks <= UINT32_MAX ? static_cast<uint32_t>(at) / static_cast<uint32_t>(blocks) : at / blocks, j = (at - i * blocks) * 8;
    auto v = load_row8<T>(in.row(i), j, cols);
    settle_row8<T>(v, j, cols);
    *reinterpret_cast<typename Eight<T>::type*>(out.row(i) + j) = v;
  }
};

// d = grad * activation'(z) where it is wanted, rounded as in few_rows_backward_kernel (d's rows have a multiple of 8 values, zeros
// behind the last), and the sums of the columns of it in 32 bits: a workgroup takes up to 512 columns and every count-th run of rows, `lanes` lanes of a wavefront a row (fewer than
// 64 for narrow rows, which lie side by side then); the sums are added up in order in the end, to the bias' gradient itself if that
// is all (count = 1).
template <typename T>
struct Slopes {
  Rows<const T> grad, z;
  int activation;
  int64_t rows, cols;
  Rows<T> d;
  int32_t lanes;
  int64_t count;
  float* parts;
  T* bias;
  static int32_t lanes_of(int64_t cols) { return cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 256 ? 32 : kWave; }
  // runs of rows: up to 64 for each place in a wavefront are left to one workgroup, without parts
  static int64_t count_of(int64_t rows, int32_t lanes)
  {
    int64_t const across = kWave / lanes;
    return rows <= 64 * across ? 1 : std::min<int64_t>((rows + 16 * across - 1) / (16 * across), 256);
  }
  int64_t workgroups() const { return (cols + 8 * lanes - 1) / (8 * lanes) * count; }
  __device__ __forceinline__ void run(int64_t block, float (*lds)[kThreads]) const
  {
    constexpr int kWaves = kThreads / kWave, kAtOnce = 4;  // rows that a lane asks for at a time
    int const across     = kWave / lanes, place = threadIdx.x / lanes, at = threadIdx.x % lanes;
    int64_t const slices = (cols + 8 * lanes - 1) / (8 * lanes), slice = block % slices, number = block / slices;
    int64_t const j      = (slice * lanes + at) * 8;
    float sum[8]         = {};
    if (j < cols) {
      int64_t const step = count * kWaves * across;
      for (int64_t first = number * kWaves * across + place; first < rows; first += kAtOnce * step) {
        typename Eight<T>::type vg[kAtOnce], vz[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          int64_t const i = first + u * step < rows ? first + u * step : first;  // (behind the last the first once more, not counted)
          vg[u]           = load_row8<T>(grad.row(i), j, cols);
          if (z) vz[u] = load_row8<T>(z.row(i), j, cols);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          int64_t const i = first + u * step;
          if (i >= rows) break;
          float g[8], v[8];
          if (cols % 8 != 0) settle_row8<T>(vg[u], j, cols);
          widen<T>(g, vg[u]);
          if (z) {
            if (cols % 8 != 0) settle_row8<T>(vz[u], j, cols);
            widen<T>(v, vz[u]);
            with_activation(activation, [&](auto which) {
#pragma unroll
              for (int k = 0; k < 8; ++k) g[k] *= slope<decltype(which)::value>(v[k]);
            });
          }
          if (d) store8(d.row(i) + j, g, 8);
#pragma unroll
          for (int k = 0; k < 8; ++k) sum[k] += g[k];
        }
      }
    }
    if (!parts && !bias) return;
#pragma unroll
    for (int k = 0; k < 8; ++k) lds[k][threadIdx.x] = sum[k];
    __syncthreads();
    if (place != 0 || j >= cols) return;
    for (int p = 1; p < kWaves * across; ++p)
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += lds[k][p * lanes + at];
    if (bias)
      store8(bias + j, sum, cols - j);
    else
      store8(parts + number * cols + j, sum, cols - j);
  }
};

// What the products need, in one launch: `first` workgroups, `second` workgroups, and `third`, the slopes'.
template <typename T>
__global__ void __launch_bounds__(kThreads) prepare_kernel(Align<T> a, int64_t first, Align<T> b, int64_t second, Slopes<T> slopes, int64_t third)
{
  __shared__ float lds[8][kThreads];
  int64_t const block = block_number();
  if (block < first)
    a.run(block);
  else if (block < first + second)
    b.run(block - first);
  else if (block < first + second + third)
    slopes.run(block - first - second, lds);
}

// The two products of a gradient in one launch: the first `first` workgroups (of which `used` have work) take that of x, those up to
// `last` that of the weights, the others, if any, the sums of the columns (where d is grad, so that nothing waits for them: a
// launch less: 4848 x 64 x 320 16 us instead of 20).
template <typename T>
__global__ void __launch_bounds__(256, 2) gradient_products_kernel(Problem<T> of_x, Problem<T> of_weight, int32_t first, int32_t used, int32_t last, Slopes<T> slopes)
{
  using Tiles = TileProduct<T, true, false, 128, 128, 2, 2>;
  __shared__ __attribute__((aligned(1024))) char lds[Tiles::kLds];
  int32_t const block = static_cast<int32_t>(blockIdx.x);
  if (block >= last)
    slopes.run(block - last, reinterpret_cast<float(*)[kThreads]>(lds));
  else if (block >= first)
    TileProduct<T, false, false, 128, 128, 2, 2>::run(of_weight, (LdsBytes)lds, block - first, last - first);
  else if (block < used)
    Tiles::run(of_x, (LdsBytes)lds, block, used);
}

// ------------------------------------------------------------------ products of 32-bit types
// The same of float, on the matrix cores' products of 16 x 16 x 4, which keep float's precision at a sixteenth of the rate: so slow
// that plain loads through registers, one stage of 16 values of k ahead, keep up, and rows may lie anyhow.  A stage lies in
// LDS as [k][row], lines 16 banks apart from each other: the four lines that a fragment is read from take all 64.
// Bound by the matrix cores: 8192 x 1024 outputs of 4096 values 610 us, 113 TFLOP/s of 157 (a product of plain additions and
// multiplications in tiles of 64 x 64: 1440).  16-bit types whose lines are too wide for load_to_lds (more than 2^23 values next to
// each other in k, else 2^24) are widened on their way and multiplied here, where places are counted in 64 bits: 128 x 64 outputs of 8388672
// values 2.0 ms (of 64 values less, in tiles, 6.5).
constexpr int kStage32 = 16;

template <typename T, bool K_NEXT, int EXT>
struct Loader32 {
  static constexpr int kPieces = EXT * kStage32 / 4 / kThreads;  // of four values a thread
  static constexpr int kLine   = EXT / 4;                        // (not K_NEXT) threads that a value of k takes
  static constexpr int kStride = EXT + 16;                       // of a line in LDS
  typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  Four v[kPieces];
  static __device__ __forceinline__ int row_of(int p) { return K_NEXT ? p * (kThreads / 4) + threadIdx.x / 4 : threadIdx.x % kLine * 4; }
  static __device__ __forceinline__ int k_of(int p) { return K_NEXT ? threadIdx.x % 4 * 4 : p * (kThreads / kLine) + threadIdx.x / kLine; }
  // rows from i0 on of `extent`, values from k0 on up to `last`; zeros behind them
  __device__ __forceinline__ void load(Side const& side, int64_t i0, int64_t extent, int64_t k0, int64_t last)
  {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      int64_t const i = i0 + row_of(p), k = k0 + k_of(p);
      int64_t const left = K_NEXT ? (i < extent ? last - k : 0) : (k < last ? extent - i : 0);
      const T* const at  = static_cast<const T*>(side.data) + (K_NEXT ? i * side.stride + k : k * side.stride + i);
      v[p]               = Four{};
      if (left >= 4) {
        v[p] = *reinterpret_cast<const Four*>(at);
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < left) v[p][e] = at[e];
      }
    }
  }
  __device__ __forceinline__ void store(float* lds) const
  {
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e) lds[(k_of(p) + (K_NEXT ? e : 0)) * kStride + row_of(p) + (K_NEXT ? 0 : e)] = static_cast<float>(v[p][e]);
  }
};

template <typename T, bool A_NEXT, bool B_NEXT, int BN>
__global__ void __launch_bounds__(kThreads, 2) product_kernel(Problem<T> problem)
{
  constexpr int BM = 128, MI = BM / 32, NI = BN / 32, kCols = NI * 16, kRowLanes = kCols / 8;  // 2 x 2 wavefronts
  constexpr int kA = kStage32 * (BM + 16), kB = kStage32 * (BN + 16);
  __shared__ __attribute__((aligned(16))) float lds[2][kA + kB];
  static_assert(4 * 16 * kCols <= 2 * (kA + kB));
  int64_t const m = problem.m, n = problem.n;
  int const wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id(), wm = wave / 2, wn = wave % 2;
  // workgroups go to the eight XCDs in turn: each takes a run of tiles
  int32_t const tiles_n = static_cast<int32_t>((n + BN - 1) / BN), tiles = static_cast<int32_t>((m + BM - 1) / BM) * tiles_n;
  int32_t const items = tiles * problem.parts, number = static_cast<int32_t>(block_number()), xcd = number % 8, per_xcd = items / 8, more = items % 8;
  if (number >= items) return;
  int32_t const item = xcd * per_xcd + (xcd < more ? xcd : more) + number / 8, part = item / tiles, tile = item % tiles;
  int64_t const i0 = static_cast<int64_t>(tile / tiles_n) * BM, j0 = static_cast<int64_t>(tile % tiles_n) * BN;
  int64_t const first = part * problem.part, last = first + problem.part < problem.depth ? first + problem.part : problem.depth;
  Loader32<T, A_NEXT, BM> a;
  Loader32<T, B_NEXT, BN> b;
  f32x4_t sum[MI][NI] = {};
  a.load(problem.a, i0, m, first, last);
  b.load(problem.b, j0, n, first, last);
  int buffer = 0;
  for (int64_t k0 = first; k0 < last; k0 += kStage32, buffer ^= 1) {
    float *const la = lds[buffer], *const lb = la + kA;
    a.store(la);
    b.store(lb);
    __syncthreads();
    a.load(problem.a, i0, m, k0 + kStage32, last);
    b.load(problem.b, j0, n, k0 + kStage32, last);
#pragma unroll
    for (int k = 0; k < kStage32; k += 4) {
      float fa[MI], fb[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = la[(k + lane / 16) * (BM + 16) + (wm * MI + i) * 16 + lane % 16];
#pragma unroll
      for (int j = 0; j < NI; ++j) fb[j] = lb[(k + lane / 16) * (BN + 16) + (wn * NI + j) * 16 + lane % 16];
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) sum[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j], fa[i], sum[i][j], 0, 0, 0);  // (transposed: a lane has four values of a row)
    }
  }
  // every wavefront turns its tile round, 16 rows at a time, as above
  __syncthreads();
  constexpr int kUnits = kCols / 4 - 1;
  float* const mine    = &lds[0][0] + wave * 16 * kCols;
  int64_t const j      = j0 + wn * kCols + lane % kRowLanes * 8;
  typename Epilogue<T>::Columns const columns(problem.end, j, n);
#pragma unroll
  for (int rows = 0; rows < MI; ++rows) {
#pragma unroll
    for (int c = 0; c < NI; ++c) *reinterpret_cast<f32x4_t*>(mine + lane % 16 * kCols + ((c * 4 + lane / 16) ^ (lane % 16 & kUnits)) * 4) = sum[rows][c];
    wave_lds_fence();
#pragma nounroll
    for (int row = lane / kRowLanes; row < 16; row += kWave / kRowLanes) {
      auto const unit = [&](int u) { return *reinterpret_cast<const f32x4_t*>(mine + row * kCols + (u ^ (row & kUnits)) * 4); };
      f32x4_t const x = unit(lane % kRowLanes * 2), y = unit(lane % kRowLanes * 2 + 1);
      float z[8]      = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      int64_t const i = i0 + (wm * MI + rows) * 16 + row;
      if (i < m && j < n) {
        if (problem.sums)
          store8(problem.sums + (part * m + i) * n + j, z, n - j);
        else
          problem.end.finish(z, columns, i, j, n);
      }
    }
    wave_lds_fence();
  }
}

// An operand of a product of `extent` rows and `depth` values of k each.
template <typename T>
struct Factor {
  Rows<const T> rows;
  bool k_next;          // value (i, k) in line i, else in line k
  bool padded = false;  // lines have a multiple of 8 values, zeros behind the last

  int64_t lines(int64_t extent, int64_t depth) const { return k_next ? extent : depth; }
  int64_t cols(int64_t extent, int64_t depth) const { return k_next ? depth : extent; }
  // the most values from a line to the next that Loader can take, of tiles of so many rows
  int64_t most_stride(int64_t tile_rows) const { return most_line(k_next ? tile_rows : kStageK); }
  // fits what Side and Loader ask for
  bool is_aligned(int64_t extent, int64_t depth) const
  {
    return reinterpret_cast<uintptr_t>(rows.data) % 16 == 0 && rows.stride % 8 == 0 && (padded || cols(extent, depth) % 8 == 0) && rows.stride <= most_stride(128);
  }
  // whether lines next to each other, as a copy has them, fit tiles of so many rows
  bool copy_fits(int64_t extent, int64_t depth, int64_t tile_rows) const { return copy_stride(cols(extent, depth)) <= most_stride(tile_rows); }
};

// How a product is shared out: tiles of 256 x 256, 128 x 128 or 128 x 64, and so many parts of the values of k.
enum class Tile { k256, k128, k64 };
struct Plan {
  Tile tile;
  int32_t parts;
  int64_t part;  // values of k a part
  int64_t rows() const { return tile == Tile::k256 ? 256 : 128; }
  int64_t cols() const { return tile == Tile::k256 ? 256 : tile == Tile::k128 ? 128 : 64; }
  int64_t tiles(int64_t m, int64_t n) const { return (m + rows() - 1) / rows() * ((n + cols() - 1) / cols()); }
};

// The one that takes the least by this measure, in microseconds, fitted to products of 256 x 256 to 4096 x 4096 with 64 to 4096
// values of k: a launch, then rounds of workgroups, each with so much for a stage of 64 values of k (more where all CUs are busy) and
// for writing its tile; parts are written and read once more.  (4096 x 4096 x 64: 14.7 us in large tiles, 15.3 in those of 128;
// x 4096: 108 and 124.  2048 x 2048 x 4096: 80 and 48; 128 x 4096 x 4096: 77 and 44 in one part, 31 and 21 in four.  In tiles of 128
// and in half ones: 512 x 512 x 512 9.3 and 7.0; 2048 x 1024 x 1024 13.2 and 10.4; 4096 x 1024 x 1024 14.7 and 14.3.)  `halves`:
// both operands have their k next to each other, which half tiles are made for.  `large`: lines are not too wide for tiles of 256 rows.
inline Plan plan_product(int64_t m, int64_t n, int64_t depth, bool halves, bool large)
{
  int64_t const cus = device_cus(), steps = std::max<int64_t>(1, (depth + kStageK - 1) / kStageK);
  Plan best{Tile::k128, 1, std::max<int64_t>(depth, 1)};
  double least = 1e300;
  for (Tile tile : {Tile::k256, Tile::k128, Tile::k64}) {
    if (tile == Tile::k64 ? !halves : tile == Tile::k256 && !large) continue;
    for (int64_t parts = 1; parts <= std::min<int64_t>(steps, 32); ++parts) {
      int64_t const each = (steps + parts - 1) / parts, really = (steps + each - 1) / each;
      if (really != parts) continue;
      Plan const plan{tile, static_cast<int32_t>(parts), each * kStageK};
      int64_t const groups = plan.tiles(m, n) * parts, load = (groups + cus - 1) / cus;  // workgroups, and of them a CU
      double const busy    = std::min(1.0, static_cast<double>(groups) / cus);
      double work          = 0;
      switch (tile) {
        case Tile::k256: work = 6 + load * (each * (1.05 + 0.45 * busy) + 5); break;
        case Tile::k128: work = load == 1 ? 6 + each * (0.4 + 0.25 * busy) : 4 + (load + 1) / 2 * (each * 0.92 + 5); break;
        case Tile::k64: work = load == 1 ? 4 + each * (0.38 + 0.14 * busy) : 3 + (load + 1) / 2 * (each * 0.66 + 2); break;
      }
      double const time = work + (parts > 1 ? 3 + parts * m * n * 8e-6 / 5 : 0);
      if (time < least) {
        least = time;
        best  = plan;
      }
    }
  }
  return best;
}

// The same for product_kernel, in tiles of 128 x 128 or 128 x 64: a stage of 16 values of k takes the matrix cores 0.9 us or half of
// that.  At most `most` parts.
inline Plan plan_product32(int64_t m, int64_t n, int64_t depth, int64_t most)
{
  int64_t const cus = device_cus(), steps = std::max<int64_t>(1, (depth + kStage32 - 1) / kStage32);
  Plan best{Tile::k128, 1, std::max<int64_t>(depth, 1)};
  double least = 1e300;
  for (Tile tile : {Tile::k128, Tile::k64}) {
    for (int64_t parts = 1; parts <= std::min<int64_t>(steps, most); ++parts) {
      int64_t const each = (steps + parts - 1) / parts;
      if ((steps + each - 1) / each != parts) continue;
      Plan const plan{tile, static_cast<int32_t>(parts), each * kStage32};
      int64_t const load = (plan.tiles(m, n) * parts + cus - 1) / cus;
      double const time  = 5 + load * (each * (tile == Tile::k128 ? 0.95 : 0.5) + 2) + (parts > 1 ? 3 + parts * m * n * 8e-6 / 5 : 0);
      if (time < least) {
        least = time;
        best  = plan;
      }
    }
  }
  return best;
}

// Whether few_rows_kernel takes less time than tiles: microseconds of either, fitted to calls of 1 to 64 rows with 64 to 8192
// inputs and outputs.  It goes through k in one workgroup for 16 outputs, which takes longer with every 16 rows; tiles may be cut along k and
// joined, and read the weights as fast as memory gives them.  Rows that tiles cannot read are copied for them, and read at half the rate here.
// (`aligned`: by their width, not by where they lie: the two add in different orders, and results are to depend on sizes alone.)
// (16 rows: 1024 to 4096 4.2 us against 8.7, 4096 to 1024 10.0 against 9.7, 8192 to 8192 34 against 27, 2051 to 1003 12.0 against 13.5; 64 rows: 7.4 against 9.2,
// 20 against 11, 73 against 29, 24 against 15.)
inline double few_rows_time(int64_t m, int64_t n, int64_t depth)
{
  double const by_16 = m <= 16 ? 1 : m <= 32 ? 2 : 4;
  return 3 + 0.95 * (depth / 1024.0) * (1 + by_16) * static_cast<double>((n + 16 * 256 - 1) / (16 * 256));
}
inline bool few_rows_are_faster(int64_t m, int64_t n, int64_t depth, bool aligned)
{
  if (m > 64) return false;
  double const few   = few_rows_time(m, n, depth);
  double const tiles = 2 + std::max(8.5 + 0.7 * (depth / 1024.0), static_cast<double>(n) * depth * 2 / 4.6e6);  // (2: memory for the parts)
  return aligned ? few < tiles : 1.9 * few < tiles + 5;
}

inline int64_t blocks_of(int64_t work) { return (work + kThreads - 1) / kThreads; }

// out (m x n) = a (m x depth) * b (n x depth)^T, by tiles: what it takes, and its launch.
template <typename T>
struct Product {
  Factor<T> a, b;
  int64_t m, n, depth;
  Epilogue<T> end;
  Plan plan{};
  bool plain = sizeof(T) == 4;  // by product_kernel
  bool copy_a = false, copy_b = false;
  float* sums = nullptr;

  bool wanted() const { return m > 0 && n > 0; }
  bool fits() const { return (m + 127) / 128 * ((n + 63) / 64) <= (1 << 25) && depth <= INT32_MAX - (1 << 20); }
  void make_plan()
  {
    // (what decides follows from sizes alone: rows further apart than they are wide are copied)
    plain = sizeof(T) == 4 || !a.copy_fits(m, depth, 128) || !b.copy_fits(n, depth, 128);
    if (plain) {
      // (very wide: as many parts as there are CUs, there is little else to share out)
      plan = plan_product32(m, n, depth, sizeof(T) == 4 ? 32 : 256);
      return;
    }
    bool const large = a.copy_fits(m, depth, 256) && b.copy_fits(n, depth, 256);
    plan             = plan_product(m, n, depth, a.k_next && b.k_next, large);
    copy_a           = depth > 0 && !(a.is_aligned(m, depth) && a.rows.stride <= a.most_stride(plan.rows()));
    copy_b           = depth > 0 && !(b.is_aligned(n, depth) && b.rows.stride <= b.most_stride(plan.rows()));
  }
  static size_t copy_bytes(Factor<T> const& f, int64_t extent, int64_t depth)
  {
    return static_cast<size_t>(f.lines(extent, depth)) * static_cast<size_t>(copy_stride(f.cols(extent, depth))) * sizeof(T);
  }
  size_t bytes_a() const { return copy_a ? copy_bytes(a, m, depth) : 0; }
  size_t bytes_b() const { return copy_b ? copy_bytes(b, n, depth) : 0; }
  size_t bytes_sums() const { return plan.parts > 1 ? static_cast<size_t>(plan.parts) * static_cast<size_t>(m * n) * sizeof(float) : 0; }
  static Align<T> align(Factor<T>& f, int64_t extent, int64_t depth, T* to)
  {
    int64_t const cols = f.cols(extent, depth);
    Align<T> const copy{f.rows, f.lines(extent, depth), cols, {to, copy_stride(cols)}};
    f.rows   = Rows<const T>{to, copy_stride(cols)};
    f.padded = true;
    return copy;
  }
  Problem<T> problem() const { return Problem<T>{{a.rows.data, a.rows.stride}, {b.rows.data, b.rows.stride}, m, n, depth, plan.part, plan.parts, sums, end}; }
  // workgroups: as many as the CUs hold at once
  int64_t workgroups() const
  {
    return std::min<int64_t>(plan.tiles(m, n) * plan.parts, (plan.tile == Tile::k256 ? 1 : 2) * static_cast<int64_t>(device_cus()));
  }
  template <bool A_NEXT, bool B_NEXT, int BM, int BN, int WAVES_M, int WAVES_N>
  void launch_as(hipStream_t stream) const
  {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(tile_product_kernel<T, A_NEXT, B_NEXT, BM, BN, WAVES_M, WAVES_N>), dim3(static_cast<unsigned>(workgroups())), dim3(WAVES_M * WAVES_N * kWave), 0,
                       stream, problem());
  }
  template <bool A_NEXT, bool B_NEXT>
  void launch_as(hipStream_t stream) const
  {
    if (plain) {
      dim3 const grid = grid_of(plan.tiles(m, n) * plan.parts, kThreads);
      if (plan.tile == Tile::k128)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(product_kernel<T, A_NEXT, B_NEXT, 128>), grid, dim3(kThreads), 0, stream, problem());
      else
        hipLaunchKernelGGL(HIP_KERNEL_NAME(product_kernel<T, A_NEXT, B_NEXT, 64>), grid, dim3(kThreads), 0, stream, problem());
    } else if constexpr (sizeof(T) == 2) {
      if (plan.tile == Tile::k256)
        launch_as<A_NEXT, B_NEXT, 256, 256, 2, 4>(stream);
      else if (plan.tile == Tile::k128)
        launch_as<A_NEXT, B_NEXT, 128, 128, 2, 2>(stream);
      else if constexpr (A_NEXT && B_NEXT)
        launch_as<A_NEXT, B_NEXT, 128, 64, 2, 2>(stream);
    }
  }
  // what the timing record calls it
  const char* name() const
  {
    if (plain) return plan.tile == Tile::k128 ? "linear_product_128" : "linear_product_64";
    return plan.tile == Tile::k256 ? "linear_tiles_256" : plan.tile == Tile::k128 ? "linear_tiles_128" : "linear_tiles_64";
  }
  void launch(hipStream_t stream) const
  {
    ProfileScope const scope(name(), stream);
    if (a.k_next && b.k_next)
      launch_as<true, true>(stream);
    else if (a.k_next)
      launch_as<true, false>(stream);
    else
      launch_as<false, false>(stream);
  }
  Join<T> join() const { return join_of(sums, plan.parts, m, n, end); }
  int64_t join_blocks() const { return wanted() && sums ? join().blocks() : 0; }
};

template <typename T>
void launch_few_rows(Rows<const T> x, Rows<const T> weight, int64_t m, int64_t n, int64_t depth, Epilogue<T> const& end, hipStream_t stream)
{
  using std::integral_constant;
  ProfileScope const scope("linear_few_rows", stream);
  auto const launch = [&](auto rows_of_16, auto waves) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_kernel<T, decltype(rows_of_16)::value, decltype(waves)::value>), grid_of((n + 15) / 16, decltype(waves)::value * kWave),
                       dim3(decltype(waves)::value * kWave), 0, stream, x, weight, m, n, depth, end);
  };
  // enough wavefronts that each has about one round of loads  (more than 32 rows of 2048 values and more go through tiles)
  auto const by_depth = [&](auto rows_of_16, auto most) {
    if (depth >= 2048)
      launch(rows_of_16, most);
    else
      launch(rows_of_16, integral_constant<int, 4>{});
  };
  if (m <= 16)
    by_depth(integral_constant<int, 1>{}, integral_constant<int, 16>{});
  else if (m <= 32)
    by_depth(integral_constant<int, 2>{}, integral_constant<int, 8>{});
  else
    launch(integral_constant<int, 4>{}, integral_constant<int, 4>{});
}

template <typename T>
nvtext_amd_status linear(Rows<const T> x, Rows<const T> weight, int64_t m, int64_t n, int64_t depth, Epilogue<T> const& end, Mr const& mr, hipStream_t stream)
{
  Product<T> p{{x, true}, {weight, true}, m, n, depth, end};
  bool const few = few_rows_are_faster(m, n, depth, sizeof(T) == 4 || depth % 8 == 0);
  if (!few) {
    if (!p.fits()) return fail(NVTEXT_AMD_OVERFLOW, "the product is too large");
    p.make_plan();
  } else if (sizeof(T) == 2 && depth % 8 == 0 && 0.9 * few_rows_time(m, n, depth) > 5) {
    // rows of such a width that lie at odd places (views) are copied, where the copy takes less than reading them at half the rate
    auto const odd = [](Rows<const T> rows) { return reinterpret_cast<uintptr_t>(rows.data) % 16 != 0 || rows.stride % 8 != 0; };
    p.copy_a       = odd(x);
    p.copy_b       = odd(weight);
  }
  TempParts<3> const temp(mr, {p.bytes_a(), p.bytes_b(), p.bytes_sums()}, p.bytes_a() + p.bytes_b() + p.bytes_sums() > 0);
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  Align<T> a{}, b{};
  if (p.copy_a) a = p.align(p.a, m, depth, temp.template part<T>(0));
  if (p.copy_b) b = p.align(p.b, n, depth, temp.template part<T>(1));
  int64_t const first = blocks_of(a.rows * ((a.cols + 7) / 8)), second = blocks_of(b.rows * ((b.cols + 7) / 8));
  if (first + second > 0) {
    ProfileScope const scope("linear_prepare", stream);
    hipLaunchKernelGGL(prepare_kernel<T>, grid_of(first + second, kThreads), dim3(kThreads), 0, stream, a, first, b, second, Slopes<T>{}, 0);
  }
  if (few) {
    launch_few_rows(p.a.rows, p.b.rows, m, n, depth, end, stream);
    return NVTEXT_AMD_SUCCESS;
  }
  if (p.plan.parts > 1) p.sums = temp.template part<float>(2);
  p.launch(stream);
  if (p.sums) {
    ProfileScope const scope("linear_join", stream);
    hipLaunchKernelGGL(join_kernel<T>, grid_of(p.join_blocks(), kThreads), dim3(kThreads), 0, stream, p.join(), p.join_blocks(), Join<T>{}, 0, JoinColumns<T>{});
  }
  return NVTEXT_AMD_SUCCESS;
}

// The parts of the outputs that few_rows_backward_kernel takes the least time with, by this measure: so much for 64 outputs, twice
// as many workgroups at a time as there are CUs, and a launch that joins the parts.
inline int64_t few_rows_parts(int64_t m, int64_t n, int64_t depth, bool slopes)
{
  double const step = (slopes ? 1.6 : 1.2) * (m <= 32 ? 1 : m <= 64 ? 1.3 : 1.8);
  int64_t const blocks = (depth + kFewEdge - 1) / kFewEdge, steps = (n + kFewEdge - 1) / kFewEdge;
  int64_t best = 1;
  double least = 1e300;
  for (int64_t parts = 1; parts <= std::min<int64_t>(steps, 64); ++parts) {
    int64_t const each = (steps + parts - 1) / parts;
    if ((steps + each - 1) / each != parts) continue;
    double const time = step * static_cast<double>(each * ((blocks * parts + 2 * device_cus() - 1) / (2 * device_cus()))) + (parts > 1 ? 5 + parts * m * depth * 8e-6 / 5 : 0);
    if (time < least) {
      least = time;
      best  = parts;
    }
  }
  return best;
}

// Whether few_rows_backward_kernel takes less time than tiles.  (d is made once for every 64 inputs, which many weights make dear.  64 rows: 576 x 1064
// weights with gelu 11.7 us against 32.5, 4096 x 4096 47 against 52, 8192 x 8192 149 against 111; 96 rows: 15.5 against 22.8, 4096 x 4096 66 against 46, and
// 1024 x 1024, where the line is drawn, 17.2 against 17.9.)
inline bool few_rows_backward_is_faster(int64_t m, int64_t n, int64_t depth)
{
  if (m <= 64) return n * depth <= (int64_t{1} << 31) / m;
  return m <= 128 && n * depth < (1 << 20);
}

template <typename T>
nvtext_amd_status few_rows_backward(FewRowsBackward<T> w, Mr const& mr, hipStream_t stream)
{
  int64_t const steps = (w.n + kFewEdge - 1) / kFewEdge, parts = few_rows_parts(w.m, w.n, w.depth, static_cast<bool>(w.z));
  w.parts             = static_cast<int32_t>(parts);
  w.part              = (steps + parts - 1) / parts * kFewEdge;
  bool const join     = w.x_grad && parts > 1;
  Temp const sums(mr, join ? static_cast<size_t>(parts) * static_cast<size_t>(w.m * w.depth) * sizeof(float) : 0);
  if (!sums.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  if (join) w.sums = sums.template as<float>();
  dim3 const grid = grid_of((w.depth + kFewEdge - 1) / kFewEdge * parts, kThreads);
  {
    ProfileScope const scope("linear_few_rows_backward", stream);
    if (w.m <= 16)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_backward_kernel<T, 1>), grid, dim3(kThreads), 0, stream, w);
    else if (w.m <= 32)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_backward_kernel<T, 2>), grid, dim3(kThreads), 0, stream, w);
    else if (w.m <= 64)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_backward_kernel<T, 4>), grid, dim3(kThreads), 0, stream, w);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(few_rows_backward_kernel<T, 8>), grid, dim3(kThreads), 0, stream, w);
  }
  if (join) {
    ProfileScope const scope("linear_join_backward", stream);
    Join<T> const j = join_of(w.sums, parts, w.m, w.depth, Epilogue<T>{{nullptr, 0}, {nullptr, 0}, w.x_grad, {nullptr, 0}, NVTEXT_AMD_ACTIVATION_NONE});
    hipLaunchKernelGGL(join_kernel<T>, grid_of(j.blocks(), kThreads), dim3(kThreads), 0, stream, j, j.blocks(), Join<T>{}, 0, JoinColumns<T>{});
  }
  return NVTEXT_AMD_SUCCESS;
}

// The gradients that are wanted (of those of x and the weights, whose `out` has data).
template <typename T>
nvtext_amd_status linear_backward(Rows<const T> grad, Rows<const T> x, Rows<const T> weight, int64_t m, int64_t n, int64_t depth, int activation, Rows<const T> z, Rows<T> x_grad,
                                  Rows<T> weight_grad, T* bias_grad, Mr const& mr, hipStream_t stream)
{
  if constexpr (sizeof(T) == 2) {
    if (m > 0 && n > 0 && depth > 0 && few_rows_backward_is_faster(m, n, depth))
      return few_rows_backward(FewRowsBackward<T>{grad, activation != NVTEXT_AMD_ACTIVATION_NONE ? z : Rows<const T>{nullptr, 0}, x, weight, x_grad, weight_grad, bias_grad, activation, m, n, depth, 0,
                                                  0, nullptr},
                               mr, stream);
  }
  auto const plain = [](Rows<T> out) { return Epilogue<T>{{nullptr, 0}, {nullptr, 0}, out, {nullptr, 0}, NVTEXT_AMD_ACTIVATION_NONE}; };
  bool const slopes = activation != NVTEXT_AMD_ACTIVATION_NONE;
  // x_grad (m x depth) = d * weight, weight_grad (n x depth) = d^T * x
  Product<T> of_x{{grad, true}, {weight, false}, x_grad ? m : 0, depth, n, plain(x_grad)}, of_weight{{grad, false}, {x, false}, weight_grad ? n : 0, depth, m, plain(weight_grad)};
  if (!of_x.fits() || !of_weight.fits()) return fail(NVTEXT_AMD_OVERFLOW, "the product is too large");
  of_x.make_plan();
  of_weight.make_plan();
  // d is written where grad is not what the products can read
  bool const write_d     = m > 0 && n > 0 && (slopes || (of_x.wanted() && of_x.copy_a) || (of_weight.wanted() && of_weight.copy_a));
  int64_t const d_stride = copy_stride(n);
  int32_t const lanes    = Slopes<T>::lanes_of(n);
  int64_t const count    = Slopes<T>::count_of(m, lanes);
  bool const sums        = bias_grad && count > 1;
  TempParts<6> const temp(mr, {write_d ? static_cast<size_t>(m) * static_cast<size_t>(d_stride) * sizeof(T) : 0, sums ? static_cast<size_t>(count * n) * sizeof(float) : 0,
                               of_x.wanted() ? of_x.bytes_b() : 0, of_weight.wanted() ? of_weight.bytes_b() : 0, of_x.wanted() ? of_x.bytes_sums() : 0,
                               of_weight.wanted() ? of_weight.bytes_sums() : 0});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  Rows<T> const d = write_d ? Rows<T>{temp.template part<T>(0), d_stride} : Rows<T>{nullptr, 0};
  if (write_d) {
    of_x.a      = Factor<T>{{d.data, d.stride}, true, true};
    of_weight.a = Factor<T>{{d.data, d.stride}, false, true};
  }
  Align<T> a{}, b{};
  if (of_x.wanted() && of_x.copy_b) a = of_x.align(of_x.b, depth, n, temp.template part<T>(2));
  if (of_weight.wanted() && of_weight.copy_b) b = of_weight.align(of_weight.b, depth, m, temp.template part<T>(3));
  Slopes<T> const act{grad, slopes ? z : Rows<const T>{nullptr, 0}, activation, m, n, d, lanes, count, sums ? temp.template part<float>(1) : nullptr, sums ? nullptr : bias_grad};
  int64_t const first = blocks_of(a.rows * ((a.cols + 7) / 8)), second = blocks_of(b.rows * ((b.cols + 7) / 8));
  int64_t const third = write_d || bias_grad ? act.workgroups() : 0;
  bool both = false;  // in one launch
  if constexpr (sizeof(T) == 2) both = of_x.wanted() && of_weight.wanted() && !of_x.plain && !of_weight.plain && of_x.plan.tile == Tile::k128 && of_weight.plan.tile == Tile::k128;
  bool const sums_beside = both && !write_d && first + second == 0 && third < (1 << 20);  // (one dimension of the launch)
  if (first + second + third > 0 && !sums_beside) {
    ProfileScope const scope("linear_prepare_backward", stream);
    hipLaunchKernelGGL(prepare_kernel<T>, grid_of(first + second + third, kThreads), dim3(kThreads), 0, stream, a, first, b, second, act, third);
  }
  if (of_x.bytes_sums()) of_x.sums = temp.template part<float>(4);
  if (of_weight.bytes_sums()) of_weight.sums = temp.template part<float>(5);
  if constexpr (sizeof(T) == 2) {
    if (both) {
      ProfileScope const scope("linear_products_backward", stream);
      int64_t const used = of_x.workgroups(), from = (used + 7) / 8 * 8, last = from + of_weight.workgroups();  // (workgroups go to the eight XCDs in turn)
      hipLaunchKernelGGL(gradient_products_kernel<T>, dim3(static_cast<unsigned>(last + (sums_beside ? third : 0))), dim3(kThreads), 0, stream, of_x.problem(), of_weight.problem(),
                         static_cast<int32_t>(from), static_cast<int32_t>(used), static_cast<int32_t>(last), act);
    }
  }
  if (of_x.wanted() && !both) of_x.launch(stream);
  if (of_weight.wanted() && !both) of_weight.launch(stream);
  int64_t const join_x = of_x.join_blocks(), join_weight = of_weight.join_blocks(), join_columns = sums ? (n + kWave - 1) / kWave : 0;
  if (join_x + join_weight + join_columns > 0) {
    ProfileScope const scope("linear_join_backward", stream);
    hipLaunchKernelGGL(join_kernel<T>, grid_of(join_x + join_weight + join_columns, kThreads), dim3(kThreads), 0, stream, of_x.join(), join_x, of_weight.join(), join_weight,
                       JoinColumns<T>{act.parts, count, n, bias_grad});
  }
  return NVTEXT_AMD_SUCCESS;
}

bool is_activation(int32_t a) { return a >= NVTEXT_AMD_ACTIVATION_NONE && a <= NVTEXT_AMD_ACTIVATION_SILU; }

// What the shapes of linear's matrices have in common with those of its gradients; nullptr if it holds.
const char* bad_shapes(const nvtext_amd_matrix* x, const nvtext_amd_matrix* weight)
{
  if (weight->cols != x->cols) return "x and weight must have the same number of inputs";
  if (weight->rows > INT32_MAX) return "invalid matrix sizes";
  return nullptr;
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_linear(const nvtext_amd_matrix* x, const nvtext_amd_matrix* weight, const nvtext_amd_matrix* bias, int32_t activation,
                                    const nvtext_amd_matrix* residual, void* stream_, const nvtext_amd_allocator* mr_, const nvtext_amd_matrix* out,
                                    const nvtext_amd_matrix* preactivation)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_linear");
  if (!x || !weight || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  for (auto* m : {x, weight, bias, residual, out, preactivation}) {
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (m && m->type != x->type) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "all matrices must be of one type");
  }
  if (const char* bad = bad_shapes(x, weight)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  int64_t const m = x->rows, n = weight->rows, depth = x->cols;
  if (bias && !is_shape(bias, 1, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "bias must be a vector of a value for each output");
  for (auto* o : {residual, out, preactivation})
    if (o && !is_shape(o, m, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out, residual and preactivation must have x's rows and weight's outputs");
  if (!is_activation(activation)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "unknown activation");
  if (m == 0 || n == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  with_type(x->type, [&](auto zero) {
    using T = decltype(zero);
    st      = linear<T>(rows_of<const T>(x), rows_of<const T>(weight), m, n, depth, {rows_of<const T>(bias), rows_of<const T>(residual), rows_of<T>(out), rows_of<T>(preactivation), activation},
                        mr, stream);
  });
  if (st != NVTEXT_AMD_SUCCESS) return st;
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

nvtext_amd_status nvtext_amd_linear_backward(const nvtext_amd_matrix* grad, const nvtext_amd_matrix* x, const nvtext_amd_matrix* weight, int32_t activation,
                                             const nvtext_amd_matrix* preactivation, void* stream_, const nvtext_amd_allocator* mr_,
                                             const nvtext_amd_matrix* x_grad, const nvtext_amd_matrix* weight_grad, const nvtext_amd_matrix* bias_grad)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_linear_backward");
  if (!grad || !x || !weight) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  for (auto* m : {grad, x, weight, preactivation, x_grad, weight_grad, bias_grad}) {
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (m && m->type != x->type) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "all matrices must be of one type");
  }
  if (const char* bad = bad_shapes(x, weight)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  int64_t const m = x->rows, n = weight->rows, depth = x->cols;
  for (auto* o : {grad, preactivation})
    if (o && !is_shape(o, m, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "grad and preactivation must have x's rows and weight's outputs");
  if (x_grad && !is_shape(x_grad, m, depth)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "x_grad must be of x's size");
  if (weight_grad && !is_shape(weight_grad, n, depth)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "weight_grad must be of weight's size");
  if (bias_grad && !is_shape(bias_grad, 1, n)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "bias_grad must be a vector of a value for each output");
  if (!is_activation(activation)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "unknown activation");
  if (activation != NVTEXT_AMD_ACTIVATION_NONE && !preactivation) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the gradient of an activation needs what it was applied to");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  with_type(x->type, [&](auto zero) {
    using T = decltype(zero);
    st      = linear_backward<T>(rows_of<const T>(grad), rows_of<const T>(x), rows_of<const T>(weight), m, n, depth, activation, rows_of<const T>(preactivation), rows_of<T>(x_grad),
                            rows_of<T>(weight_grad), bias_grad ? static_cast<T*>(bias_grad->data) : nullptr, mr, stream);
  });
  if (st != NVTEXT_AMD_SUCCESS) return st;
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
