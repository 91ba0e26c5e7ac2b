// The gradient of attention.
#include "attention.cuh"

namespace nvtext_amd {
namespace {

// Two launches, the first for q, the second (of wide heads, a second and a third) for k and v: each makes the scores anew and adds up what is its own in registers, in one order at every
// call.  (One launch for all three would have to add up q's gradient in memory, over all workgroups of keys: in parts of float32 or in any order.)
//
// Blocks of 32 rows of a tile that go through one stream of fragments.  Of heads of 128, two, which spares the wait for the first fragments of the second (16384 tokens in four rows: 3.56 -> 3.12 ms
// with the forward pass).  Of narrower ones, whose rows are often short, one, so that none is gone through that has no row (131071 in 1024, heads of 64: 1.12 ms either way; 32768 in 64, of 96:
// 660 us, with two 650); of wider ones one, whose registers are few as it is (8192 in eight rows, 16 heads of 192 in bfloat16 720 us, with two 748, in float16 794 and 766, of 256 907 and 940).
template <typename T, int D>
constexpr int kBlocksAtOnce = sizeof(T) == 2 && D == 128 ? 2 : 1;
// Two rows' values and a sum of 1024 bytes are more than a lane's registers hold with the rest: one of the rows is read again, two products ahead, for every block
// of 32, whose 384 products take longer than that (1135 tokens, 12 heads of 216 values in float32: that of q 307 -> 288 us, of k 253 -> 213).  Some stay in memory all the same: 39 registers
// of q's with four wavefronts, 87 with one; with one, of k's about as many.
template <typename T, int D>
constexpr bool kReadAgain = D * sizeof(T) > 768;

// Which rows a wavefront has alone (in float32, where the products take longest, rows of 128 tokens, 8 heads of 64: 1350 us with four wavefronts, 1150 with one).
template <typename T>
constexpr int32_t kShort = sizeof(T) == 4 ? 2 * kShortRow : kShortRow;

// What is rounded to float16 before it is multiplied is brought into its range first.  d = p (grad . v - grad . out) lies anywhere: with gradients of 1e-3, a row of 4096 tokens
// has d of 1e-6, where float16 has steps of 6e-8 (q's gradient was off by 0.53 %, of 1e-4 over 8192 tokens by 10 %; with its bits it is by 0.07 and 0.93, its own rounding), and of a
// loss that has been scaled up it may pass 65504.  So a column multiplies its d by a power of 2 of its own and its sums by the reciprocal at the end.  Its largest d so far lies between
// 2^8 and 2^15 (or below, while the power is the first one), and only a larger one changes the power, and with it what has been added up: what is 2^-22 of
// it and more keeps all its bits, and the rest is off by 2^-33 of it.  bfloat16 has the exponents of float32.  (Steps take 3 to 4 % longer for it: 131071 tokens in 1024 rows, 12 heads
// of 64, 1121 -> 1165 us; 8192 in eight rows, 16 heads of 192, 720 -> 795, of 256 920 -> 968.)
template <typename T>
constexpr bool kLifted = std::is_same_v<T, half_t>;
// And so are the probabilities that the gradient of v adds up, in which a key of little weight has 2^-20 (where one of 2000 keys has nearly all, the others' gradients were off by 1.9 %, and are by 0.03): they
// are 1 at most, and go through the products 2^15 times as large.
template <typename T>
constexpr float kWeightLift = kLifted<T> ? 15.f : 0.f;
struct Lift {
  static constexpr float kMost = 0x1p15f;
  float up = 0x1p60f;  // (d of inputs in float16 is below 2^41, of such probabilities 2^56)
  // d of 32 rows, of which this lane has 16, times the power; where that changes, what has been added up as well
  template <int COLUMNS>
  __device__ __forceinline__ void apply(f32x16_t& d, f32x16_t (&sums)[COLUMNS])
  {
    float high = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      d[r] *= up;
      high = fmaxf(high, fabsf(d[r]));
    }
    Halves const both = halves(high);
    high              = fmaxf(both.low, both.high);
    if (__ballot(high > kMost)) {
      float const by = high > kMost ? __builtin_amdgcn_ldexpf(1.f, 9 - __builtin_amdgcn_frexp_expf(high)) : 1.f;
      up *= by;
      d *= by;
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c) sums[c] *= by;
    }
  }
};

// Wide heads in float16 go through tiles of one block of 32 rows: with a second loop, over a tile's blocks, around the place where the sums may change their power, the compiler keeps
// 61 to 111 registers of them in memory.
template <typename T, int D, int WAVES>
constexpr int kTileOfGradient = kLifted<T> && D > 192 ? 32 : kTileOf<T, D, WAVES>;

template <typename T, int D, int WAVES>
struct GradientShape {
  static constexpr int kRows = 32 * WAVES, kShift = __builtin_ctz(kRows), kTile = kTileOfGradient<T, D, WAVES>, kBytes = Tile<T, D, kTile>::kBytes, kStage = 2 * kBytes, kLds = 2 * kStage;
  static constexpr int kWavesASimd = D * sizeof(T) <= 256 ? 2 : 1;
};

// The gradient of q: as forward, a lane has a token's scores, and what they are multiplied with comes from LDS, keys as they lie and transposed.
// Bound as the forward pass is (16384 tokens in four rows, 32 heads of 128 over 8, causal, bfloat16: 0.85 ms, 0.97 PFLOP/s, matrix cores busy for 57 % of the time; 131071
// tokens in 1024 rows, 12 heads of 64: 0.40 ms, 14 %).
template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave, (GradientShape<T, D, WAVES>::kWavesASimd)) query_gradient_tiles_kernel(Backward<T> f, Split split)
{
  using Shape = GradientShape<T, D, WAVES>;
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds = (LdsBytes)lds_;
  constexpr int kSteps = D / 16, kColumns = D / 32, kTile = Shape::kTile, kAtOnce = kTile == 32 ? 1 : kBlocksAtOnce<T, D>;
  Work w;
  int32_t const each = f.heads / f.kv_heads;
  if (!work_of(block_number(), f.runs.blocks(Shape::kShift), f.kv_heads, each, split.splits, w)) return;
  int32_t const run    = f.runs.run_of(w.block, Shape::kShift);
  int32_t const begin  = uniform(f.runs.begin(run)), tokens = uniform(f.runs.begin(run + 1)) - begin;
  int64_t const in_run = (w.block - f.runs.first_block(run, Shape::kShift)) << Shape::kShift;
  if (in_run >= tokens) return;
  int const wave = uniform(threadIdx.x / kWave), lane = lane_id(), column = lane % 32, half = lane / 32;
  int32_t const block0 = static_cast<int32_t>(in_run), rest = uniform(tokens - block0);
  int32_t first = 0, keys = 0;
  if (f.is_row(run)) f.keys_of(run, first, keys);
  first = uniform(first);
  keys  = uniform(keys);
  int32_t const wave0 = wave * 32, wave1 = wave0 + 32 < rest ? wave0 + 32 : rest;
  int32_t const all   = uniform(f.seen(block0 + (rest < Shape::kRows ? rest : Shape::kRows) - 1, tokens, keys));
  int32_t const least = uniform(wave0 < rest ? f.seen(block0 + wave0, tokens, keys) : 0), most = uniform(wave0 < rest ? f.seen(block0 + wave1 - 1, tokens, keys) : 0);
  int32_t const all_tiles = (all + kTile - 1) / kTile, shares = shares_of(all_tiles, split.splits);
  if (w.share >= shares) return;
  int32_t const first_tile = uniform(share_begin(all_tiles, w.share, shares)), tiles = uniform(share_begin(all_tiles, w.share + 1, shares));
  bool const there    = wave0 + column < rest;
  int64_t const t     = static_cast<int64_t>(begin) + block0 + (there ? wave0 + column : 0);
  int32_t const seen  = there ? f.seen(block0 + wave0 + column, tokens, keys) : 0;

  TileLoader<T, D, WAVES, kTile> load_k, load_v;
  load_k.aim(f.k, first + first_tile * kTile, w.kv_head, f.width, wave, lane);
  load_v.aim(f.v, first + first_tile * kTile, w.kv_head, f.width, wave, lane);
  auto const load = [&](int32_t tile) {
    LdsBytes const to = lds + (tile & 1) * Shape::kStage;
    load_k.load(to, keys - tile * kTile, wave);
    load_v.load(to + Shape::kBytes, keys - tile * kTile, wave);
  };
  if (tiles > first_tile) load(first_tile);
  int64_t const at = static_cast<int64_t>(w.head) * f.runs.tokens + t;
  constexpr bool kAgain = kReadAgain<T, D>;
  Fragment<T> q[kSteps], g[kAgain ? 3 : kSteps];
  const T* const grad = f.grad.at(t, w.head);
  float delta         = 0.f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    q[s]                  = fragment_of(f.q.at(t, w.head), 16 * s + 8 * half, f.width, there);
    Fragment<T> const of  = fragment_of(grad, 16 * s + 8 * half, f.width, there);
    if constexpr (!kAgain) g[s] = of;
    Fragment<T> const out = fragment_of(f.out.at(t, w.head), 16 * s + 8 * half, f.width, there);
    bool rests = false;
    if constexpr (sizeof(T) == 2) rests = f.rest != nullptr;
    if (rests) {
      auto const rest = load_raw8(f.rest + at * f.width + 16 * s + 8 * half, there ? f.width - 16 * s - 8 * half : 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) delta = fmaf(static_cast<float>(of[k]), with_rest(out[k], rest[k]), delta);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) delta = fmaf(static_cast<float>(of[k]), static_cast<float>(out[k]), delta);
    }
  }
  Halves const both = halves(delta);
  delta             = seen > 0 ? both.low + both.high : 0.f;
  float const log   = there ? f.logsum[at] * kLog2e : 0.f;
  if (there && half == 0 && w.share == 0) {
    f.deltas[at] = delta;
    f.logs[at]   = log - kWeightLift<T>;
  }
  Lift lift;
  f32x16_t d[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) d[c] = f32x16_t{};
  TileReader<T, D> const read(lane);
  float const scale = f.scale * kLog2e;
  for (int32_t tile = first_tile; tile < tiles; ++tile) {
    LdsBytes const k_tile = lds + (tile & 1) * Shape::kStage;
    stage_barrier<0>();
    if (tile + 1 < tiles) load(tile + 1);
    int32_t const key0 = tile * kTile;
    // Of each block of 32 keys, scores and products of g and v, then what they come to, multiplied with the keys.
    constexpr int kFirst = 2 * kSteps, kOfBlock = kFirst + 2 * kColumns;
    f32x16_t s, p;
    Fragment<T> ds[2];
#pragma unroll 1
    for (int32_t from = key0; from < key0 + kTile && from < most; from += 32 * kAtOnce) {
      LdsBytes const k_block = k_tile + (from - key0) * Tile<T, D>::kLine, v_block = k_block + Shape::kBytes;
      stream<T, D, kAtOnce * kOfBlock>(
        [&](auto slot) {
          constexpr int b = slot / kOfBlock, i = slot % kOfBlock;
          if constexpr (i < kSteps) return read.rows(k_block, b, i);
          else if constexpr (i < kFirst) return read.rows(v_block, b, i - kSteps);
          else return read.columns(k_block, (i - kFirst) % kColumns, 2 * b + (i - kFirst) / kColumns);
        },
        [&](auto slot, Fragment<T> const& x) {
          constexpr int b = slot / kOfBlock, i = slot % kOfBlock, ahead = i + 2 - kSteps;
          int32_t const key = from + 32 * b;
          if constexpr (kAgain && ahead >= 0 && ahead < kSteps) g[ahead % 3] = fragment_of(grad, 16 * ahead + 8 * half, f.width, there);
          if constexpr (i < kSteps) {
            if constexpr (i == 0) s = f32x16_t{};
            s = multiply32(x, q[i], s);
          } else if constexpr (i < kFirst) {
            if constexpr (i == kSteps) p = f32x16_t{};
            p = multiply32(x, g[kAgain ? (i - kSteps) % 3 : i - kSteps], p);
          } else {
            if constexpr (i == kFirst) {
#pragma unroll
              for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], scale, -log)) * (p[r] - delta);
              if (key + 32 > least) {
                int32_t const left = seen - key - 4 * half;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + r % 4 < left ? s[r] : 0.f;
              }
              if constexpr (kLifted<T>) lift.apply(s, d);
              ds[0] = rounded<T>(s, 0);
              ds[1] = rounded<T>(s, 1);
            }
            d[(i - kFirst) % kColumns] = multiply32(x, ds[(i - kFirst) / kColumns], d[(i - kFirst) % kColumns]);
          }
        });
    }
  }
  if (wave0 >= rest) return;
  if constexpr (kLifted<T>) {
    float const down = 1.f / lift.up;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) d[c] *= down;
  }
  if (shares > 1) {
    if (there) store_columns<float, kColumns>(split.sums + (split.slot(w.block, w.head, f.heads, w.share) * Shape::kRows + wave0 + column) * D, d, half, D);
    return;
  }
  float check = 0.f;
#pragma unroll
  for (int c = 0; c < kColumns; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      d[c][r] = seen > 0 ? d[c][r] * f.scale : 0.f;
      check   = fmaf(d[c][r], 0.f, check);
    }
  // (as forward: a key that is not seen may have been multiplied by 0; NaN in the log or in delta makes NaN of all)
  uint64_t odd = f.causal ? __ballot(there && check != 0.f && log == log && delta == delta) : 0;
  if (odd != 0) {
    int32_t const loaded = (most + kTile - 1) / kTile * kTile;
    if (!holds_odd(f.k, static_cast<int64_t>(first) + least, (loaded < keys ? loaded : keys) - least, w.kv_head, f.width)) odd = 0;
  }
  odd = (odd | odd >> 32) & 0xffffffffu;
  if (there && !(odd >> column & 1)) store_columns<T, kColumns>(f.q_grad.at(t, w.head), d, half, f.width);
  for (; odd; odd &= odd - 1) query_gradient_row(f, begin + block0 + wave0 + __builtin_ctzll(odd), w.head);
}

// The gradients of k and v: a wavefront has 32 keys in its registers, a lane a key's scores, and the tokens of all heads that see them come through LDS
// with their gradients, 64 at a time, with their logs and deltas.  (The same rows as above: 1.0 ms for k and 0.73 for v, matrix cores 45 %; 0.50 ms, 18 %.  All
// heads that share keys go through one wavefront: each key's gradient is added up in one place.)
template <typename T, int D, int WAVES>
struct KeyShape {
  static constexpr int kRows = 32 * WAVES, kShift = __builtin_ctz(kRows), kTile = kTileOfGradient<T, D, WAVES>, kBytes = Tile<T, D, kTile>::kBytes, kTiles = 2 * kBytes;
  static constexpr int kStage = kTiles + 2 * kWave * 4, kLds = 2 * kStage;  // (with logs and deltas)
  static constexpr int kWavesASimd = sizeof(T) == 2 && D <= 128 ? 2 : 1;
};
// Whether one of `count` tokens from `first` on holds an infinity or NaN in what the gradients of k and v, those that are wanted, add up.
template <typename T>
__device__ __forceinline__ bool tokens_hold_odd(Backward<T> const& f, int32_t first, int32_t count, int32_t kv_head, bool of_k, bool of_v)
{
  int32_t const each = f.heads / f.kv_heads;
#pragma unroll 1
  for (int32_t h = kv_head * each; h < (kv_head + 1) * each; ++h)
    if ((of_k && holds_odd(f.q, first, count, h, f.width)) || (of_v && holds_odd(f.grad, first, count, h, f.width))) return true;
  return false;
}
// PART: the gradients of both, or of k or v alone: of heads of more than 96 values there are not the registers for both, and what the compiler keeps in memory instead
// waits for the loads of the next tile at every use.
enum Part { kBoth, kOfK, kOfV };
template <typename T, int D, int WAVES, Part PART>
__global__ void __launch_bounds__(WAVES * kWave, (KeyShape<T, D, WAVES>::kWavesASimd)) key_gradient_tiles_kernel(Backward<T> f, Split split)
{
  using Shape = KeyShape<T, D, WAVES>;
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds = (LdsBytes)lds_;
  constexpr bool kK = PART != kOfV, kV = PART != kOfK;
  constexpr int kSteps = D / 16, kColumns = D / 32, kTile = Shape::kTile, kAtOnce = kTile == 32 ? 1 : kBlocksAtOnce<T, D>;
  Work w;
  if (!work_of(block_number(), f.key_runs.blocks(Shape::kShift), f.kv_heads, 1, split.splits, w)) return;
  w.block              = f.key_runs.blocks(Shape::kShift) - 1 - w.block;  // (of a long row, the first keys are those that most tokens see)
  int32_t const run    = f.key_runs.run_of(w.block, Shape::kShift), each = f.heads / f.kv_heads;
  int32_t const first  = uniform(f.key_runs.begin(run)), places = uniform(f.key_runs.begin(run + 1)) - first;
  int64_t const in_run = (w.block - f.key_runs.first_block(run, Shape::kShift)) << Shape::kShift;
  if (in_run >= places) return;
  int const wave = uniform(threadIdx.x / kWave), lane = lane_id(), column = lane % 32, half = lane / 32;
  int32_t const block0 = static_cast<int32_t>(in_run), rest = uniform(places - block0);  // (places: with those behind the row's keys, whose gradients are zeros)
  int32_t begin = 0, tokens = 0, keys = 0, ignored = 0;
  if (f.is_row(run)) {
    f.keys_of(run, ignored, keys);
    begin  = f.runs.begin(run);
    tokens = f.runs.begin(run + 1) - begin;
  }
  begin  = uniform(begin);
  tokens = uniform(tokens > 0 ? tokens : 0);
  keys   = uniform(keys);
  int32_t const wave0 = wave * 32, key = block0 + wave0 + column;
  bool const there    = wave0 + column < rest;
  int64_t const t     = static_cast<int64_t>(first) + (there ? key : block0);
  // the first token that sees a key, of the row's
  auto const from_of = [&](int32_t j) {
    int64_t const i = f.causal ? static_cast<int64_t>(j) + tokens - keys : 0;
    return static_cast<int32_t>(i < 0 ? 0 : i < tokens ? i : tokens);
  };
  int32_t const start = uniform(block0 < keys ? from_of(block0) / kTile : 0), tiles = uniform(block0 < keys ? (tokens + kTile - 1) / kTile : 0);
  // The tiles of one head after another are one stream of loads, of which this is a share.
  int32_t const of_head = tiles - start > 0 ? tiles - start : 0, total = of_head * each, shares = shares_of(total, split.splits);
  if (w.share >= shares) return;
  int32_t const begin_tile = uniform(share_begin(total, w.share, shares)), end_tile = uniform(share_begin(total, w.share + 1, shares));
  int32_t const last_from = uniform(from_of(block0 + wave0 + 31)), first_from = uniform(from_of(block0 + wave0));

  constexpr bool kAgain = kReadAgain<T, D>;
  Fragment<T> k[kSteps], v[kAgain ? 3 : kK ? kSteps : 1];
  const T* const values = f.v.at(t, w.kv_head);
  int32_t const from = from_of(key);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    k[s] = fragment_of(f.k.at(t, w.kv_head), 16 * s + 8 * half, f.width, there && key < keys);
    if constexpr (kK && !kAgain) v[s] = fragment_of(values, 16 * s + 8 * half, f.width, there && key < keys);
  }
  TileReader<T, D> const read(lane);
  float const scale = f.scale * kLog2e;
  f32x16_t dk[kK ? kColumns : 1], dv[kV ? kColumns : 1];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    if constexpr (kK) dk[c] = f32x16_t{};
    if constexpr (kV) dv[c] = f32x16_t{};
  }
  Lift lift;
  TileLoader<T, D, WAVES, kTile> load_q, load_g;
  int32_t loaded = uniform(of_head > 0 ? begin_tile % of_head : 0), next_head = uniform(w.kv_head * each + (of_head > 0 ? begin_tile / of_head : 0));  // the tile of the head that is loaded next
  bool aimed = false;
  auto const load = [&](LdsBytes to) {
    if (loaded == 0 || !aimed) {
      load_q.aim(f.q, begin + (start + loaded) * kTile, next_head, f.width, wave, lane);
      load_g.aim(f.grad, begin + (start + loaded) * kTile, next_head, f.width, wave, lane);
      aimed = true;
    }
    int32_t const token = (start + loaded) * kTile, here = tokens - token;
    load_q.load(to, here, wave);
    load_g.load(to + Shape::kBytes, here, wave);
    int64_t const at = static_cast<int64_t>(next_head) * f.runs.tokens + begin + token;
    uint32_t const range = uniform(static_cast<uint32_t>(here < kTile ? here : kTile) * 4);
    if (wave == 0) load_words_to_lds(uniform(reinterpret_cast<const char*>(f.logs + at)), range, to + Shape::kTiles, lane * 4);
    if (wave == WAVES - 1) load_words_to_lds(uniform(reinterpret_cast<const char*>(f.deltas + at)), range, to + Shape::kTiles + kWave * 4, lane * 4);
    if (++loaded == of_head) {
      loaded = 0;
      ++next_head;
    }
  };
  int32_t tile = start + loaded - 1;
  if (end_tile > begin_tile) load(lds + (begin_tile & 1) * Shape::kStage);
  for (int32_t n = begin_tile; n < end_tile; ++n) {
    LdsBytes const q_tile = lds + (n & 1) * Shape::kStage;
    stage_barrier<0>();
    if (n + 1 < end_tile) load(lds + (~n & 1) * Shape::kStage);
    if (++tile == tiles) tile = start;
    int32_t const token0 = tile * kTile;
    constexpr int kFirst = (kK ? 2 : 1) * kSteps, kOfStep = (kK && kV ? 2 : 1) * kColumns, kOfBlock = kFirst + 2 * kOfStep;
    f32x16_t s, p;
    Fragment<T> weight[2], ds[2];
#pragma unroll 1
    for (int32_t block = token0; block < token0 + kTile && block < tokens; block += 32 * kAtOnce) {
      if (block + 32 * kAtOnce <= first_from) continue;
      LdsBytes const q_block = q_tile + (block - token0) * Tile<T, D>::kLine, g_block = q_block + Shape::kBytes, words = q_tile + Shape::kTiles + 16 * half + (block - token0) * 4;
      stream<T, D, kAtOnce * kOfBlock>(
        [&](auto slot) {
          constexpr int b = slot / kOfBlock, i = slot % kOfBlock;
          if constexpr (i < kSteps) return read.rows(q_block, b, i);
          else if constexpr (i < kFirst) return read.rows(g_block, b, i - kSteps);
          else {
            constexpr int j = i - kFirst, step = 2 * b + j / kOfStep, c = j % kOfStep;
            if constexpr (kV && c < kColumns) return read.columns(g_block, c, step);
            else return read.columns(q_block, c % kColumns, step);
          }
        },
        [&](auto slot, Fragment<T> const& x) {
          constexpr int b = slot / kOfBlock, i = slot % kOfBlock, ahead = i + 2 - kSteps;
          int32_t const row0 = block + 32 * b;
          if constexpr (kK && kAgain && ahead >= 0 && ahead < kSteps) v[ahead % 3] = fragment_of(values, 16 * ahead + 8 * half, f.width, there && key < keys);
          if constexpr (i < kSteps) {
            if constexpr (i == 0) s = f32x16_t{};
            s = multiply32(x, k[i], s);
          } else if constexpr (i < kFirst) {
            if constexpr (i == kSteps) p = f32x16_t{};
            p = multiply32(x, v[kAgain ? (i - kSteps) % 3 : i - kSteps], p);
          } else {
            if constexpr (i == kFirst) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                f32x4_t const log = *reinterpret_cast<__attribute__((address_space(3))) f32x4_t*>(words + 128 * b + 32 * j);
                f32x4_t delta{};
                if constexpr (kK) delta = *reinterpret_cast<__attribute__((address_space(3))) f32x4_t*>(words + kWave * 4 + 128 * b + 32 * j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  int const r = 4 * j + e;
                  s[r]        = __builtin_amdgcn_exp2f(fmaf(s[r], scale, -log[e]));
                  if constexpr (kK) p[r] = s[r] * (p[r] - delta[e]);
                }
              }
              if (row0 < last_from || row0 + 32 > tokens) {
                int32_t const before = from - row0 - 4 * half, behind = tokens - row0 - 4 * half;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  bool const sees = 8 * (r / 4) + r % 4 >= before && 8 * (r / 4) + r % 4 < behind;
                  if constexpr (kV) s[r] = sees ? s[r] : 0.f;
                  if constexpr (kK) p[r] = sees ? p[r] : 0.f;
                }
              }
              if constexpr (kK && kLifted<T>) lift.apply(p, dk);
#pragma unroll
              for (int step = 0; step < 2; ++step) {
                if constexpr (kV) weight[step] = rounded<T>(s, step);
                if constexpr (kK) ds[step] = rounded<T>(p, step);
              }
            }
            constexpr int j = i - kFirst, step = j / kOfStep, c = j % kOfStep;
            if constexpr (kV && c < kColumns) dv[c] = multiply32(x, weight[step], dv[c]);
            else dk[c % kColumns] = multiply32(x, ds[step], dk[c % kColumns]);
          }
        });
    }
  }
  if constexpr (kLifted<T>) {
    constexpr float kDown = 1.f / (1 << static_cast<int>(kWeightLift<T>));
    float const down      = kDown / lift.up;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) {
      if constexpr (kK) dk[c] *= down;  // (whose d are made of the same probabilities)
      if constexpr (kV) dv[c] *= kDown;
    }
  }
  if (shares > 1) {
    if (!there) return;
    float* const part = split.sums + (split.slot(w.block, w.kv_head, f.kv_heads, w.share) * Shape::kRows + wave0 + column) * (2 * D);
    if constexpr (kK) store_columns<float, kColumns>(part, dk, half, D);
    if constexpr (kV) store_columns<float, kColumns>(part + D, dv, half, D);
    if (key >= keys && w.share == 0) {  // (which is no key: nothing is joined for it)
      f32x16_t const zeros[kColumns] = {};
      if constexpr (kK) store_columns<T, kColumns>(f.k_grad.at(t, w.kv_head), zeros, half, f.width);
      if constexpr (kV) store_columns<T, kColumns>(f.v_grad.at(t, w.kv_head), zeros, half, f.width);
    }
    return;
  }
  float check = 0.f;
#pragma unroll
  for (int c = 0; c < kColumns; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (kK) {
        dk[c][r] = key < keys ? dk[c][r] * f.scale : 0.f;
        check    = fmaf(dk[c][r], 0.f, check);
      }
      if constexpr (kV) {
        dv[c][r] = key < keys ? dv[c][r] : 0.f;
        check    = fmaf(dv[c][r], 0.f, check);
      }
    }
  uint64_t odd = f.causal ? __ballot(there && check != 0.f) : 0;
  if (odd != 0) {
    // (tokens that went through the products, up to the first that sees all of the keys)
    int32_t const border = first_from / (32 * kAtOnce) * (32 * kAtOnce), count = (last_from < tokens ? last_from : tokens) - border;
    if (!tokens_hold_odd(f, begin + border, count, w.kv_head, kK, kV) || is_odd_anyway(f, begin, last_from, tokens, w.kv_head, kK, kV)) odd = 0;
  }
  odd = (odd | odd >> 32) & 0xffffffffu;
  if (there && !(odd >> column & 1)) {
    if constexpr (kK) store_columns<T, kColumns>(f.k_grad.at(t, w.kv_head), dk, half, f.width);
    if constexpr (kV) store_columns<T, kColumns>(f.v_grad.at(t, w.kv_head), dv, half, f.width);
  }
  for (; odd; odd &= odd - 1) key_gradient_row(f, first + block0 + wave0 + __builtin_ctzll(odd), w.kv_head, kK, kV);
}

// Adds up the shares of a head of a token (of q) or a key, a wavefront for each; the numbers of shares are those that the kernels before found.
template <int D>
__device__ __forceinline__ Some<D> add_shares(const float* at, int64_t step, int32_t shares, float scale)
{
  Some<D> sum;
#pragma unroll 8
  for (int32_t c = 0; c < shares; ++c) sum.add(at + c * step, scale);
  return sum;
}

// Writes a row of a gradient.
template <typename T, int D>
__device__ __forceinline__ void write_row(T* head, Some<D> const& sum, int32_t width)
{
#pragma unroll
  for (int k = 0; k < Some<D>::kEach; ++k)
    if (sum.first() + k < width) head[sum.first() + k] = static_cast<T>(sum.v[k]);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) query_gradient_join_kernel(Backward<T> f, Split split, int shift)
{
  constexpr int kTile = kTileOfGradient<T, D, kTileWaves>;
  int64_t const item  = block_number() * (kThreads / kWave) + threadIdx.x / kWave;
  if (item >= static_cast<int64_t>(f.runs.tokens) * f.heads) return;
  int32_t const t = static_cast<int32_t>(item / f.heads), head = static_cast<int32_t>(item % f.heads), run = run_with(f.runs, t);
  if (!f.is_row(run)) return;
  int32_t first, keys;
  f.keys_of(run, first, keys);
  int32_t const begin = f.runs.begin(run), tokens = f.runs.begin(run + 1) - begin, i = t - begin, last = i | ((1 << shift) - 1);
  int32_t const all = f.seen(last < tokens ? last : tokens - 1, tokens, keys), shares = shares_of((all + kTile - 1) / kTile, split.splits);
  if (shares < 2) return;
  int64_t const at = (split.slot(f.runs.first_block(run, shift) + (i >> shift), head, f.heads, 0) << shift) + (i & ((1 << shift) - 1));
  int32_t const seen = f.seen(i, tokens, keys), loaded = (all + kTile - 1) / kTile * kTile;
  // (a token that sees nothing may have 0 times what others see among its sums)
  Some<D> sum{};
  if (seen > 0) sum = add_shares<D>(split.sums + at * D, static_cast<int64_t>(D) << shift, shares, f.scale);
  int64_t const row = static_cast<int64_t>(head) * f.runs.tokens + t;
  if (f.causal && !sum.finite(f.width) && f.logs[row] == f.logs[row] && f.deltas[row] == f.deltas[row] &&
      holds_odd(f.k, static_cast<int64_t>(first) + seen, (loaded < keys ? loaded : keys) - seen, head / (f.heads / f.kv_heads), f.width))
    query_gradient_row(f, t, head);
  else
    write_row<T, D>(f.q_grad.at(t, head), sum, f.width);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) key_gradient_join_kernel(Backward<T> f, Split split, int shift)
{
  constexpr int kTile = kTileOfGradient<T, D, kTileWaves>;
  int64_t const item  = block_number() * (kThreads / kWave) + threadIdx.x / kWave;
  if (item >= static_cast<int64_t>(f.key_runs.tokens) * f.kv_heads) return;
  int32_t const t = static_cast<int32_t>(item / f.kv_heads), head = static_cast<int32_t>(item % f.kv_heads), run = run_with(f.key_runs, t);
  if (!f.is_row(run)) return;
  int32_t first, keys;
  f.keys_of(run, first, keys);
  int32_t const tokens = f.runs.begin(run + 1) - f.runs.begin(run), i = t - first, block0 = i >> shift << shift;
  if (i >= keys || tokens <= 0) return;
  int64_t const from = f.causal ? static_cast<int64_t>(block0) + tokens - keys : 0;
  int32_t const start = static_cast<int32_t>(from < 0 ? 0 : from < tokens ? from : tokens) / kTile, tiles = (tokens + kTile - 1) / kTile;
  int32_t const shares = shares_of((tiles - start) * (f.heads / f.kv_heads), split.splits);
  if (shares < 2) return;
  int64_t const at   = (split.slot(f.key_runs.first_block(run, shift) + (i >> shift), head, f.kv_heads, 0) << shift) + (i & ((1 << shift) - 1));
  int64_t const step = static_cast<int64_t>(2 * D) << shift;
  Some<D> const sum_k = add_shares<D>(split.sums + at * (2 * D), step, shares, f.scale), sum_v = add_shares<D>(split.sums + at * (2 * D) + D, step, shares, 1.f);
  bool of_k = false, of_v = false;  // (what is made once more)
  if (f.causal) {
    int32_t const begin = f.runs.begin(run), own = static_cast<int32_t>(std::min<int64_t>(std::max<int64_t>(static_cast<int64_t>(i) + tokens - keys, 0), tokens));
    auto const again    = [&](Some<D> const& sum, bool k) {
      return !sum.finite(f.width) && tokens_hold_odd(f, begin + start * kTile, own - start * kTile, head, k, !k) && !is_odd_anyway(f, begin, own, tokens, head, k, !k);
    };
    of_k = again(sum_k, true);
    of_v = again(sum_v, false);
    if (of_k || of_v) key_gradient_row(f, t, head, of_k, of_v);
  }
  if (!of_k) write_row<T, D>(f.k_grad.at(t, head), sum_k, f.width);
  if (!of_v) write_row<T, D>(f.v_grad.at(t, head), sum_v, f.width);
}

// ------------------------------------------------------------------ launches
template <typename T, int D, int WAVES, Part PART>
nvtext_amd_status key_gradient_tiles(Backward<T> const& f, Split const& split, hipStream_t stream)
{
  using Shape = KeyShape<T, D, WAVES>;
  ProfileScope const scope("attention_key_gradient", stream);
  NVTEXT_HIP_TRY(allow_lds(key_gradient_tiles_kernel<T, D, WAVES, PART>, Shape::kLds));
  int64_t const items = work_items(f.key_runs.blocks(Shape::kShift), f.kv_heads, 1, split.splits);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(key_gradient_tiles_kernel<T, D, WAVES, PART>), grid_of(items, WAVES * kWave), dim3(WAVES * kWave), Shape::kLds, stream, f, split);
  return NVTEXT_AMD_SUCCESS;
}

template <typename T, int D, int WAVES>
nvtext_amd_status key_gradient_parts(Backward<T> const& f, Split const& split, hipStream_t stream)
{
  if constexpr (D > 96) {
    nvtext_amd_status const st = key_gradient_tiles<T, D, WAVES, kOfK>(f, split, stream);
    return st == NVTEXT_AMD_SUCCESS ? key_gradient_tiles<T, D, WAVES, kOfV>(f, split, stream) : st;
  } else {
    return key_gradient_tiles<T, D, WAVES, kBoth>(f, split, stream);
  }
}

template <typename T, int D, int WAVES>
nvtext_amd_status query_gradient_tiles(Backward<T> const& f, Split const& split, hipStream_t stream)
{
  using Shape = GradientShape<T, D, WAVES>;
  ProfileScope const scope("attention_query_gradient", stream);
  NVTEXT_HIP_TRY(allow_lds(query_gradient_tiles_kernel<T, D, WAVES>, Shape::kLds));
  int64_t const items = work_items(f.runs.blocks(Shape::kShift), f.kv_heads, f.heads / f.kv_heads, split.splits);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(query_gradient_tiles_kernel<T, D, WAVES>), grid_of(items, WAVES * kWave), dim3(WAVES * kWave), Shape::kLds, stream, f, split);
  return NVTEXT_AMD_SUCCESS;
}

template <typename T, int D>
nvtext_amd_status gradient_tiles(Backward<T> const& f, Mr const& mr, hipStream_t stream)
{
  using OfQ = GradientShape<T, D, kTileWaves>;
  using OfK = KeyShape<T, D, kTileWaves>;
  constexpr int kLds = 4 * Tile<T, D>::kBytes;  // (where tiles are smaller, a CU has one workgroup for the registers that it takes)
  Split of_q{splits_of<T, D, 3>(f, f.runs, f.heads, OfQ::kShift, f.key_runs, 1, kLds), nullptr, nullptr};
  Split of_k{splits_of<T, D, (D > 96 ? 5 : 4)>(f, f.key_runs, f.kv_heads, OfK::kShift, f.runs, f.heads / f.kv_heads, kLds), nullptr, nullptr};
  TempParts<2> const temp(mr, {of_q.splits > 1 ? static_cast<size_t>(f.runs.blocks(OfQ::kShift) * f.heads * of_q.splits * OfQ::kRows * D) * sizeof(float) : 0,
                               of_k.splits > 1 ? static_cast<size_t>(f.key_runs.blocks(OfK::kShift) * f.kv_heads * of_k.splits * OfK::kRows * D) * 2 * sizeof(float) : 0});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  of_q.sums = temp.template part<float>(0);
  of_k.sums = temp.template part<float>(1);
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  if (f.runs.tokens > 0) st = of_q.splits == 1 && is_short(f, kShort<T>) ? query_gradient_tiles<T, D, 1>(f, of_q, stream) : query_gradient_tiles<T, D, kTileWaves>(f, of_q, stream);
  if (st != NVTEXT_AMD_SUCCESS) return st;
  if (of_q.splits > 1) {
    ProfileScope const scope("attention_query_gradient_join", stream);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(query_gradient_join_kernel<T, D>), grid_of((static_cast<int64_t>(f.runs.tokens) * f.heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f, of_q,
                       int{OfQ::kShift});
  }
  if (f.key_runs.tokens == 0) return NVTEXT_AMD_SUCCESS;
  st = of_k.splits == 1 && is_short(f, kShort<T>) ? key_gradient_parts<T, D, 1>(f, of_k, stream) : key_gradient_parts<T, D, kTileWaves>(f, of_k, stream);
  if (st != NVTEXT_AMD_SUCCESS || of_k.splits == 1) return st;
  ProfileScope const scope("attention_key_gradient_join", stream);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(key_gradient_join_kernel<T, D>), grid_of((static_cast<int64_t>(f.key_runs.tokens) * f.kv_heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f, of_k,
                     int{OfK::kShift});
  return NVTEXT_AMD_SUCCESS;
}

template <typename T>
nvtext_amd_status attention_backward(Backward<T> f, Mr const& mr, hipStream_t stream)
{
  Alignment<T> align(f.width);
  for (auto* x : {&f.q, &f.grad, &f.out}) align.add(*x, f.runs.tokens, f.heads);
  for (auto* x : {&f.k, &f.v}) align.add(*x, f.key_runs.tokens, f.kv_heads);
  size_t const values = static_cast<size_t>(f.heads) * static_cast<size_t>(f.runs.tokens) * sizeof(float);
  TempParts<3> const temp(mr, {values, values, align.bytes()});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  f.deltas = temp.template part<float>(0);
  f.logs   = temp.template part<float>(1);
  align.launch(temp.template part<char>(2), stream);
  return with_tiles(f.width, [&](auto d) { return gradient_tiles<T, decltype(d)::value>(f, mr, stream); });
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_attention_backward(const nvtext_amd_heads* grad, const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, const nvtext_amd_heads* out,
                                                const float* logsum, const int8_t* rest, int32_t rows, const int32_t* offsets, const int32_t* key_offsets, const int32_t* key_lengths, int32_t causal,
                                                double scale, void* stream_, const nvtext_amd_allocator* mr_, const nvtext_amd_heads* q_grad, const nvtext_amd_heads* k_grad,
                                                const nvtext_amd_heads* v_grad)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_attention_backward");
  if (!grad || !q || !k || !v || !out || !q_grad || !k_grad || !v_grad) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_attention(q, k, v, rows, offsets, key_offsets, key_lengths, scale)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  for (auto* x : {grad, out}) {
    if (const char* bad = bad_heads(x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (x->type != q->type || !is_like(x, q)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "grad and out must be of q's size and type");
  }
  for (auto* x : {q_grad, k_grad, v_grad}) {
    if (const char* bad = bad_result(x)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
    if (x->type != q->type || !is_like(x, x == q_grad ? q : k)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the gradients must be of the size and type of what they are those of");
  }
  if (q->heads == 0 || q->width == 0 || (q->tokens == 0 && k->tokens == 0)) return NVTEXT_AMD_SUCCESS;
  if (q->tokens > 0 && !logsum) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  with_type(q->type, [&](auto zero) {
    using T = decltype(zero);
    Backward<T> b{problem_of<T>(q, k, v, rows, offsets, key_offsets, key_lengths, causal, scale)};
    b.grad   = heads_of<const T>(grad);
    b.out    = heads_of<const T>(out);
    b.logsum = logsum;
    b.rest   = q->type == NVTEXT_AMD_TYPE_FLOAT32 ? nullptr : rest;
    b.q_grad = heads_of<T>(q_grad);
    b.k_grad = heads_of<T>(k_grad);
    b.v_grad = heads_of<T>(v_grad);
    st       = attention_backward<T>(b, mr, stream);
  });
  if (st != NVTEXT_AMD_SUCCESS) return st;
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
