// Attention of a row's tokens over its keys, and its gradient.
#include "attention.cuh"

#include <cmath>
#include <type_traits>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;
constexpr int kTileWaves = 4;  // wavefronts that share the tiles in LDS

// ------------------------------------------------------------------ forward, in tiles
// The work of a launch: blocks of tokens, of every head, in `splits` shares.  The heads that share a key head come one after the other on one XCD (workgroups go
// to the eight XCDs in turn), and so do, where the number of key heads allows, the blocks of a key head: its keys come from that XCD's L2.  The last
// blocks come first: of a long row they are those with the most keys to see.
struct Work {
  int64_t block;
  int32_t kv_head, head, share;
};
constexpr int kXcds = 8;
inline int64_t work_items(int64_t blocks, int32_t kv_heads, int32_t each, int32_t splits) { return (blocks * kv_heads + kXcds - 1) / kXcds * kXcds * each * splits; }
// false: nothing to do
template <typename Int>
__device__ __forceinline__ bool work_in(Int item, Int blocks, int32_t kv_heads, int32_t each, int32_t splits, Work& w)
{
  Int const n = item / kXcds / static_cast<Int>(splits), units = n / static_cast<Int>(each), unit = units * kXcds + item % kXcds;
  if (unit >= blocks * static_cast<Int>(kv_heads)) return false;
  Int const behind = unit / static_cast<Int>(kv_heads);
  w.block          = static_cast<int64_t>(blocks - 1 - behind);
  w.kv_head        = static_cast<int32_t>(unit - behind * static_cast<Int>(kv_heads));
  w.head           = w.kv_head * each + static_cast<int32_t>(n - units * static_cast<Int>(each));
  w.share          = static_cast<int32_t>(item / kXcds - n * static_cast<Int>(splits));
  return true;
}
__device__ __forceinline__ bool work_of(int64_t item, int64_t blocks, int32_t kv_heads, int32_t each, int32_t splits, Work& w)
{
  // (divisions of 64 bits take a hundred instructions each)
  if (blocks * kv_heads < (int64_t{1} << 32) - kXcds && item < int64_t{1} << 32) return work_in<uint32_t>(item, blocks, kv_heads, each, splits, w);
  return work_in<uint64_t>(item, blocks, kv_heads, each, splits, w);
}

// Where there are few workgroups, each one's tiles are shared by up to `splits`, which leave what they add up in memory, [block][head][share][row][D] in
// float32, for another launch to join.  A share has at least kLeastTiles: in how many shares `tiles` go, and what one of them has.
constexpr int kLeastTiles = 2;
__device__ __forceinline__ int32_t shares_of(int32_t tiles, int32_t splits) { return splits == 1 || tiles < 2 * kLeastTiles ? 1 : min(splits, tiles / kLeastTiles); }
__device__ __forceinline__ int32_t share_begin(int32_t tiles, int32_t share, int32_t shares) { return static_cast<int32_t>(static_cast<int64_t>(tiles) * share / shares); }

struct Split {
  int32_t splits;
  float* sums;
  float2* tops;  // (forward) [block][head][share][row]: top, and the sum of the exponentials
  __device__ __forceinline__ int64_t slot(int64_t block, int32_t head, int32_t heads, int32_t share) const { return (block * heads + head) * splits + share; }
};

template <typename T, int D, int WAVES>
struct ForwardShape {
  static constexpr int kTokens = 32 * WAVES, kShift = __builtin_ctz(kTokens), kTile = Tile<T, D>::kHeads, kLds = 4 * Tile<T, D>::kBytes, kWavesASimd = D * sizeof(T) <= 128 ? 4 : D * sizeof(T) <= 256 ? 2 : 1;
};

// What a wavefront holds of 32 heads of tokens, columns of the products, while keys pass: q, and the sums of out, transposed.  Scores are products with the
// keys as rows, so a lane has all of a column's scores (with the one 32 further on), and exponentials are in its registers as the second product
// takes them: no lane needs another's but for the maximum.  Sums are kept in proportion to 2^top, where top is a maximum that may be 8 too small:
// only then are they multiplied anew.
template <typename T, int D>
struct Attending {
  static constexpr int kSteps = D / 16, kColumns = D / 32, kTile = Tile<T, D>::kHeads, kBlocks = kTile / 32;
  static constexpr float kSlack = 8.f;
  Fragment<T> q[kSteps];
  f32x16_t o[kColumns];
  float top, sum;
  int32_t seen;  // keys that the column sees

  __device__ __forceinline__ void begin(const T* head, int32_t width, bool there, int half)
  {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = fragment_of(head, 16 * s + 8 * half, width, there);
    top = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) o[c] = f32x16_t{};
  }

  // A tile of keys from key0 on; partly: not all columns see all of it.  Fragments are read kAhead products before they are multiplied, and what vector instructions
  // have to do is spread between the products: the maximum of a block of 32 keys while the next one's scores are made, exponentials of 16 keys while those
  // before are multiplied with v.  (Left to itself, the compiler reads a fragment, waits for it and multiplies.)
  __device__ __forceinline__ void pass(LdsBytes k_tile, LdsBytes v_tile, TileReader<T, D> const& read, int32_t key0, bool partly, float scale, int half)
  {
    f32x16_t s[kBlocks];
    {
      constexpr int kSlots = kBlocks * kSteps;
      stream<T, kSlots>([&](auto i) { return read.rows(k_tile, i / kSteps, i % kSteps); },
                        [&](auto i, Fragment<T> const& k) {
                          constexpr int b = i / kSteps, step = i % kSteps;
                          if constexpr (step == 0) s[b] = f32x16_t{};
                          s[b] = multiply32(k, q[step], s[b]);
                        });
    }
    if (partly) {
      int32_t const left = seen - key0 - 4 * half;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = 32 * b + 8 * (r / 4) + r % 4 < left ? s[b][r] : -INFINITY;
    }
    float high = s[0][0];
#pragma unroll
    for (int r = 1; r < 16 * kBlocks; ++r) high = fmaxf(high, s[r / 16][r % 16]);
    Halves const both = halves(high);
    high              = fmaxf(both.low, both.high) * scale;
    // (a column that sees nothing yet keeps top at -infinity; NaN in a score is found in out at the end)
    if (__ballot(high > top + kSlack || top == -INFINITY)) {
      float const now  = fmaxf(top, high);
      float const fade = now == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
      top              = now;
      sum *= fade;
#pragma unroll
      for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[c][r] *= fade;
    }
    constexpr int kRounds = 2 * kBlocks;
    float const base = top == -INFINITY ? 0.f : top;
    auto const exponential = [&](int step, int e) {
      int const r    = 8 * (step % 2) + e;
      float const x  = __builtin_amdgcn_exp2f(fmaf(s[step / 2][r], scale, -base));
      s[step / 2][r] = x;
      sum += x;
    };
    Fragment<T> p;
    stream<T, kRounds * kColumns>([&](auto i) { return read.columns(v_tile, i % kColumns, i / kColumns); },
                                  [&](auto i, Fragment<T> const& v) {
                                    constexpr int step = i / kColumns, c = i % kColumns;
                                    if constexpr (i == 0) {
#pragma unroll
                                      for (int e = 0; e < 8; ++e) exponential(0, e);
                                      p = rounded<T>(s[0], 0);
                                    }
                                    o[c] = multiply32(v, p, o[c]);
                                    if constexpr (step + 1 < kRounds) {
#pragma unroll
                                      for (int e = c * 8 / kColumns; e < (c + 1) * 8 / kColumns; ++e) exponential(step + 1, e);
                                      if constexpr (c == kColumns - 1) p = rounded<T>(s[(step + 1) / 2], (step + 1) % 2);
                                    }
                                  });
  }

  // Writes out and logsum of a column, head h of token t, where it is `there`; of those whose result is not finite, the lanes' numbers.  That may come from keys that the
  // token does not see, whose exponentials of 0 were multiplied: such columns are done once more, by themselves.
  __device__ __forceinline__ uint32_t finish(Forward<T> const& f, int64_t t, int32_t h, bool there, int half, int column)
  {
    Halves const both = halves(sum);
    float const total = both.low + both.high, part = seen > 0 ? 1.f / total : 0.f;
    float check       = 0.f;  // (NaN if any is infinite or NaN)
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[c][r] *= part;
        check = fmaf(o[c][r], 0.f, check);
      }
    uint64_t odd = __ballot(there && seen > 0 && check != 0.f);
    odd          = (odd | odd >> 32) & 0xffffffffu;
    if (there && !(odd >> column & 1)) {
      store_columns<T, kColumns>(f.out.at(t, h), o, half, f.width);
      int64_t const at = static_cast<int64_t>(h) * f.runs.tokens + t;
      if constexpr (sizeof(T) == 2)
        if (f.rest) store_rests<T, kColumns>(f.rest + at * f.width, o, half, f.width);
      if (f.logsum && half == 0) f.logsum[at] = seen > 0 ? (top + __builtin_amdgcn_logf(total)) * kLn2 : -INFINITY;
    }
    return static_cast<uint32_t>(odd);
  }
};

// A workgroup has kTokens tokens of a head, a wavefront 32 of them.  Keys come through LDS, 64 at a time, the next ones while these are multiplied.
template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave, (ForwardShape<T, D, WAVES>::kWavesASimd)) attend_tiles_kernel(Forward<T> f, Split split)
{
  using Shape = ForwardShape<T, D, WAVES>;
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds  = (LdsBytes)lds_;
  constexpr int kTile = Shape::kTile, kStage = 2 * Tile<T, D>::kBytes;
  Work w;
  int32_t const each = f.heads / f.kv_heads;
  if (!work_of(block_number(), f.runs.blocks(Shape::kShift), f.kv_heads, each, split.splits, w)) return;
  int32_t const run   = f.runs.run_of(w.block, Shape::kShift);
  int32_t const begin = uniform(f.runs.begin(run)), tokens = uniform(f.runs.begin(run + 1)) - begin;
  int64_t const in_run = (w.block - f.runs.first_block(run, Shape::kShift)) << Shape::kShift;
  if (in_run >= tokens) return;
  int const wave = uniform(threadIdx.x / kWave), lane = lane_id(), column = lane % 32, half = lane / 32;
  int32_t const block0 = static_cast<int32_t>(in_run), rest = uniform(tokens - block0);  // the first token in the run, tokens from there on
  int32_t first = 0, keys = 0;
  if (f.is_row(run)) f.keys_of(run, first, keys);
  first = uniform(first);
  keys  = uniform(keys);
  // keys that the workgroup's last token sees, and the wavefront's first and last
  int32_t const wave0 = wave * 32, wave1 = wave0 + 32 < rest ? wave0 + 32 : rest;
  int32_t const all   = uniform(f.seen(block0 + (rest < Shape::kTokens ? rest : Shape::kTokens) - 1, tokens, keys));
  int32_t const least = uniform(wave0 < rest ? f.seen(block0 + wave0, tokens, keys) : 0), most = uniform(wave0 < rest ? f.seen(block0 + wave1 - 1, tokens, keys) : 0);
  bool const there    = wave0 + column < rest;
  int64_t const t     = static_cast<int64_t>(begin) + block0 + (there ? wave0 + column : 0);

  int32_t const all_tiles = (all + kTile - 1) / kTile, shares = shares_of(all_tiles, split.splits);
  if (w.share >= shares) return;
  int32_t const from = uniform(share_begin(all_tiles, w.share, shares)), tiles = uniform(share_begin(all_tiles, w.share + 1, shares));

  Attending<T, D> a;
  a.seen = there ? f.seen(block0 + wave0 + column, tokens, keys) : 0;
  a.begin(f.q.at(t, w.head), f.width, there, half);
  TileLoader<T, D, WAVES> load_k, load_v;
  load_k.aim(f.k, first + from * kTile, w.kv_head, f.width, wave, lane);
  load_v.aim(f.v, first + from * kTile, w.kv_head, f.width, wave, lane);
  auto const load = [&](int32_t tile) {
    LdsBytes const to = lds + (tile & 1) * kStage;
    load_k.load(to, keys - tile * kTile, wave);
    load_v.load(to + Tile<T, D>::kBytes, keys - tile * kTile, wave);
  };
  TileReader<T, D> const read(lane);
  float const scale = f.scale * kLog2e;
  if (tiles > from) load(from);
  for (int32_t tile = from; tile < tiles; ++tile) {
    LdsBytes const k_tile = lds + (tile & 1) * kStage;
    stage_barrier<0>();
    if (tile + 1 < tiles) load(tile + 1);
    int32_t const key0 = tile * kTile;
    if (key0 < most) a.pass(k_tile, k_tile + Tile<T, D>::kBytes, read, key0, key0 + kTile > least, scale, half);
  }
  if (wave0 >= rest) return;
  if (shares > 1) {
    int64_t const part = split.slot(w.block, w.head, f.heads, w.share) * Shape::kTokens + wave0 + column;
    Halves const both  = halves(a.sum);
    if (there) {
      store_columns<float, D / 32>(split.sums + part * D, a.o, half, D);
      if (half == 0) split.tops[part] = make_float2(a.top, both.low + both.high);
    }
    return;
  }
  uint32_t odd = a.finish(f, t, w.head, there, half, column);
  for (; odd; odd &= odd - 1) attend_row(f, begin + block0 + wave0 + __builtin_ctz(odd), w.head);
}

// ------------------------------------------------------------------ forward, in chunks of keys
// Few tokens a row, as where texts go on token by token: one wavefront has all of a row's tokens and of all heads that share a key head, up to 32 together,
// as the columns of its products, and a chunk of 2^shift of the row's keys; what it adds up is joined with that of the row's other chunks by another
// launch.  Bound by memory: the keys are read once.  The chunks of key tokens are numbered as the blocks of tokens are elsewhere, so they are
// alike in size however long the rows are.  A row of a single chunk is finished at once; so is one of more columns, by the workgroup of its first chunk
// alone, 32 columns after the other.
// Parts of a row of several chunks lie from number 2 * first / 2^shift on: it has at least half as many numbers up to the next row's as it has chunks.
constexpr int kPartColumns = 32;

template <typename T>
struct ForwardChunks : Forward<T> {
  int shift;
  float* sums;    // [part][key head][column][D]
  float2* tops;   // [part][key head][column]: top, and the sum of the exponentials
  __device__ __forceinline__ int64_t part(int32_t first, int32_t chunk, int32_t kv_head) const
  {
    return ((static_cast<int64_t>(first) * 2 >> shift) + chunk) * this->kv_heads + kv_head;
  }
  __device__ __forceinline__ int32_t chunks_of(int32_t keys) const { return keys > 0 ? ((keys - 1) >> shift) + 1 : 1; }
  __device__ __forceinline__ bool is_split(int32_t tokens, int32_t chunks) const { return chunks > 1 && static_cast<int64_t>(tokens) * (this->heads / this->kv_heads) <= kPartColumns; }
};
inline int64_t most_parts(int64_t key_tokens, int shift) { return (key_tokens * 2 >> shift) + 2; }

template <typename T, int D>
__global__ void __launch_bounds__(kWave, 1) attend_chunks_kernel(ForwardChunks<T> f)
{
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds  = (LdsBytes)lds_;
  constexpr int kTile = Tile<T, D>::kHeads;
  Work w;
  if (!work_of(block_number(), f.key_runs.blocks(f.shift), f.kv_heads, 1, 1, w)) return;
  int32_t const run = f.key_runs.run_of(w.block, f.shift), each = f.heads / f.kv_heads;
  int32_t first = 0, keys = 0;
  if (f.is_row(run)) f.keys_of(run, first, keys);
  first = uniform(first);
  keys  = uniform(keys);
  int32_t const begin = uniform(f.runs.begin(run)), tokens = uniform(f.runs.begin(run + 1)) - begin, chunks = f.chunks_of(keys);
  int64_t const chunk = w.block - f.key_runs.first_block(run, f.shift);
  bool const split    = f.is_split(tokens, chunks);
  if (chunk >= (split ? chunks : 1)) return;
  int const lane = lane_id(), column = lane % 32, half = lane / 32;
  int32_t const key_first = split ? static_cast<int32_t>(chunk << f.shift) : 0, key_last = split && keys - key_first > 1 << f.shift ? key_first + (1 << f.shift) : keys;
  int64_t const columns   = static_cast<int64_t>(tokens > 0 ? tokens : 0) * each;
  TileReader<T, D> const read(lane);
  float const scale = f.scale * kLog2e;
  for (int64_t column0 = 0; column0 < columns; column0 += kPartColumns) {
    int64_t const mine = column0 + column;
    bool const there   = mine < columns;
    int32_t const i    = there ? static_cast<int32_t>(mine / each) : 0, head = w.kv_head * each + (there ? static_cast<int32_t>(mine - static_cast<int64_t>(i) * each) : 0);
    int64_t const t    = static_cast<int64_t>(begin) + i;
    int32_t const last = static_cast<int32_t>(((column0 + kPartColumns < columns ? column0 + kPartColumns : columns) - 1) / each);  // the last column's token
    Attending<T, D> a;
    a.seen = there ? f.seen(i, tokens, keys) : 0;
    a.begin(f.q.at(t, head), f.width, there, half);
    int32_t const least = uniform(f.seen(static_cast<int32_t>(column0 / each), tokens, keys)), all = uniform(f.seen(last, tokens, keys)), end = all < key_last ? all : key_last;
    int32_t const tiles = end > key_first ? (end - key_first + kTile - 1) / kTile : 0;
    TileLoader<T, D, 1> load_k, load_v;
    load_k.aim(f.k, first + key_first, w.kv_head, f.width, 0, lane);
    load_v.aim(f.v, first + key_first, w.kv_head, f.width, 0, lane);
    if (tiles > 0) {
      load_k.load(lds, key_last - key_first, 0);
      load_v.load(lds + Tile<T, D>::kBytes, key_last - key_first, 0);
    }
    for (int32_t tile = 0; tile < tiles; ++tile) {
      LdsBytes const k_tile = lds + (tile & 1) * 2 * Tile<T, D>::kBytes;
      int32_t const key0    = key_first + tile * kTile;
      stage_barrier<0>();
      if (tile + 1 < tiles) {
        LdsBytes const next = lds + (~tile & 1) * 2 * Tile<T, D>::kBytes;
        load_k.load(next, key_last - key0 - kTile, 0);
        load_v.load(next + Tile<T, D>::kBytes, key_last - key0 - kTile, 0);
      }
      a.pass(k_tile, k_tile + Tile<T, D>::kBytes, read, key0, key0 + kTile > least || key0 + kTile > key_last, scale, half);
    }
    stage_barrier<0>();  // (the next columns' loads come into the same places)
    if (split) {
      int64_t const part = f.part(first, static_cast<int32_t>(chunk), w.kv_head) * kPartColumns + column;
      Halves const both  = halves(a.sum);
      if (there) {
        store_columns<float, D / 32>(f.sums + part * D, a.o, half, D);
        if (half == 0) f.tops[part] = make_float2(a.top, both.low + both.high);
      }
      continue;
    }
    for (uint32_t odd = a.finish(f, t, head, there, half, column); odd; odd &= odd - 1) {
      int const which = __builtin_ctz(odd);
      attend_row(f, __builtin_amdgcn_readlane(static_cast<int32_t>(t), which), __builtin_amdgcn_readlane(head, which));
    }
  }
}

// A wavefront's share of a row of D values.
template <int D>
using Some = float __attribute__((ext_vector_type(D / kWave)));

template <int D>
__device__ __forceinline__ void add_part(Some<D>& sum, float& total, float top, float2 of, const float* part)
{
  float const weight = of.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(of.x - top);
  total += of.y * weight;
  sum += *reinterpret_cast<const Some<D>*>(part + lane_id() * (D / kWave)) * weight;
}

// What Attending::finish does, for sums that a wavefront holds side by side.
template <typename T, int D>
__device__ __forceinline__ void finish_row(Forward<T> const& f, int32_t t, int32_t head, int32_t seen, Some<D> sum, float total, float top)
{
  constexpr int kEach = D / kWave;
  int const lane      = lane_id();
  bool finite         = true;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    sum[k] = seen > 0 ? sum[k] / total : 0.f;
    finite = finite && (lane * kEach + k >= f.width || fabsf(sum[k]) < INFINITY);
  }
  if (seen > 0 && __ballot(!finite)) {
    attend_row(f, t, head);
    return;
  }
  T* const out = f.out.at(t, head);
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (lane * kEach + k < f.width) {
      out[lane * kEach + k] = static_cast<T>(sum[k]);
      if (f.rest) f.rest[(static_cast<int64_t>(head) * f.runs.tokens + t) * f.width + lane * kEach + k] = rest_of(sum[k], static_cast<T>(sum[k]));
    }
  if (f.logsum && lane == 0) f.logsum[static_cast<int64_t>(head) * f.runs.tokens + t] = seen > 0 ? (top + __builtin_amdgcn_logf(total)) * kLn2 : -INFINITY;
}

// Joins the parts of a head of a token, a workgroup for each: its wavefronts take every fourth part.
constexpr int kJoinWaves = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWaves * kWave) attend_join_kernel(ForwardChunks<T> f)
{
  __shared__ float tops[kJoinWaves], totals[kJoinWaves];
  __shared__ Some<D> sums[kJoinWaves][kWave];
  int64_t const item = block_number();
  if (item >= static_cast<int64_t>(f.runs.tokens) * f.heads) return;
  int32_t const t = static_cast<int32_t>(item / f.heads), head = static_cast<int32_t>(item % f.heads), run = run_with(f.runs, t);
  if (!f.is_row(run)) return;
  int32_t first, keys;
  f.keys_of(run, first, keys);
  int32_t const begin = f.runs.begin(run), tokens = f.runs.begin(run + 1) - begin, chunks = f.chunks_of(keys), each = f.heads / f.kv_heads;
  if (!f.is_split(tokens, chunks)) return;
  int const wave = threadIdx.x / kWave, lane = lane_id();
  int32_t const column = (t - begin) * each + head % each;
  int64_t const at = f.part(first, 0, head / each) * kPartColumns + column, step = static_cast<int64_t>(f.kv_heads) * kPartColumns;
  float top = -INFINITY;
  for (int32_t c = threadIdx.x; c < chunks; c += kJoinWaves * kWave) top = fmaxf(top, f.tops[at + c * step].x);
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) top = fmaxf(top, tops[w]);
  float total = 0.f;
  Some<D> sum{};
#pragma unroll 8
  for (int32_t c = wave; c < chunks; c += kJoinWaves) add_part<D>(sum, total, top, f.tops[at + c * step], f.sums + (at + c * step) * D);
  sums[wave][lane] = sum;
  if (lane == 0) totals[wave] = total;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) {
    total += totals[w];
    sum += sums[w][lane];
  }
  finish_row<T, D>(f, t, head, f.seen(t - begin, tokens, keys), sum, total, top);
}

// The same for the shares of a block of 2^shift tokens, a wavefront for each head of a token.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attend_join_shares_kernel(Forward<T> f, Split split, int shift)
{
  constexpr int kTile = Tile<T, D>::kHeads;
  int64_t const item = block_number() * (kThreads / kWave) + threadIdx.x / kWave;
  if (item >= static_cast<int64_t>(f.runs.tokens) * f.heads) return;
  int32_t const t = static_cast<int32_t>(item / f.heads), head = static_cast<int32_t>(item % f.heads), run = run_with(f.runs, t);
  if (!f.is_row(run)) return;
  int32_t first, keys;
  f.keys_of(run, first, keys);
  int32_t const begin = f.runs.begin(run), tokens = f.runs.begin(run + 1) - begin, i = t - begin, last = i | ((1 << shift) - 1);
  int32_t const all = f.seen(last < tokens ? last : tokens - 1, tokens, keys), shares = shares_of((all + kTile - 1) / kTile, split.splits);
  if (shares < 2) return;
  int64_t const at = (split.slot(f.runs.first_block(run, shift) + (i >> shift), head, f.heads, 0) << shift) + (i & ((1 << shift) - 1));
  float top = -INFINITY;
  for (int32_t c = 0; c < shares; ++c) top = fmaxf(top, split.tops[at + (static_cast<int64_t>(c) << shift)].x);
  Some<D> sum{};
  float total = 0.f;
#pragma unroll 4
  for (int32_t c = 0; c < shares; ++c) add_part<D>(sum, total, top, split.tops[at + (static_cast<int64_t>(c) << shift)], split.sums + (at + (static_cast<int64_t>(c) << shift)) * D);
  finish_row<T, D>(f, t, head, f.seen(i, tokens, keys), sum, total, top);
}

// ------------------------------------------------------------------ the gradients, in tiles
// Two launches, the first for q, the second for k and v: each makes the scores anew and adds up what is its own in registers, in one order at every
// call.  (One launch for all three would have to add up q's gradient in memory, over all workgroups of keys: in parts of float32 or in any order.)
template <typename T, int D, int WAVES>
struct GradientShape {
  static constexpr int kRows = 32 * WAVES, kShift = __builtin_ctz(kRows), kTile = Tile<T, D>::kHeads, kStage = 2 * Tile<T, D>::kBytes, kLds = 2 * kStage, kWavesASimd = D * sizeof(T) <= 256 ? 2 : 1;
};

// The gradient of q: as forward, a lane has a token's scores, and what they are multiplied with comes from LDS, keys as they lie and transposed.
template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave, (GradientShape<T, D, WAVES>::kWavesASimd)) query_gradient_tiles_kernel(Backward<T> f, Split split)
{
  using Shape = GradientShape<T, D, WAVES>;
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds = (LdsBytes)lds_;
  constexpr int kSteps = D / 16, kColumns = D / 32, kTile = Shape::kTile, kBlocks = kTile / 32;
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

  TileLoader<T, D, WAVES> load_k, load_v;
  load_k.aim(f.k, first + first_tile * kTile, w.kv_head, f.width, wave, lane);
  load_v.aim(f.v, first + first_tile * kTile, w.kv_head, f.width, wave, lane);
  auto const load = [&](int32_t tile) {
    LdsBytes const to = lds + (tile & 1) * Shape::kStage;
    load_k.load(to, keys - tile * kTile, wave);
    load_v.load(to + Tile<T, D>::kBytes, keys - tile * kTile, wave);
  };
  if (tiles > first_tile) load(first_tile);
  int64_t const at = static_cast<int64_t>(w.head) * f.runs.tokens + t;
  Fragment<T> q[kSteps], g[kSteps];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    q[s] = fragment_of(f.q.at(t, w.head), 16 * s + 8 * half, f.width, there);
    g[s] = fragment_of(f.grad.at(t, w.head), 16 * s + 8 * half, f.width, there);
    Fragment<T> const out = fragment_of(f.out.at(t, w.head), 16 * s + 8 * half, f.width, there);
    bool rests = false;
    if constexpr (sizeof(T) == 2) rests = f.rest != nullptr;
    if (rests) {
      auto const rest = load_raw8(f.rest + at * f.width + 16 * s + 8 * half, there ? f.width - 16 * s - 8 * half : 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) delta = fmaf(static_cast<float>(g[s][k]), with_rest(out[k], rest[k]), delta);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) delta = fmaf(static_cast<float>(g[s][k]), static_cast<float>(out[k]), delta);
    }
  }
  Halves const both = halves(delta);
  delta             = seen > 0 ? both.low + both.high : 0.f;
  float const log   = there ? f.logsum[at] * kLog2e : 0.f;
  if (there && half == 0 && w.share == 0) {
    f.deltas[at] = delta;
    f.logs[at]   = log;
  }
  f32x16_t d[kColumns];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) d[c] = f32x16_t{};
  TileReader<T, D> const read(lane);
  float const scale = f.scale * kLog2e;
  for (int32_t tile = first_tile; tile < tiles; ++tile) {
    LdsBytes const k_tile = lds + (tile & 1) * Shape::kStage, v_tile = k_tile + Tile<T, D>::kBytes;
    stage_barrier<0>();
    if (tile + 1 < tiles) load(tile + 1);
    int32_t const key0 = tile * kTile;
    if (key0 >= most) continue;
    // Of each block of 32 keys, scores and products of g and v, then what they come to, multiplied with the keys: a stream of fragments, read kAhead before
    // they are multiplied.
    constexpr int kFirst = 2 * kSteps, kOfBlock = kFirst + 2 * kColumns;
    f32x16_t s, p;
    Fragment<T> ds[2];
    stream<T, kBlocks * kOfBlock>(
      [&](auto slot) {
        constexpr int b = slot / kOfBlock, i = slot % kOfBlock;
        if constexpr (i < kSteps) return read.rows(k_tile, b, i);
        else if constexpr (i < kFirst) return read.rows(v_tile, b, i - kSteps);
        else return read.columns(k_tile, (i - kFirst) % kColumns, 2 * b + (i - kFirst) / kColumns);
      },
      [&](auto slot, Fragment<T> const& x) {
        constexpr int b = slot / kOfBlock, i = slot % kOfBlock;
        if constexpr (i < kSteps) {
          if constexpr (i == 0) s = f32x16_t{};
          s = multiply32(x, q[i], s);
        } else if constexpr (i < kFirst) {
          if constexpr (i == kSteps) p = f32x16_t{};
          p = multiply32(x, g[i - kSteps], p);
        } else {
          if constexpr (i == kFirst) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], scale, -log)) * (p[r] - delta);
            if (key0 + 32 * b + 32 > least) {
              int32_t const left = seen - key0 - 32 * b - 4 * half;
#pragma unroll
              for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + r % 4 < left ? s[r] : 0.f;
            }
            ds[0] = rounded<T>(s, 0);
            ds[1] = rounded<T>(s, 1);
          }
          d[(i - kFirst) % kColumns] = multiply32(x, ds[(i - kFirst) / kColumns], d[(i - kFirst) % kColumns]);
        }
      });
  }
  if (wave0 >= rest) return;
  if (shares > 1) {
    if (there) store_columns<float, kColumns>(split.sums + (split.slot(w.block, w.head, f.heads, w.share) * Shape::kRows + wave0 + column) * D, d, half, D);
    return;
  }
  float check = 0.f;
#pragma unroll
  for (int c = 0; c < kColumns; ++c)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      d[c][r] *= f.scale;
      check = fmaf(d[c][r], 0.f, check);
    }
  // (as forward: a key that is not seen may have been multiplied by 0)
  uint64_t odd = __ballot(there && seen > 0 && check != 0.f);
  odd          = (odd | odd >> 32) & 0xffffffffu;
  if (there && !(odd >> column & 1)) store_columns<T, kColumns>(f.q_grad.at(t, w.head), d, half, f.width);
  for (; odd; odd &= odd - 1) query_gradient_row(f, begin + block0 + wave0 + __builtin_ctzll(odd), w.head);
}

// The gradients of k and v: a wavefront has 32 keys in its registers, a lane a key's scores, and the tokens of all heads that see them come through LDS
// with their gradients, 64 at a time, with their logs and deltas.
template <typename T, int D, int WAVES>
struct KeyShape {
  static constexpr int kRows = 32 * WAVES, kShift = __builtin_ctz(kRows), kTile = Tile<T, D>::kHeads, kTiles = 2 * Tile<T, D>::kBytes;
  static constexpr int kStage = kTiles + 2 * kWave * 4, kLds = 2 * kStage;  // (with logs and deltas)
  static constexpr int kWavesASimd = sizeof(T) == 2 && D <= 128 ? 2 : 1;
};
// PART: the gradients of both, or of k or v alone (of wide heads there are not the registers for both).
enum Part { kBoth, kOfK, kOfV };
template <typename T, int D, int WAVES, Part PART>
__global__ void __launch_bounds__(WAVES * kWave, (KeyShape<T, D, WAVES>::kWavesASimd)) key_gradient_tiles_kernel(Backward<T> f, Split split)
{
  using Shape = KeyShape<T, D, WAVES>;
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds = (LdsBytes)lds_;
  constexpr bool kK = PART != kOfV, kV = PART != kOfK;
  constexpr int kSteps = D / 16, kColumns = D / 32, kTile = Shape::kTile, kBlocks = kTile / 32;
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

  Fragment<T> k[kSteps], v[kK ? kSteps : 1];
  int32_t const from = from_of(key);
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    k[s] = fragment_of(f.k.at(t, w.kv_head), 16 * s + 8 * half, f.width, there && key < keys);
    if constexpr (kK) v[s] = fragment_of(f.v.at(t, w.kv_head), 16 * s + 8 * half, f.width, there && key < keys);
  }
  TileReader<T, D> const read(lane);
  float const scale = f.scale * kLog2e;
  f32x16_t dk[kK ? kColumns : 1], dv[kV ? kColumns : 1];
#pragma unroll
  for (int c = 0; c < kColumns; ++c) {
    if constexpr (kK) dk[c] = f32x16_t{};
    if constexpr (kV) dv[c] = f32x16_t{};
  }
  TileLoader<T, D, WAVES> load_q, load_g;
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
    load_g.load(to + Tile<T, D>::kBytes, here, wave);
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
    LdsBytes const q_tile = lds + (n & 1) * Shape::kStage, g_tile = q_tile + Tile<T, D>::kBytes, words = q_tile + Shape::kTiles + 16 * half;
    stage_barrier<0>();
    if (n + 1 < end_tile) load(lds + (~n & 1) * Shape::kStage);
    if (++tile == tiles) tile = start;
    int32_t const token0 = tile * kTile;
    if (token0 + kTile <= first_from) continue;
    // (as in the gradient of q: a stream of fragments)
    constexpr int kFirst = (kK ? 2 : 1) * kSteps, kOfBlock = kFirst + 2 * (kK && kV ? 2 : 1) * kColumns;
    f32x16_t s, p;
    Fragment<T> weight[2], ds[2];
    stream<T, kBlocks * kOfBlock>(
      [&](auto slot) {
        constexpr int b = slot / kOfBlock, i = slot % kOfBlock;
        if constexpr (i < kSteps) return read.rows(q_tile, b, i);
        else if constexpr (i < kFirst) return read.rows(g_tile, b, i - kSteps);
        else {
          constexpr int j = i - kFirst, step = j / ((kK && kV ? 2 : 1) * kColumns), c = j % ((kK && kV ? 2 : 1) * kColumns);
          if constexpr (kV && c < kColumns) return read.columns(g_tile, c, 2 * b + step);
          else return read.columns(q_tile, c % kColumns, 2 * b + step);
        }
      },
      [&](auto slot, Fragment<T> const& x) {
        constexpr int b = slot / kOfBlock, i = slot % kOfBlock;
        if constexpr (i < kSteps) {
          if constexpr (i == 0) s = f32x16_t{};
          s = multiply32(x, k[i], s);
        } else if constexpr (i < kFirst) {
          if constexpr (i == kSteps) p = f32x16_t{};
          p = multiply32(x, v[i - kSteps], p);
        } else {
          if constexpr (i == kFirst) {
            int32_t const row0 = token0 + 32 * b;
            bool const partly  = row0 < last_from || row0 + 32 > tokens;
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
            if (partly) {
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                int32_t const token = row0 + 8 * (r / 4) + 4 * half + r % 4;
                bool const sees     = token >= from && token < tokens;
                if constexpr (kV) s[r] = sees ? s[r] : 0.f;
                if constexpr (kK) p[r] = sees ? p[r] : 0.f;
              }
            }
#pragma unroll
            for (int step = 0; step < 2; ++step) {
              if constexpr (kV) weight[step] = rounded<T>(s, step);
              if constexpr (kK) ds[step] = rounded<T>(p, step);
            }
          }
          constexpr int j = i - kFirst, step = j / ((kK && kV ? 2 : 1) * kColumns), c = j % ((kK && kV ? 2 : 1) * kColumns);
          if constexpr (kV && c < kColumns) dv[c] = multiply32(x, weight[step], dv[c]);
          else dk[c % kColumns] = multiply32(x, ds[step], dk[c % kColumns]);
        }
      });
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
  uint64_t odd = __ballot(there && check != 0.f);
  odd          = (odd | odd >> 32) & 0xffffffffu;
  if (there && !(odd >> column & 1)) {
    if constexpr (kK) store_columns<T, kColumns>(f.k_grad.at(t, w.kv_head), dk, half, f.width);
    if constexpr (kV) store_columns<T, kColumns>(f.v_grad.at(t, w.kv_head), dv, half, f.width);
  }
  for (; odd; odd &= odd - 1) key_gradient_row(f, first + block0 + wave0 + __builtin_ctzll(odd), w.kv_head, kK, kV);
}

// Adds up the shares of a head of a token (of q) or a key, a wavefront for each; the numbers of shares are those that the kernels before found.
template <int D>
__device__ __forceinline__ Some<D> add_shares(const float* at, int64_t step, int32_t shares)
{
  Some<D> sum{};
#pragma unroll 4
  for (int32_t c = 0; c < shares; ++c) sum += *reinterpret_cast<const Some<D>*>(at + c * step + lane_id() * (D / kWave));
  return sum;
}

// Writes a row of a gradient; false: not, what it holds is not finite.
template <typename T, int D>
__device__ __forceinline__ bool write_row(T* head, Some<D> sum, int32_t width)
{
  constexpr int kEach = D / kWave;
  bool finite         = true;
#pragma unroll
  for (int k = 0; k < kEach; ++k) finite = finite && (lane_id() * kEach + k >= width || fabsf(sum[k]) < INFINITY);
  if (__ballot(!finite)) return false;
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (lane_id() * kEach + k < width) head[lane_id() * kEach + k] = static_cast<T>(sum[k]);
  return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) query_gradient_join_kernel(Backward<T> f, Split split, int shift)
{
  constexpr int kTile = Tile<T, D>::kHeads;
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
  if (!write_row<T, D>(f.q_grad.at(t, head), add_shares<D>(split.sums + at * D, static_cast<int64_t>(D) << shift, shares) * f.scale, f.width)) query_gradient_row(f, t, head);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) key_gradient_join_kernel(Backward<T> f, Split split, int shift)
{
  constexpr int kTile = Tile<T, D>::kHeads;
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
  bool const of_k    = write_row<T, D>(f.k_grad.at(t, head), add_shares<D>(split.sums + at * (2 * D), step, shares) * f.scale, f.width);
  bool const of_v    = write_row<T, D>(f.v_grad.at(t, head), add_shares<D>(split.sums + at * (2 * D) + D, step, shares), f.width);
  if (!of_k || !of_v) key_gradient_row(f, t, head, !of_k, !of_v);
}

// ------------------------------------------------------------------ launches
// Whether the tiles' loads can read heads as they lie: pieces of 16 bytes, and lines of a tile within the 31 bits of their offsets.
template <typename T>
bool reads_as_it_lies(Heads<const T> const& x, int32_t width)
{
  constexpr int kEach = 16 / sizeof(T);
  return width % kEach == 0 && x.stride % kEach == 0 && x.head_stride % kEach == 0 && reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.stride < (int64_t{1} << 23);
}

// Heads that the tiles cannot read are copied first: head after head, token after token, each filled up with zeros to a multiple of 16 bytes.
template <typename T>
struct Copy {
  static constexpr int kEach = 16 / sizeof(T);
  Heads<const T> from;
  T* to;
  int64_t tokens, pieces;  // of all heads; 0: nothing to copy
};
constexpr int kCopies = 5;
template <typename T>
struct Copies {
  Copy<T> copy[kCopies];
  int32_t width;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) copy_heads_kernel(Copies<T> c)
{
  constexpr int kEach   = Copy<T>::kEach;
  int64_t item          = block_number() * kThreads + threadIdx.x;
  int32_t const of_head = (c.width + kEach - 1) / kEach;
#pragma unroll
  for (int n = 0; n < kCopies; ++n) {
    Copy<T> const& x = c.copy[n];
    if (item >= 0 && item < x.pieces) {
      int64_t const head = item / of_head / x.tokens, t = item / of_head % x.tokens, j = item % of_head * kEach;
      const T* const from = x.from.at(t, head) + j;
      typedef T Piece __attribute__((ext_vector_type(kEach)));
      Piece p{};
#pragma unroll
      for (int k = 0; k < kEach; ++k)
        if (j + k < c.width) p[k] = from[k];
      *reinterpret_cast<Piece*>(x.to + item * kEach) = p;
    }
    item -= x.pieces;
  }
}

// Which of up to five heads are copied, what that takes, and the launch that does it.
template <typename T>
struct Alignment {
  Copies<T> copies{};
  Heads<const T>* heads[kCopies]{};
  int count{0};
  explicit Alignment(int32_t width) { copies.width = width; }
  void add(Heads<const T>& x, int64_t tokens, int64_t of_token)
  {
    heads[count]  = &x;
    Copy<T>& c    = copies.copy[count++];
    c.from        = x;
    c.tokens      = tokens;
    c.pieces      = reads_as_it_lies(x, copies.width) ? 0 : tokens * of_token * ((copies.width + Copy<T>::kEach - 1) / Copy<T>::kEach);
  }
  size_t bytes() const
  {
    size_t sum = 0;
    for (auto const& c : copies.copy) sum += static_cast<size_t>(c.pieces) * 16;
    return sum;
  }
  void launch(char* memory, hipStream_t stream)
  {
    int64_t all = 0;
    for (int n = 0; n < count; ++n) {
      Copy<T>& c = copies.copy[n];
      if (c.pieces == 0) continue;
      int64_t const line = (copies.width + Copy<T>::kEach - 1) / Copy<T>::kEach * Copy<T>::kEach;
      c.to               = reinterpret_cast<T*>(memory);
      *heads[n]          = {c.to, line, c.tokens * line};
      memory += c.pieces * 16;
      all += c.pieces;
    }
    if (all == 0) return;
    ProfileScope const scope("attention_copy", stream);
    hipLaunchKernelGGL(copy_heads_kernel<T>, grid_of((all + kThreads - 1) / kThreads, kThreads), dim3(kThreads), 0, stream, copies);
  }
};

// (where kernels take more than 64 KB of LDS, the runtime wants to be told)
template <typename Kernel>
hipError_t allow_lds(Kernel kernel, int bytes)
{
  return bytes > 65536 ? hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) : hipSuccess;
}

// In how many shares the tiles of a workgroup go: so many that there are twice as many workgroups as run at once, two a CU, if that many have kLeastTiles
// tiles on average; and none where there are that many workgroups, or tiles take no longer than another launch.
inline int32_t splits_of(int64_t workgroups, int64_t tiles)
{
  int64_t const at_once = 2 * device_cus();
  if (workgroups >= at_once || workgroups <= 0 || tiles < 3 * kLeastTiles) return 1;
  return static_cast<int32_t>(std::min<int64_t>({(2 * at_once + workgroups - 1) / workgroups, tiles / kLeastTiles, 16}));
}

// Workgroups with something to do, and what they have, as far as the host knows: rows are taken to be alike.
struct Estimate {
  int64_t workgroups, tiles;
};
template <typename T>
Estimate estimate(Problem<T> const& p, Runs const& blocks, int32_t heads, int shift, Runs const& other, int tile, int64_t times)
{
  int64_t const rows = std::max(1, blocks.rows), length = (blocks.tokens + rows - 1) / rows;
  int64_t const seen = (other.tokens + rows - 1) / rows, tiles = (seen + tile - 1) / tile;
  // (causal, with as many tokens as keys: half of them on average)
  return {rows * ((length + (1 << shift) - 1) >> shift) * heads, (p.causal && other.tokens <= blocks.tokens ? (tiles + 1) / 2 : tiles) * times};
}

template <typename T, int D>
nvtext_amd_status attend_tiles(Forward<T> const& f, Mr const& mr, hipStream_t stream)
{
  using Shape      = ForwardShape<T, D, kTileWaves>;
  Estimate const e = estimate(f, f.runs, f.heads, Shape::kShift, f.key_runs, Shape::kTile, 1);
  Split split{splits_of(e.workgroups, e.tiles), nullptr, nullptr};
  size_t const rows = split.splits > 1 ? static_cast<size_t>(f.runs.blocks(Shape::kShift) * f.heads * split.splits) << Shape::kShift : 0;
  TempParts<2> const temp(mr, {rows * D * sizeof(float), rows * sizeof(float2)});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  split.sums = temp.template part<float>(0);
  split.tops = temp.template part<float2>(1);
  NVTEXT_HIP_TRY(allow_lds(attend_tiles_kernel<T, D, kTileWaves>, Shape::kLds));
  {
    ProfileScope const scope("attention_tiles", stream);
    int64_t const items = work_items(f.runs.blocks(Shape::kShift), f.kv_heads, f.heads / f.kv_heads, split.splits);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_tiles_kernel<T, D, kTileWaves>), grid_of(items, kTileWaves * kWave), dim3(kTileWaves * kWave), Shape::kLds, stream, f, split);
  }
  if (split.splits == 1) return NVTEXT_AMD_SUCCESS;
  ProfileScope const scope("attention_join", stream);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_join_shares_kernel<T, D>), grid_of((static_cast<int64_t>(f.runs.tokens) * f.heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f, split,
                     int{Shape::kShift});
  return NVTEXT_AMD_SUCCESS;
}

template <typename T, int D>
nvtext_amd_status attend_chunks(ForwardChunks<T> const& f, hipStream_t stream)
{
  constexpr int kLds = 4 * Tile<T, D>::kBytes;
  NVTEXT_HIP_TRY(allow_lds(attend_chunks_kernel<T, D>, kLds));
  {
    ProfileScope const scope("attention_chunks", stream);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_chunks_kernel<T, D>), grid_of(work_items(f.key_runs.blocks(f.shift), f.kv_heads, 1, 1), kWave), dim3(kWave), kLds, stream, f);
  }
  ProfileScope const scope("attention_join", stream);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_join_kernel<T, D>), grid_of(static_cast<int64_t>(f.runs.tokens) * f.heads, kJoinWaves * kWave), dim3(kJoinWaves * kWave), 0, stream, f);
  return NVTEXT_AMD_SUCCESS;
}

// calls f with the width of the tiles that heads of `width` values go through
template <typename F>
nvtext_amd_status with_tiles(int32_t width, F&& f)
{
  if (width <= 64) return f(std::integral_constant<int, 64>{});
  if (width <= 128) return f(std::integral_constant<int, 128>{});
  return f(std::integral_constant<int, 256>{});
}

template <typename T>
nvtext_amd_status attention(Forward<T> f, Mr const& mr, hipStream_t stream)
{
  Alignment<T> align(f.width);
  align.add(f.q, f.runs.tokens, f.heads);
  align.add(f.k, f.key_runs.tokens, f.kv_heads);
  align.add(f.v, f.key_runs.tokens, f.kv_heads);
  bool const chunks = f.runs.rows > 0 && static_cast<int64_t>(f.runs.tokens) * (f.heads / f.kv_heads) <= static_cast<int64_t>(f.runs.rows) * kPartColumns;
  int shift = 7;
  while (shift < 30 && (static_cast<int64_t>(f.key_runs.tokens) * f.kv_heads >> shift) > 2048) ++shift;
  return with_tiles(f.width, [&](auto d) {
    constexpr int kD        = decltype(d)::value;
    size_t const parts      = chunks ? static_cast<size_t>(most_parts(f.key_runs.tokens, shift)) * static_cast<size_t>(f.kv_heads) * kPartColumns : 0;
    TempParts<3> const temp(mr, {align.bytes(), parts * kD * sizeof(float), parts * sizeof(float2)});
    if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
    align.launch(temp.template part<char>(0), stream);
    if (chunks) return attend_chunks<T, kD>({f, shift, temp.template part<float>(1), temp.template part<float2>(2)}, stream);
    return attend_tiles<T, kD>(f, mr, stream);
  });
}

template <typename T, int D, Part PART>
nvtext_amd_status key_gradient_tiles(Backward<T> const& f, Split const& split, hipStream_t stream)
{
  using Shape = KeyShape<T, D, kTileWaves>;
  ProfileScope const scope("attention_key_gradient", stream);
  NVTEXT_HIP_TRY(allow_lds(key_gradient_tiles_kernel<T, D, kTileWaves, PART>, Shape::kLds));
  int64_t const items = work_items(f.key_runs.blocks(Shape::kShift), f.kv_heads, 1, split.splits);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(key_gradient_tiles_kernel<T, D, kTileWaves, PART>), grid_of(items, kTileWaves * kWave), dim3(kTileWaves * kWave), Shape::kLds, stream, f, split);
  return NVTEXT_AMD_SUCCESS;
}

template <typename T, int D>
nvtext_amd_status gradient_tiles(Backward<T> const& f, Mr const& mr, hipStream_t stream)
{
  using OfQ        = GradientShape<T, D, kTileWaves>;
  using OfK        = KeyShape<T, D, kTileWaves>;
  Estimate const q = estimate(f, f.runs, f.heads, OfQ::kShift, f.key_runs, OfQ::kTile, 1), k = estimate(f, f.key_runs, f.kv_heads, OfK::kShift, f.runs, OfK::kTile, f.heads / f.kv_heads);
  Split of_q{f.runs.tokens > 0 ? splits_of(q.workgroups, q.tiles) : 1, nullptr, nullptr}, of_k{f.key_runs.tokens > 0 ? splits_of(k.workgroups, k.tiles) : 1, nullptr, nullptr};
  TempParts<2> const temp(mr, {of_q.splits > 1 ? static_cast<size_t>(f.runs.blocks(OfQ::kShift) * f.heads * of_q.splits * OfQ::kRows * D) * sizeof(float) : 0,
                               of_k.splits > 1 ? static_cast<size_t>(f.key_runs.blocks(OfK::kShift) * f.kv_heads * of_k.splits * OfK::kRows * D) * 2 * sizeof(float) : 0});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  of_q.sums = temp.template part<float>(0);
  of_k.sums = temp.template part<float>(1);
  if (f.runs.tokens > 0) {
    ProfileScope const scope("attention_query_gradient", stream);
    NVTEXT_HIP_TRY(allow_lds(query_gradient_tiles_kernel<T, D, kTileWaves>, OfQ::kLds));
    int64_t const items = work_items(f.runs.blocks(OfQ::kShift), f.kv_heads, f.heads / f.kv_heads, of_q.splits);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(query_gradient_tiles_kernel<T, D, kTileWaves>), grid_of(items, kTileWaves * kWave), dim3(kTileWaves * kWave), OfQ::kLds, stream, f, of_q);
  }
  if (of_q.splits > 1) {
    ProfileScope const scope("attention_query_gradient_join", stream);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(query_gradient_join_kernel<T, D>), grid_of((static_cast<int64_t>(f.runs.tokens) * f.heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f, of_q,
                       int{OfQ::kShift});
  }
  if (f.key_runs.tokens == 0) return NVTEXT_AMD_SUCCESS;
  nvtext_amd_status st;
  if constexpr (D > 64) {
    st = key_gradient_tiles<T, D, kOfK>(f, of_k, stream);
    if (st == NVTEXT_AMD_SUCCESS) st = key_gradient_tiles<T, D, kOfV>(f, of_k, stream);
  } else {
    st = key_gradient_tiles<T, D, kBoth>(f, of_k, stream);
  }
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

// What both directions ask of their arguments; nullptr if it holds.
const char* bad_attention(const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, int32_t rows, const int32_t* offsets, const int32_t* key_offsets,
                          const int32_t* key_lengths, double scale)
{
  for (auto* x : {q, k, v})
    if (const char* bad = bad_heads(x)) return bad;
  if (k->type != q->type || v->type != q->type) return "q, k and v must be of one type";
  if (!is_like(v, k)) return "v must be of k's size";
  if (k->width != q->width) return "k and v must be of q's width";
  if (q->width > kMostWidth) return "heads may have 256 values at most";
  if (q->heads > 0 ? k->heads == 0 || q->heads % k->heads != 0 : k->heads != 0) return "the heads of k and v must be a divisor of q's";
  if (const char* bad = bad_rows(rows, offsets)) return bad;
  if (key_lengths && !key_offsets) return "key_lengths need key_offsets";
  if (!key_offsets && k->tokens != q->tokens) return "without offsets of their own, k and v must have q's tokens";
  if (!(scale >= 0) || !std::isfinite(static_cast<float>(scale))) return "scale must be finite and not negative";
  return nullptr;
}

template <typename T>
Problem<T> problem_of(const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, int32_t rows, const int32_t* offsets, const int32_t* key_offsets,
                      const int32_t* key_lengths, int32_t causal, double scale)
{
  return {heads_of<const T>(q), heads_of<const T>(k), heads_of<const T>(v), static_cast<int32_t>(q->heads), static_cast<int32_t>(k->heads), static_cast<int32_t>(q->width),
          Runs{offsets, rows, static_cast<int32_t>(q->tokens)}, Runs{key_offsets ? key_offsets : offsets, rows, static_cast<int32_t>(k->tokens)}, key_lengths, causal != 0,
          static_cast<float>(scale)};
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_attention(const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, int32_t rows, const int32_t* offsets, const int32_t* key_offsets,
                                       const int32_t* key_lengths, int32_t causal, double scale, void* stream_, const nvtext_amd_allocator* mr_, const nvtext_amd_heads* out, float* logsum,
                                       int8_t* rest)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_attention");
  if (!q || !k || !v || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_attention(q, k, v, rows, offsets, key_offsets, key_lengths, scale)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (const char* bad = bad_result(out)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (out->type != q->type || !is_like(out, q)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out must be of q's size and type");
  if (q->tokens == 0 || q->heads == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  with_type(q->type, [&](auto zero) {
    using T = decltype(zero);
    st      = attention<T>({problem_of<T>(q, k, v, rows, offsets, key_offsets, key_lengths, causal, scale), heads_of<T>(out), logsum, q->type == NVTEXT_AMD_TYPE_FLOAT32 ? nullptr : rest}, mr, stream);
  });
  if (st != NVTEXT_AMD_SUCCESS) return st;
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

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
  if (q->heads == 0 || (q->tokens == 0 && k->tokens == 0)) return NVTEXT_AMD_SUCCESS;
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
