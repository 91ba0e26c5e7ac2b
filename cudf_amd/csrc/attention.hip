// Attention of a row's tokens over its keys.
#include "attention.cuh"

namespace nvtext_amd {
namespace {

// Rows of few tokens go in chunks of keys, where all tokens and heads that share a key head are columns of one wavefront's products, the others in tiles:
// rows of at most kPartColumns columns, and, if they have the smallest chunk's keys or fewer, of kFewColumns.
constexpr int kPartColumns = 32, kFewColumns = 64, kFewKeys = 128;
template <typename T>
__device__ __forceinline__ bool goes_in_chunks(Forward<T> const& f, int32_t tokens, int32_t keys)
{
  if (!f.in_tiles || !f.in_chunks) return f.in_chunks;
  int64_t const columns = static_cast<int64_t>(tokens) * (f.heads / f.kv_heads);
  return columns <= kPartColumns || (columns <= kFewColumns && keys <= kFewKeys);
}

// ------------------------------------------------------------------ forward, in tiles
template <typename T, int D, int WAVES>
struct ForwardShape {
  static constexpr int kTokens = 32 * WAVES, kShift = __builtin_ctz(kTokens), kTile = kTileOf<T, D, WAVES>, kBytes = Tile<T, D, kTile>::kBytes, kLds = 4 * kBytes;
  static constexpr int kWavesASimd = D * sizeof(T) <= 128 ? 4 : D * sizeof(T) <= 256 ? 2 : 1;
};

// What a wavefront holds of 32 heads of tokens, columns of the products, while keys pass: q, and the sums of out, transposed.  Scores are products with the
// keys as rows, so a lane has all of a column's scores (with the one 32 further on), and exponentials are in its registers as the second product
// takes them: no lane needs another's but for the maximum.  Sums are kept in proportion to 2^top, where top is a maximum that may be 8 too small:
// only then are they multiplied anew.  In float16 top is 7 less, so that exponentials go up to 2^15 of the 65504 that it holds: its normal numbers end at 2^-14, and a weight is off by 2^-32 of
// the largest at most, where without these 7 a long row's many weights of less than 2^-25 were lost (131071 of 2^-24.4: 0.6 % of the sum, a third of it off).
template <typename T, int D, int TILE = Tile<T, D>::kHeads>
struct Attending {
  static constexpr int kSteps = D / 16, kColumns = D / 32, kTile = TILE, kBlocks = kTile / 32;
  static constexpr float kSlack = 8.f, kRoom = std::is_same_v<T, half_t> ? 7.f : 0.f;
  Fragment<T> q[kSteps];
  f32x16_t o[kColumns];
  float top, sum;
  float weight;  // (16-bit types) the sum of the exponentials as they are multiplied with v, rounded: what out is divided by, so that weights add up to 1
  int32_t seen;  // keys that the column sees

  __device__ __forceinline__ void begin(const T* head, int32_t width, bool there, int half)
  {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = fragment_of(head, 16 * s + 8 * half, width, there);
    top = -INFINITY;
    sum = weight = 0.f;
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
      stream<T, D, kSlots>([&](auto i) { return read.rows(k_tile, i / kSteps, i % kSteps); },
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
    high              = fmaf(fmaxf(both.low, both.high), scale, -kRoom);
    // (a column that sees nothing yet keeps top at -infinity; NaN in a score is found in out at the end)
    if (__ballot(high > top + kSlack || top == -INFINITY)) {
      float const now  = fmaxf(top, high);
      float const fade = now == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
      top              = now;
      sum *= fade;
      weight *= fade;
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
    auto const round = [&](int step) {
      p = rounded<T>(s[step / 2], step % 2);
      if constexpr (sizeof(T) == 2) weight = plus(weight, p);
    };
    stream<T, D, kRounds * kColumns>([&](auto i) { return read.columns(v_tile, i % kColumns, i / kColumns); },
                                  [&](auto i, Fragment<T> const& v) {
                                    constexpr int step = i / kColumns, c = i % kColumns;
                                    if constexpr (i == 0) {
#pragma unroll
                                      for (int e = 0; e < 8; ++e) exponential(0, e);
                                      round(0);
                                    }
                                    o[c] = multiply32(v, p, o[c]);
                                    if constexpr (step + 1 < kRounds) {
#pragma unroll
                                      for (int e = c * 8 / kColumns; e < (c + 1) * 8 / kColumns; ++e) exponential(step + 1, e);
                                      if constexpr (c == kColumns - 1) round(step + 1);
                                    }
                                  });
  }

  // what both lanes of a column have of a sum; what its o is divided by
  __device__ __forceinline__ static float whole(float part)
  {
    Halves const both = halves(part);
    return both.low + both.high;
  }
  __device__ __forceinline__ float divisor() const { return whole(sizeof(T) == 2 ? weight : sum); }

  // Writes out and logsum of a column, head h of token t, where it is `there`.  Returns the lanes' numbers of those whose result is not finite for keys that
  // they do not see, of which `border` says whether one is not finite: they are made once more, by themselves.  (NaN in a score makes NaN of the sum, and of all.)  A column that sees
  // nothing has zeros, whatever was added up.
  template <typename Border>
  __device__ __forceinline__ uint32_t finish(Forward<T> const& f, int64_t t, int32_t h, bool there, int half, int column, Border&& border)
  {
    float const total = whole(sum), part = 1.f / divisor();
    float check       = 0.f;  // (NaN if any is infinite or NaN)
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[c][r] = seen > 0 ? o[c][r] * part : 0.f;
        check   = fmaf(o[c][r], 0.f, check);
      }
    uint64_t odd = f.causal ? __ballot(there && check != 0.f && total == total) : 0;
    if (odd != 0 && !border()) odd = 0;
    odd = (odd | odd >> 32) & 0xffffffffu;
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

// A workgroup has kTokens tokens of a head, a wavefront 32 of them.  Keys come through LDS, 64 at a time, the next ones while these are multiplied.  Four
// wavefronts share a tile: with eight, and with two, prompts and short texts are slower.
// Of wide 16-bit heads bound by the matrix cores and the vector instructions of the exponentials in turn (32768 tokens in six rows, 32 heads of 128 over 8,
// bfloat16: 1.67 ms, 1.0 PFLOP/s; matrix cores busy for 54 % of the time, vector instructions 55, LDS 27 and without conflicts); of short rows by
// what a workgroup does once (512011 tokens in 4001 rows, 16 heads of 64: 1.33 ms, 3.2 TB/s, half of the columns and keys of its tiles are there); of
// float32 by the matrix cores and the last workgroups (8191 tokens in 61 rows, 12 heads of 64: 149 us, matrix cores 29 %).
template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave, (ForwardShape<T, D, WAVES>::kWavesASimd)) attend_tiles_kernel(Forward<T> f, Split split)
{
  using Shape = ForwardShape<T, D, WAVES>;
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds  = (LdsBytes)lds_;
  constexpr int kTile = Shape::kTile, kStage = 2 * Shape::kBytes;
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
  if (goes_in_chunks(f, tokens, keys)) return;
  // keys that the workgroup's last token sees, and the wavefront's first and last
  int32_t const wave0 = wave * 32, wave1 = wave0 + 32 < rest ? wave0 + 32 : rest;
  int32_t const all   = uniform(f.seen(block0 + (rest < Shape::kTokens ? rest : Shape::kTokens) - 1, tokens, keys));
  int32_t const least = uniform(wave0 < rest ? f.seen(block0 + wave0, tokens, keys) : 0), most = uniform(wave0 < rest ? f.seen(block0 + wave1 - 1, tokens, keys) : 0);
  bool const there    = wave0 + column < rest;
  int64_t const t     = static_cast<int64_t>(begin) + block0 + (there ? wave0 + column : 0);

  int32_t const all_tiles = (all + kTile - 1) / kTile, shares = shares_of(all_tiles, split.splits);
  if (w.share >= shares) return;
  int32_t const from = uniform(share_begin(all_tiles, w.share, shares)), tiles = uniform(share_begin(all_tiles, w.share + 1, shares));

  Attending<T, D, kTile> a;
  a.seen = there ? f.seen(block0 + wave0 + column, tokens, keys) : 0;
  a.begin(f.q.at(t, w.head), f.width, there, half);
  TileLoader<T, D, WAVES, kTile> load_k, load_v;
  load_k.aim(f.k, first + from * kTile, w.kv_head, f.width, wave, lane);
  load_v.aim(f.v, first + from * kTile, w.kv_head, f.width, wave, lane);
  auto const load = [&](int32_t tile) {
    LdsBytes const to = lds + (tile & 1) * kStage;
    load_k.load(to, keys - tile * kTile, wave);
    load_v.load(to + Shape::kBytes, keys - tile * kTile, wave);
  };
  TileReader<T, D> const read(lane);
  float const scale = f.exponent_scale();
  if (tiles > from) load(from);
  for (int32_t tile = from; tile < tiles; ++tile) {
    LdsBytes const k_tile = lds + (tile & 1) * kStage;
    stage_barrier<0>();
    if (tile + 1 < tiles) load(tile + 1);
    int32_t const key0 = tile * kTile;
    if (key0 < most) a.pass(k_tile, k_tile + Shape::kBytes, read, key0, key0 + kTile > least, scale, half);
  }
  if (wave0 >= rest) return;
  if (shares > 1) {
    int64_t const part = split.slot(w.block, w.head, f.heads, w.share) * Shape::kTokens + wave0 + column;
    float const total = a.whole(a.sum), divisor = a.divisor();
    if (there) {
      store_columns<float, D / 32>(split.sums + part * D, a.o, half, D);
      if (half == 0) split.tops[part] = make_float4(a.top, total, divisor, 0.f);
    }
    return;
  }
  uint32_t odd = a.finish(f, t, w.head, there, half, column, [&] {
    int32_t const loaded = (most + kTile - 1) / kTile * kTile;
    return holds_odd(f.v, static_cast<int64_t>(first) + least, (loaded < keys ? loaded : keys) - least, w.kv_head, f.width);
  });
  for (; odd; odd &= odd - 1) attend_row(f, begin + block0 + wave0 + __builtin_ctz(odd), w.head);
}

// ------------------------------------------------------------------ forward, in chunks of keys
// Few tokens a row, as where texts go on token by token: one wavefront has all of a row's tokens and of all heads that share a key head, up to 32 together,
// as the columns of its products, and a chunk of 2^shift of the row's keys; what it adds up is joined with that of the row's other chunks by another
// launch.  Bound by memory: the keys are read once (24 rows of one token over 1501 keys on average, 32 heads of 128 over 8: 35 us, 4.2 TB/s, and 6 for the join; one token over
// 131071: 100 us, 5.4 TB/s, and 11).  Tiles of 32 keys, so that a CU has room for five workgroups of heads of 128: 35 and 100 us where 64 take 40 and 102.  The chunks of key tokens are numbered as the blocks of tokens are elsewhere, so they are
// alike in size however long the rows are.  A row of a single chunk is finished at once; so is one of more columns, 32 of them after the other by each of
// the workgroups that its chunks have.
// Parts of a row of several chunks lie from number 2 * first / 2^shift on: it has at least half as many numbers up to the next row's as it has chunks.
constexpr int kChunkTile = 32;
template <typename T>
struct ForwardChunks : Forward<T> {
  float* sums;    // [part][key head][column][D]
  float4* tops;   // [part][key head][column]: top, the sum of the exponentials, and what out is divided by
  __device__ __forceinline__ int64_t part(int32_t first, int32_t chunk, int32_t kv_head) const
  {
    return ((static_cast<int64_t>(first) * 2 >> this->shift) + chunk) * this->kv_heads + kv_head;
  }
  __device__ __forceinline__ int32_t chunks_of(int32_t keys) const { return keys > 0 ? ((keys - 1) >> this->shift) + 1 : 1; }
  __device__ __forceinline__ bool is_split(int32_t tokens, int32_t chunks) const { return chunks > 1 && static_cast<int64_t>(tokens) * (this->heads / this->kv_heads) <= kPartColumns; }
};
inline int64_t most_parts(int64_t key_tokens, int shift) { return (key_tokens * 2 >> shift) + 2; }

template <typename T, int D>
__global__ void __launch_bounds__(kWave, 1) attend_chunks_kernel(ForwardChunks<T> f)
{
  extern __shared__ __align__(16) char lds_[];
  LdsBytes const lds  = (LdsBytes)lds_;
  constexpr int kTile = kChunkTile, kBytes = Tile<T, D, kTile>::kBytes;
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
  if (chunk >= chunks || !goes_in_chunks<T>(f, tokens, keys)) return;
  int const lane = lane_id(), column = lane % 32, half = lane / 32;
  int32_t const key_first = split ? static_cast<int32_t>(chunk << f.shift) : 0, key_last = split && keys - key_first > 1 << f.shift ? key_first + (1 << f.shift) : keys;
  int64_t const columns   = static_cast<int64_t>(tokens > 0 ? tokens : 0) * each;
  TileReader<T, D> const read(lane);
  float const scale = f.exponent_scale();
  for (int64_t column0 = split ? 0 : chunk * kPartColumns; column0 < columns; column0 += split ? columns : static_cast<int64_t>(chunks) * kPartColumns) {
    int64_t const mine = column0 + column;
    bool const there   = mine < columns;
    int32_t const i    = there ? static_cast<int32_t>(mine / each) : 0, head = w.kv_head * each + (there ? static_cast<int32_t>(mine - static_cast<int64_t>(i) * each) : 0);
    int64_t const t    = static_cast<int64_t>(begin) + i;
    int32_t const last = static_cast<int32_t>(((column0 + kPartColumns < columns ? column0 + kPartColumns : columns) - 1) / each);  // the last column's token
    Attending<T, D, kTile> a;
    a.seen = there ? f.seen(i, tokens, keys) : 0;
    a.begin(f.q.at(t, head), f.width, there, half);
    int32_t const least = uniform(f.seen(static_cast<int32_t>(column0 / each), tokens, keys)), all = uniform(f.seen(last, tokens, keys)), end = all < key_last ? all : key_last;
    int32_t const tiles = end > key_first ? (end - key_first + kTile - 1) / kTile : 0;
    TileLoader<T, D, 1, kTile> load_k, load_v;
    load_k.aim(f.k, first + key_first, w.kv_head, f.width, 0, lane);
    load_v.aim(f.v, first + key_first, w.kv_head, f.width, 0, lane);
    if (tiles > 0) {
      load_k.load(lds, key_last - key_first, 0);
      load_v.load(lds + kBytes, key_last - key_first, 0);
    }
    for (int32_t tile = 0; tile < tiles; ++tile) {
      LdsBytes const k_tile = lds + (tile & 1) * 2 * kBytes;
      int32_t const key0    = key_first + tile * kTile;
      stage_barrier<0>();
      if (tile + 1 < tiles) {
        LdsBytes const next = lds + (~tile & 1) * 2 * kBytes;
        load_k.load(next, key_last - key0 - kTile, 0);
        load_v.load(next + kBytes, key_last - key0 - kTile, 0);
      }
      a.pass(k_tile, k_tile + kBytes, read, key0, key0 + kTile > least || key0 + kTile > key_last, scale, half);
    }
    stage_barrier<0>();  // (the next columns' loads come into the same places)
    if (split) {
      int64_t const part = f.part(first, static_cast<int32_t>(chunk), w.kv_head) * kPartColumns + column;
      float const total = a.whole(a.sum), divisor = a.divisor();
      if (there) {
        store_columns<float, D / 32>(f.sums + part * D, a.o, half, D);
        if (half == 0) f.tops[part] = make_float4(a.top, total, divisor, 0.f);
      }
      continue;
    }
    auto const border = [&] {
      int32_t const loaded = tiles * kTile;  // (from the first key on: what is not split is a whole row)
      return holds_odd(f.v, static_cast<int64_t>(first) + least, (loaded < keys ? loaded : keys) - least, w.kv_head, f.width);
    };
    for (uint32_t odd = a.finish(f, t, head, there, half, column, border); odd; odd &= odd - 1) {
      int const which = __builtin_ctz(odd);
      attend_row(f, __builtin_amdgcn_readlane(static_cast<int32_t>(t), which), __builtin_amdgcn_readlane(head, which));
    }
  }
}

template <int D>
__device__ __forceinline__ void add_part(Some<D>& sum, float2& total, float top, float4 of, const float* part)
{
  float const weight = of.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(of.x - top);
  total.x += of.y * weight;
  total.y += of.z * weight;
  sum.add(part, weight);
}

// What Attending::finish does, for sums that a wavefront holds side by side; `border`: keys behind those that the token sees, which lie from `first` on, that have been multiplied as well.
template <typename T, int D>
__device__ __forceinline__ void finish_row(Forward<T> const& f, int32_t t, int32_t head, int32_t first, int32_t seen, int32_t border, Some<D> sum, float2 total, float top)
{
#pragma unroll
  for (int k = 0; k < Some<D>::kEach; ++k) sum.v[k] = seen > 0 ? sum.v[k] / total.y : 0.f;
  if (f.causal && total.x == total.x && !sum.finite(f.width) && holds_odd(f.v, static_cast<int64_t>(first) + seen, border, head / (f.heads / f.kv_heads), f.width)) {
    attend_row(f, t, head);
    return;
  }
  T* const out     = f.out.at(t, head);
  int64_t const at = static_cast<int64_t>(head) * f.runs.tokens + t;
#pragma unroll
  for (int k = 0; k < Some<D>::kEach; ++k) {
    int32_t const j = sum.first() + k;
    if (j < f.width) {
      out[j] = static_cast<T>(sum.v[k]);
      if (f.rest) f.rest[at * f.width + j] = rest_of(sum.v[k], static_cast<T>(sum.v[k]));
    }
  }
  if (f.logsum && lane_id() == 0) f.logsum[at] = seen > 0 ? (top + __builtin_amdgcn_logf(total.x)) * kLn2 : -INFINITY;
}

// Joins the parts of a head of a row's tokens, a workgroup for every `apart`th token, whose wavefronts take the parts in turn.
template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave) attend_join_kernel(ForwardChunks<T> f, int32_t apart)
{
  __shared__ float tops[WAVES];
  __shared__ float2 totals[WAVES];
  __shared__ float sums_[WAVES * kWave * Some<D>::kEach];
  auto const sums    = reinterpret_cast<Some<D>(*)[kWave]>(sums_);
  int64_t const item = block_number(), of_row = static_cast<int64_t>(f.heads) * apart;
  if (item >= f.runs.rows * of_row) return;
  int32_t const row = static_cast<int32_t>(item / of_row), head = static_cast<int32_t>(item - row * of_row) / apart, run = row + 1;
  int32_t first, keys;
  f.keys_of(run, first, keys);
  int32_t const begin = f.runs.begin(run), tokens = f.runs.begin(run + 1) - begin, chunks = f.chunks_of(keys), each = f.heads / f.kv_heads;
  if (!f.is_split(tokens, chunks)) return;  // (what is split goes in chunks)
  int const wave     = threadIdx.x / kWave, lane = lane_id();
  int64_t const step = static_cast<int64_t>(f.kv_heads) * kPartColumns;
  for (int32_t i = static_cast<int32_t>(item % apart); i < tokens; i += apart) {
    int64_t const at = f.part(first, 0, head / each) * kPartColumns + i * each + head % each;
    float top        = -INFINITY;
    for (int32_t c = threadIdx.x; c < chunks; c += WAVES * kWave) top = fmaxf(top, f.tops[at + c * step].x);
    top = wave_max(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
    float2 total{};
    Some<D> sum{};
#pragma unroll 8
    for (int32_t c = wave; c < chunks; c += WAVES) add_part<D>(sum, total, top, f.tops[at + c * step], f.sums + (at + c * step) * D);
    sums[wave][lane] = sum;
    if (lane == 0) totals[wave] = total;
    __syncthreads();
    if (wave != 0) continue;  // (they write totals and sums again behind the next token's first barrier)
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      total.x += totals[w].x;
      total.y += totals[w].y;
#pragma unroll
      for (int k = 0; k < Some<D>::kEach; ++k) sum.v[k] += sums[w][lane].v[k];
    }
    int32_t const seen = f.seen(i, tokens, keys);
    finish_row<T, D>(f, begin + i, head, first, seen, keys - seen, sum, total, top);
  }
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
  if (goes_in_chunks(f, tokens, keys)) return;
  int32_t const all = f.seen(last < tokens ? last : tokens - 1, tokens, keys), shares = shares_of((all + kTile - 1) / kTile, split.splits);
  if (shares < 2) return;
  int64_t const at = (split.slot(f.runs.first_block(run, shift) + (i >> shift), head, f.heads, 0) << shift) + (i & ((1 << shift) - 1));
  // (at most kMostShares shares: a lane has the sums of one)
  float4 const mine  = lane_id() < shares ? split.tops[at + (static_cast<int64_t>(lane_id()) << shift)] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
  float const top    = wave_max(mine.x), weight = mine.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine.x - top);
  float2 const total = make_float2(wave_sum(mine.y * weight), wave_sum(mine.z * weight));
  Some<D> sum{};
#pragma unroll 8
  for (int32_t c = 0; c < shares; ++c) sum.add(split.sums + (at + (static_cast<int64_t>(c) << shift)) * D, __shfl(weight, c));
  int32_t const seen = f.seen(i, tokens, keys), loaded = (all + kTile - 1) / kTile * kTile;
  finish_row<T, D>(f, t, head, first, seen, (loaded < keys ? loaded : keys) - seen, sum, total, top);
}

// ------------------------------------------------------------------ launches
template <typename T, int D, int WAVES>
nvtext_amd_status launch_tiles(Forward<T> const& f, Split const& split, hipStream_t stream)
{
  using Shape = ForwardShape<T, D, WAVES>;
  ProfileScope const scope("attention_tiles", stream);
  NVTEXT_HIP_TRY(allow_lds(attend_tiles_kernel<T, D, WAVES>, Shape::kLds));
  int64_t const items = work_items(f.runs.blocks(Shape::kShift), f.kv_heads, f.heads / f.kv_heads, split.splits);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_tiles_kernel<T, D, WAVES>), grid_of(items, WAVES * kWave), dim3(WAVES * kWave), Shape::kLds, stream, f, split);
  return NVTEXT_AMD_SUCCESS;
}

template <typename T, int D>
nvtext_amd_status attend_tiles(Forward<T> const& f, Mr const& mr, hipStream_t stream)
{
  using Shape = ForwardShape<T, D, kTileWaves>;
  Split split{splits_of<T, D, 2>(f, f.runs, f.heads, Shape::kShift, f.key_runs, 1, Shape::kLds), nullptr, nullptr};
  size_t const rows = split.splits > 1 ? static_cast<size_t>(f.runs.blocks(Shape::kShift) * f.heads * split.splits) << Shape::kShift : 0;
  TempParts<2> const temp(mr, {rows * D * sizeof(float), rows * sizeof(float4)});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  split.sums = temp.template part<float>(0);
  split.tops = temp.template part<float4>(1);
  if (split.splits == 1) return is_short(f) ? launch_tiles<T, D, 1>(f, split, stream) : launch_tiles<T, D, kTileWaves>(f, split, stream);
  nvtext_amd_status const st = launch_tiles<T, D, kTileWaves>(f, split, stream);
  if (st != NVTEXT_AMD_SUCCESS) return st;
  ProfileScope const scope("attention_join", stream);
  hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_join_shares_kernel<T, D>), grid_of((static_cast<int64_t>(f.runs.tokens) * f.heads + 3) / 4, kThreads), dim3(kThreads), 0, stream, f, split,
                     int{Shape::kShift});
  return NVTEXT_AMD_SUCCESS;
}

template <typename T, int D>
nvtext_amd_status attend_chunks(ForwardChunks<T> const& f, hipStream_t stream)
{
  constexpr int kLds = 4 * Tile<T, D, kChunkTile>::kBytes;
  NVTEXT_HIP_TRY(allow_lds(attend_chunks_kernel<T, D>, kLds));
  {
    ProfileScope const scope("attention_chunks", stream);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_chunks_kernel<T, D>), grid_of(work_items(f.key_runs.blocks(f.shift), f.kv_heads, 1, 1), kWave), dim3(kWave), kLds, stream, f);
  }
  // A row that sees its own tokens has a single chunk.
  if (f.own_keys()) return NVTEXT_AMD_SUCCESS;
  // As many workgroups a head of a row as it has tokens on average, and no more than one that is split can have, nor than one where rows have a chunk on average.
  int64_t const rows = f.runs.rows, tokens = (f.runs.tokens + rows - 1) / rows, most = rows << f.shift < f.key_runs.tokens ? std::max(1, kPartColumns / (f.heads / f.kv_heads)) : 1;
  int32_t const apart = static_cast<int32_t>(std::clamp<int64_t>(tokens, 1, most));
  int64_t const items = rows * f.heads * apart;
  ProfileScope const scope("attention_join", stream);
  auto const join = [&](auto waves) {
    constexpr int kWaves = decltype(waves)::value;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_join_kernel<T, D, kWaves>), grid_of(items, kWaves * kWave), dim3(kWaves * kWave), 0, stream, f, apart);
  };
  // (where there are fewer than CUs, a row's parts are many: 1 row of 131,071 keys, 32 heads 18.8 us with 4 wavefronts)
  if (items < device_cus())
    join(std::integral_constant<int, 16>{});
  else
    join(std::integral_constant<int, 4>{});
  return NVTEXT_AMD_SUCCESS;
}

template <typename T>
nvtext_amd_status attention(Forward<T> f, Mr const& mr, hipStream_t stream)
{
  Alignment<T> align(f.width);
  align.add(f.q, f.runs.tokens, f.heads);
  align.add(f.k, f.key_runs.tokens, f.kv_heads);
  align.add(f.v, f.key_runs.tokens, f.kv_heads);
  // By what rows have on average; where there are more tokens than rows, some may have many all the same.  Rows that see their own tokens go in chunks
  // where four heads or more share keys: 1000 rows of 12 tokens, 16 heads of 128 over 4 of keys, 100 us in tiles, 92 in both; of 20 tokens, 16 heads of 64 over 8, 54
  // and 71.
  int64_t const columns = static_cast<int64_t>(f.runs.tokens) * (f.heads / f.kv_heads), rows = f.runs.rows;
  f.in_chunks           = rows > 0 && (f.own_keys() ? f.heads >= 4 * static_cast<int64_t>(f.kv_heads) && columns <= rows * kFewColumns : columns <= rows * kPartColumns);
  f.in_tiles            = !f.in_chunks || f.runs.tokens > rows;
  f.shift               = 7;
  while (f.shift < 30 && (static_cast<int64_t>(f.key_runs.tokens) * f.kv_heads >> f.shift) > 2048) ++f.shift;
  return with_tiles(f.width, [&](auto d) {
    constexpr int kD        = decltype(d)::value;
    // (rows over their own keys have one chunk each, or are not split)
    size_t const parts      = f.in_chunks && !f.own_keys() ? static_cast<size_t>(most_parts(f.key_runs.tokens, f.shift)) * static_cast<size_t>(f.kv_heads) * kPartColumns : 0;
    TempParts<3> const temp(mr, {align.bytes(), parts * kD * sizeof(float), parts * sizeof(float4)});
    if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
    align.launch(temp.template part<char>(0), stream);
    nvtext_amd_status const st = f.in_chunks ? attend_chunks<T, kD>({f, temp.template part<float>(1), temp.template part<float4>(2)}, stream) : NVTEXT_AMD_SUCCESS;
    return st == NVTEXT_AMD_SUCCESS && f.in_tiles ? attend_tiles<T, kD>(f, mr, stream) : st;
  });
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
  if (q->tokens == 0 || q->heads == 0 || (q->width == 0 && !logsum)) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  nvtext_amd_status st = NVTEXT_AMD_SUCCESS;
  with_type(q->type, [&](auto zero) {
    using T = decltype(zero);
    st      = attention<T>({problem_of<T>(q, k, v, rows, offsets, key_offsets, key_lengths, causal, scale), heads_of<T>(out), logsum, q->type == NVTEXT_AMD_TYPE_FLOAT32 ? nullptr : rest, true, false, 0}, mr, stream);
  });
  if (st != NVTEXT_AMD_SUCCESS) return st;
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
