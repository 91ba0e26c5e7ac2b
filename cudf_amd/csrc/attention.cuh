// Shared by attention and its gradient: what the kernels are given, the formulas a row at a time, and tiles of keys in LDS.
#pragma once

#include "heads.cuh"
#include "matrix.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace nvtext_amd {

constexpr int kMostWidth  = 256, kMostHeads = 65536, kMostTokens = INT32_MAX - 1024;
constexpr float kLog2e    = 1.4426950408889634f;
constexpr float kLn2      = 0.6931471805599453f;

// What the kernels of both directions are given.
template <typename T>
struct Problem {
  Heads<const T> q, k, v;
  int32_t heads, kv_heads, width;
  Runs runs, key_runs;
  const int32_t* key_lengths;
  bool causal;
  float scale;

  // What the tiles multiply a score with for an exponent of 2: at least the smallest number there is, which changes no exponent by more than 2^-21 and leaves the -infinity of a masked
  // one what it is; a scale of 0 would make it NaN.
  __device__ __forceinline__ float exponent_scale() const { return fmaxf(scale * kLog2e, 0x1p-149f); }
  // whether keys are those of the tokens themselves, all of them
  bool own_keys() const { return key_runs.offsets == runs.offsets && key_runs.tokens == runs.tokens && !key_lengths; }
  // The keys of run `i` (a row's), of which there are `length`, from token `first` on.
  __device__ __forceinline__ void keys_of(int32_t i, int32_t& first, int32_t& length) const
  {
    first  = key_runs.begin(i);
    length = key_runs.begin(i + 1) - first;
    if (key_lengths) {
      int32_t const l = key_lengths[i - 1];
      length          = l < length ? l : length;
    }
    length = length > 0 ? length : 0;
  }
  __device__ __forceinline__ bool is_row(int32_t i) const { return i > 0 && i <= runs.rows; }
  // How many keys token `i` of a row of `tokens` sees, of `keys`.
  __device__ __forceinline__ int32_t seen(int32_t i, int32_t tokens, int32_t keys) const
  {
    int64_t const n = causal ? static_cast<int64_t>(i) + 1 + keys - tokens : keys;
    return static_cast<int32_t>(n < 0 ? 0 : n < keys ? n : keys);
  }
};

// ------------------------------------------------------------------ a row at a time
// The formulas as they stand, a wavefront for a token and a head, 64 keys at a time: a lane for a key in the scores, a lane for a column in the
// sums.  Nothing that a token does not see is multiplied by anything: the tiles multiply it by 0, which makes NaN of an infinity or NaN.  A row takes some hundred times as long as in a tile,
// so one is only made again where its sums are not finite and need not be so for what it sees, and where something that it does not see, at the border between what the block's
// tokens see and what they do not, is not finite.  (Without `causal` there is no such border.)  A step over 8192 tokens, 32 heads of 128 over 8, causal, bfloat16, takes 2.7 ms, and 4.7 to 6.9 with
// NaN in one token's k or v, in a late token's gradient, or everywhere, where it took 1.5 to 2.8 s with all rows made again; with NaN in an early q, whose block's
// other 31 keys are made again over all tokens, 32.  Values or gradients that are not finite here and there in nearly every block of tokens still take as long as rows do: 0.4 s forward
// and 1.4 s back, one in 1000 infinite.

template <typename T>
__device__ __forceinline__ float dot(const T* a, const T* b, int32_t width)
{
  float sum = 0.f;
  for (int32_t j = 0; j < width; ++j) sum = fmaf(static_cast<float>(a[j]), static_cast<float>(b[j]), sum);
  return sum;
}

__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
  for (int by = 32; by > 0; by /= 2) v = fmaxf(v, __shfl_xor(v, by));
  return v;
}

// What rounding to a 16-bit type leaves off, in 8 bits more: the difference of the two values' bits as float32, in 2^-8 of a step of the type.  (Signs
// are alike, so bits differ as values do; zeros and the smallest numbers, whose steps are others, get what 8 bits hold of it, and
// beside an infinity they are of no meaning.)  With them a sum of products
// with out is as good as one with out in float32 for what is rounded to 16 bits afterwards.
template <typename T>
__device__ __forceinline__ int8_t rest_of(float x, T rounded)
{
  constexpr int kShift = sizeof(T) == 4 ? 0 : std::is_same_v<T, half_t> ? 5 : 8;
  int32_t const off    = (__builtin_bit_cast(int32_t, x) - __builtin_bit_cast(int32_t, static_cast<float>(rounded)) + (1 << kShift >> 1)) >> kShift;
  return static_cast<int8_t>(off < -127 ? -127 : off > 127 ? 127 : off);
}
template <typename T>
__device__ __forceinline__ float with_rest(T rounded, int32_t rest)
{
  constexpr int kShift = std::is_same_v<T, half_t> ? 5 : 8;
  return __builtin_bit_cast(float, __builtin_bit_cast(int32_t, static_cast<float>(rounded)) + rest * (1 << kShift));
}

// Whether one of `count` heads from token `first` on holds an infinity or NaN, for the whole wavefront.
template <typename T>
__device__ __forceinline__ bool holds_odd(Heads<const T> const& x, int64_t first, int32_t count, int32_t head, int32_t width)
{
  float check = 0.f;
#pragma unroll 1
  for (int32_t i = lane_id(); i < count * width; i += kWave) check = fmaf(static_cast<float>(x.at(first + i / width, head)[i % width]), 0.f, check);
  return __ballot(check != 0.f) != 0;
}

template <typename T>
struct Forward : Problem<T> {
  Heads<T> out;
  float* logsum;
  int8_t* rest;  // [heads, tokens, width], of 16-bit types; or nullptr
  // Which launches there are; and of the one in chunks, that a chunk has 2^shift keys.
  bool in_tiles, in_chunks;
  int32_t shift;
};

// The run that token t is in, the same in all lanes of the (whole) wavefront, which look at 64 runs at once as in Runs::run_of().
__device__ __forceinline__ int32_t run_with(Runs const& runs, int32_t t)
{
  int32_t lo = 0, count = runs.rows + 2;
  while (count > 1) {
    int32_t const each = (count + kWave - 1) / kWave;
    int32_t const i    = lane_id() * each;
    uint64_t const all = __ballot(i < count && runs.begin(lo + i) <= t) | 1;
    int32_t const last = 63 - __clzll(static_cast<long long>(all));
    lo += last * each;
    count = count - last * each < each ? count - last * each : each;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

template <typename T>
__device__ void attend_row(Forward<T> const& f, int32_t t, int32_t h)
{
  int const lane    = lane_id();
  int32_t const run = run_with(f.runs, t);
  int32_t first = 0, keys = 0, seen = 0;
  if (f.is_row(run)) {
    f.keys_of(run, first, keys);
    seen = f.seen(t - f.runs.begin(run), f.runs.begin(run + 1) - f.runs.begin(run), keys);
  }
  int32_t const kh   = h / (f.heads / f.kv_heads);
  float const scale  = f.scale * kLog2e;
  const T* const q   = f.q.at(t, h);
  float top = -INFINITY, sum = 0.f, o[kMostWidth / kWave] = {};
  for (int32_t base = 0; base < seen; base += kWave) {
    int32_t const n = seen - base < kWave ? seen - base : kWave;
    float const s   = lane < n ? dot(q, f.k.at(first + base + lane, kh), f.width) * scale : -INFINITY;
    float const now = fmaxf(top, wave_max(s)), level = now == -INFINITY ? 0.f : now;  // (keys of no weight in front of others are no reason for NaN)
    float const p   = lane < n ? __builtin_amdgcn_exp2f(s - level) : 0.f, fade = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
    sum = sum * fade + wave_sum(p);
#pragma unroll
    for (int c = 0; c < kMostWidth / kWave; ++c) o[c] *= fade;
    for (int32_t j = 0; j < n; ++j) {
      float const pj = __shfl(p, j);
#pragma unroll
      for (int c = 0; c < kMostWidth / kWave; ++c)
        if (c * kWave + lane < f.width) o[c] = fmaf(pj, static_cast<float>(f.v.at(first + base + j, kh)[c * kWave + lane]), o[c]);
    }
    top = now;
  }
#pragma unroll
  for (int c = 0; c < kMostWidth / kWave; ++c)
    if (c * kWave + lane < f.width) {
      float const x                      = seen > 0 ? o[c] / sum : 0.f;
      f.out.at(t, h)[c * kWave + lane] = static_cast<T>(x);
      if (f.rest) f.rest[(static_cast<int64_t>(h) * f.runs.tokens + t) * f.width + c * kWave + lane] = rest_of(x, static_cast<T>(x));
    }
  if (f.logsum && lane == 0) f.logsum[static_cast<int64_t>(h) * f.runs.tokens + t] = seen > 0 ? (top + __builtin_amdgcn_logf(sum)) * kLn2 : -INFINITY;
}

template <typename T>
struct Backward : Problem<T> {
  Heads<const T> grad, out;
  const float* logsum;
  const int8_t* rest;  // out's, or nullptr
  float* deltas;  // [heads, tokens]: grad . out
  float* logs;    // [heads, tokens]: logsum in powers of 2, as the tiles of k's and v's gradients take it
  Heads<T> q_grad, k_grad, v_grad;
};

// The gradient of token t's head h of q, and its delta.
template <typename T>
__device__ void query_gradient_row(Backward<T> const& f, int32_t t, int32_t h)
{
  int const lane    = lane_id();
  int32_t const run = run_with(f.runs, t);
  int32_t first = 0, keys = 0, seen = 0;
  if (f.is_row(run)) {
    f.keys_of(run, first, keys);
    seen = f.seen(t - f.runs.begin(run), f.runs.begin(run + 1) - f.runs.begin(run), keys);
  }
  int32_t const kh = h / (f.heads / f.kv_heads);
  const T *const q = f.q.at(t, h), *const g = f.grad.at(t, h);
  int64_t const at  = static_cast<int64_t>(h) * f.runs.tokens + t;
  float const log   = f.logsum[at] * kLog2e, scale = f.scale * kLog2e;
  float delta       = 0.f;
  if (seen > 0 && f.rest) {
    for (int32_t j = 0; j < f.width; ++j)
      delta = fmaf(static_cast<float>(g[j]), with_rest(f.out.at(t, h)[j], f.rest[at * f.width + j]), delta);
  } else if (seen > 0) {
    delta = dot(g, f.out.at(t, h), f.width);
  }
  if (lane == 0) f.deltas[at] = delta;
  float d[kMostWidth / kWave] = {};
  for (int32_t base = 0; base < seen; base += kWave) {
    int32_t const n = seen - base < kWave ? seen - base : kWave;
    float ds        = 0.f;
    if (lane < n) {
      float const p = __builtin_amdgcn_exp2f(dot(q, f.k.at(first + base + lane, kh), f.width) * scale - log);
      ds            = p * (dot(g, f.v.at(first + base + lane, kh), f.width) - delta) * f.scale;
    }
    for (int32_t j = 0; j < n; ++j) {
      float const dj = __shfl(ds, j);
#pragma unroll
      for (int c = 0; c < kMostWidth / kWave; ++c)
        if (c * kWave + lane < f.width) d[c] = fmaf(dj, static_cast<float>(f.k.at(first + base + j, kh)[c * kWave + lane]), d[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kMostWidth / kWave; ++c)
    if (c * kWave + lane < f.width) f.q_grad.at(t, h)[c * kWave + lane] = static_cast<T>(d[c]);
}

// The gradients of key token t's head kh of k and v, those that are wanted.
template <typename T>
__device__ void key_gradient_row(Backward<T> const& f, int32_t t, int32_t kh, bool of_k, bool of_v)
{
  int const lane    = lane_id();
  int32_t const run = run_with(f.key_runs, t), each = f.heads / f.kv_heads;
  float dk[kMostWidth / kWave] = {}, dv[kMostWidth / kWave] = {};
  int32_t first = 0, keys = 0;
  if (f.is_row(run)) f.keys_of(run, first, keys);
  int32_t const j = t - first;
  if (f.is_row(run) && j < keys) {
    int32_t const begin = f.runs.begin(run), tokens = f.runs.begin(run + 1) - begin;
    // token i sees key j from i = j + tokens - keys on
    int64_t const from = f.causal ? static_cast<int64_t>(j) + tokens - keys : 0;
    const T *const k = f.k.at(t, kh), *const v = f.v.at(t, kh);
    float const scale = f.scale * kLog2e;
    for (int32_t h = kh * each; h < (kh + 1) * each; ++h) {
      for (int64_t base = from < 0 ? 0 : from; base < tokens; base += kWave) {
        int32_t const n = static_cast<int32_t>(tokens - base < kWave ? tokens - base : kWave), token = static_cast<int32_t>(begin + base);
        float p = 0.f, ds = 0.f;
        if (lane < n) {
          int64_t const at = static_cast<int64_t>(h) * f.runs.tokens + token + lane;
          p                = __builtin_amdgcn_exp2f(dot(f.q.at(token + lane, h), k, f.width) * scale - f.logsum[at] * kLog2e);
          ds               = p * (dot(f.grad.at(token + lane, h), v, f.width) - f.deltas[at]) * f.scale;
        }
        for (int32_t i = 0; i < n; ++i) {
          float const pi = __shfl(p, i), di = __shfl(ds, i);
#pragma unroll
          for (int c = 0; c < kMostWidth / kWave; ++c)
            if (c * kWave + lane < f.width) {
              dv[c] = fmaf(pi, static_cast<float>(f.grad.at(token + i, h)[c * kWave + lane]), dv[c]);
              dk[c] = fmaf(di, static_cast<float>(f.q.at(token + i, h)[c * kWave + lane]), dk[c]);
            }
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kMostWidth / kWave; ++c)
    if (c * kWave + lane < f.width) {
      if (of_k) f.k_grad.at(t, kh)[c * kWave + lane] = static_cast<T>(dk[c]);
      if (of_v) f.v_grad.at(t, kh)[c * kWave + lane] = static_cast<T>(dv[c]);
    }
}

// Of keys whose gradients are not finite, whether all of them are so for tokens that they see, from token `seen` of a row's on: NaN in such a token's log makes NaN of both, in its delta
// of that of k, and a token without a finite value in its gradient leaves none in that of v.
template <typename T>
__device__ __forceinline__ bool is_odd_anyway(Backward<T> const& f, int32_t begin, int32_t seen, int32_t tokens, int32_t kv_head, bool of_k, bool of_v)
{
  int32_t const each = f.heads / f.kv_heads;
#pragma unroll 1
  for (int32_t h = kv_head * each; h < (kv_head + 1) * each; ++h) {
    bool odd_v = !of_v;
    if (of_v && seen < tokens) {
      const T* const grad = f.grad.at(static_cast<int64_t>(begin) + tokens - 1, h);
      bool finite         = false;
      for (int32_t j = lane_id(); j < f.width; j += kWave) finite = finite || fabsf(static_cast<float>(grad[j])) < INFINITY;
      odd_v = __ballot(finite) == 0;
      if (odd_v && !of_k) return true;
    }
#pragma unroll 1
    for (int32_t i = seen; i < tokens; i += kWave) {
      int64_t const at  = static_cast<int64_t>(h) * f.runs.tokens + begin + i + lane_id();
      bool const there  = i + lane_id() < tokens;
      float const log   = there ? f.logsum[at] : 0.f, delta = there && odd_v ? f.deltas[at] : 0.f;
      if (__ballot(log != log || delta != delta)) return true;
    }
  }
  return false;
}

// ------------------------------------------------------------------ tiles
// Products of 32 x 32 on the matrix cores, 16 deep.  A lane has 8 values of a row (or column) of each operand, number l % 32, from 8 * (l / 32) on;
// of the result column l % 32, and of it rows 8 * (r / 4) + 4 * (l / 32) + r % 4 for r = 0 .. 15.
typedef float f32x16_t __attribute__((ext_vector_type(16)));
__device__ __forceinline__ f32x16_t multiply32(Fragment<bf16_t> a, Fragment<bf16_t> b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16_t multiply32(Fragment<half_t> a, Fragment<half_t> b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// (2 deep, eight times: value k of every lane of a half goes into product k)
__device__ __forceinline__ f32x16_t multiply32(Fragment<float> a, Fragment<float> b, f32x16_t c)
{
#pragma unroll
  for (int k = 0; k < 8; ++k) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[k], b[k], c, 0, 0, 0);
  return c;
}

// A tile of heads of D values (a multiple of 32) of as many tokens or keys, as it lies in LDS: in pieces of 16 bytes, whose order is turned with the head's
// number so that what is read at once lies in all of the 256 bytes of LDS's banks: pieces of one number of 16 neighbouring heads (the reads of rows), units
// of two pieces of 4 neighbouring heads and the units beside them (the transposing reads of columns), 8 pieces of a head and of the one 4 further
// on (columns of 32-bit types).
// There are 64 heads in a tile, of 1024 bytes 32: two tiles, twice, fill no more than 128 KB.
constexpr int heads_of_tile(int bytes) { return bytes > 512 ? 32 : 64; }
template <typename T, int D, int HEADS = heads_of_tile(D * sizeof(T))>
struct Tile {
  static_assert(D % 32 == 0 && D <= kMostWidth);
  static constexpr int kHeads = HEADS;
  static constexpr int kLine = D * sizeof(T), kBytes = kHeads * kLine, kPieces = kLine / 16;  // bytes of a head, of all, pieces of 16 bytes of a head
  __device__ __forceinline__ static constexpr uint32_t turn(uint32_t head)
  {
    uint32_t const last = head >> 3 & 1, third = head >> 2 & 1;
    if constexpr (sizeof(T) == 4) return (kPieces % 16 == 0 ? third << 3 : 0) | (head & 3) << 1 | last;  // (no piece leaves its head)
    if constexpr (kLine % 256 == 0) return (head & 3) << 2 | third << 1 | last;
    if constexpr (kLine % 128 == 0) return (head & 2) << 1 | third << 1 | last;  // (neighbouring heads begin 128 bytes apart)
    return third << 1 | last;                                                   // (they begin 64 bytes apart, in some order)
  }
};

// What a wavefront of WAVES loads of a tile: straight into LDS, 64 pieces of 16 bytes at a time, zeros for what is not there.
template <typename T, int D, int WAVES, int HEADS = Tile<T, D>::kHeads>
struct TileLoader {
  using Of = Tile<T, D, HEADS>;
  static constexpr int kAll = Of::kHeads * Of::kPieces / kWave, kLoads = (kAll + WAVES - 1) / WAVES, kEach = 16 / sizeof(T);
  uint32_t offset[kLoads];
  uint32_t line, width;  // bytes from a head to the next, of one
  const char* base;      // of the next tile

  __device__ __forceinline__ void aim(Heads<const T> const& x, int32_t first, int32_t head, int32_t columns, int wave, int lane)
  {
    base  = reinterpret_cast<const char*>(x.at(first, head));
    line  = static_cast<uint32_t>(x.stride * sizeof(T));
    width = static_cast<uint32_t>((columns + kEach - 1) / kEach * 16);  // (whole pieces: those of an odd width have been copied, and end in zeros)
#pragma unroll
    for (int p = 0; p < kLoads; ++p) {
      int const slot = (p * WAVES + wave) * kWave + lane, row = slot / Of::kPieces, piece = slot % Of::kPieces;
      int const from = static_cast<int>(static_cast<uint32_t>(piece) ^ Of::turn(row));
      offset[p]      = from * kEach < columns ? row * line + from * 16 : kFar;
    }
  }
  // The next tile, of which `here` heads are there.
  __device__ __forceinline__ void load(LdsBytes to, int32_t here, int wave)
  {
    uint32_t const range = uniform(static_cast<uint32_t>(here < Of::kHeads ? here - 1 : Of::kHeads - 1) * line + width);
    const char* const at = uniform(base);
#pragma unroll
    for (int p = 0; p < kLoads; ++p)
      if (kAll % WAVES == 0 || p * WAVES + wave < kAll) load_to_lds(at, range, to + (p * WAVES + wave) * 1024, offset[p]);
    base += static_cast<int64_t>(Of::kHeads) * line;
  }
};

// Where a lane finds fragments of a tile.
template <typename T, int D>
struct TileReader {
  static constexpr int kLine = Tile<T, D>::kLine;
  uint32_t row, column, turn_row, turn_column;
  __device__ __forceinline__ explicit TileReader(int lane)
  {
    int const h = lane / 32, i = lane % 16;
    row         = (lane % 32) * kLine;
    turn_row    = Tile<T, D>::turn(lane % 32);
    if constexpr (sizeof(T) == 2) {
      turn_row ^= h;
      int const k = 4 * h + i / 4;
      column      = k * kLine + i % 2 * 8;
      turn_column = Tile<T, D>::turn(k) ^ (lane / 16 % 2 * 2 + i / 2 % 2);
    } else {
      turn_row ^= 2 * h;
      column      = 4 * h * kLine + lane % 4 * 4;
      turn_column = Tile<T, D>::turn(4 * h) ^ (lane % 32 / 4);
    }
  }
  // 32 heads from 32 * block on, values 16 * step .. 16 * step + 15 of each
  __device__ __forceinline__ Fragment<T> rows(LdsBytes tile, int block, int step) const
  {
    LdsBytes const p = tile + row + block * (32 * kLine);
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<__attribute__((address_space(3))) Fragment<T>*>(p + ((2 * step) ^ turn_row) * 16);
    } else {
      f32x4_t const low  = *reinterpret_cast<__attribute__((address_space(3))) f32x4_t*>(p + ((4 * step) ^ turn_row) * 16);
      f32x4_t const high = *reinterpret_cast<__attribute__((address_space(3))) f32x4_t*>(p + ((4 * step + 1) ^ turn_row) * 16);
      return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // transposed: values 32 * block .. 32 * block + 31 of 16 heads from 16 * step on, in the order of heads that a result of 32 x 32 leaves in its registers
  __device__ __forceinline__ Fragment<T> columns(LdsBytes tile, int block, int step) const
  {
    if constexpr (sizeof(T) == 2) {
      LdsBytes const p   = tile + column + step * (16 * kLine);
      s16x4_t const low  = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(p + ((4 * block) ^ turn_column) * 16));
      s16x4_t const high = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s16x4_t*>(p + ((4 * block + 1) ^ turn_column) * 16 + 8 * kLine));
      return __builtin_bit_cast(Fragment<T>, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      Fragment<T> f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t const piece = (8 * block) ^ turn_column ^ Tile<T, D>::turn(8 * (k / 4) + k % 4);
        f[k]                 = *reinterpret_cast<__attribute__((address_space(3))) T*>(tile + column + piece * 16 + (16 * step + 8 * (k / 4) + k % 4) * kLine);
      }
      return f;
    }
  }
};

// use(0, read(0)), ... use(SLOTS - 1, read(SLOTS - 1)), with each fragment read some uses before its own: a read of LDS takes as long as a few products, and
// the compiler, left to itself, reads a fragment, waits for it and multiplies.
template <typename T, int D, int SLOTS, typename Read, typename Use>
__device__ __forceinline__ void stream(Read&& read, Use&& use)
{
  // (a fragment of 32-bit values is eight products: there is less to wait for, and of wide heads no register for it)
  constexpr int kAhead = sizeof(T) == 2 ? 3 : D < 192 ? 1 : 0;
  Fragment<T> x[kAhead + 1];
  for_each<kAhead>([&](auto i) { x[i] = read(i); });
  __builtin_amdgcn_sched_barrier(0);
  for_each<SLOTS>([&](auto slot) {
    constexpr int i = decltype(slot)::value;
    if constexpr (i + kAhead < SLOTS) x[(i + kAhead) % (kAhead + 1)] = read(std::integral_constant<int, i + kAhead>{});
    use(slot, x[i % (kAhead + 1)]);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// v of the lane of the lower 32 with this one's number among them, and of that of the upper 32
struct Halves {
  float low, high;
};
__device__ __forceinline__ Halves halves(float v)
{
  uint32_t const a = __builtin_bit_cast(uint32_t, v);
  auto const both  = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  uint32_t const low = both[0], high = both[1];  // (bit_cast of an element of a vector takes the first one, whichever is named)
  return {__builtin_bit_cast(float, low), __builtin_bit_cast(float, high)};
}

// Values 8 * step .. 8 * step + 7 of a result's registers, rounded, as an operand.
template <typename T>
__device__ __forceinline__ Fragment<T> rounded(f32x16_t const& x, int step)
{
  Fragment<T> f;
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = static_cast<T>(x[8 * step + k]);
  return f;
}

// sum and eight values, as they are after rounding
__device__ __forceinline__ float plus(float sum, Fragment<bf16_t> const& x)
{
  typedef bf16_t Two __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int k = 0; k < 8; k += 2) sum = __builtin_amdgcn_fdot2_f32_bf16(Two{x[k], x[k + 1]}, Two{bf16_t(1.f), bf16_t(1.f)}, sum, false);
  return sum;
}
__device__ __forceinline__ float plus(float sum, Fragment<half_t> const& x)
{
  typedef half_t Two __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int k = 0; k < 8; k += 2) sum = __builtin_amdgcn_fdot2(Two{x[k], x[k + 1]}, Two{half_t(1.f), half_t(1.f)}, sum, false);
  return sum;
}

// Eight of a head's values from j on, zeros behind the last or where it is not `there`; widths and strides are of whole pieces of 16 bytes
template <typename T>
__device__ __forceinline__ Fragment<T> fragment_of(const T* head, int32_t j, int32_t width, bool there)
{
  Fragment<T> f{};
  if constexpr (sizeof(T) == 2) {
    if (there && j < width) f = *reinterpret_cast<const Fragment<T>*>(head + j);
  } else {
    f32x4_t low{}, high{};
    if (there && j < width) low = *reinterpret_cast<const f32x4_t*>(head + j);
    if (there && j + 4 < width) high = *reinterpret_cast<const f32x4_t*>(head + j + 4);
    f = __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  return f;
}

// Writes a lane's column of results, transposed: with what its neighbour of the other half has, eight values of a head next to each other (stores of 16 bytes take
// any address that the type has).  Those of a width that is no multiple of eight end one by one.
template <typename U, int COLUMNS, typename Make>
__device__ __forceinline__ void store_eights(U* head, int half, int32_t width, Make&& make)
{
  typedef U Eight_t __attribute__((ext_vector_type(8), aligned(sizeof(U))));
  typedef uint32_t Words __attribute__((ext_vector_type(sizeof(U))));  // four values
#pragma unroll
  for (int c = 0; c < COLUMNS; ++c)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      // (this lane has values 4 * half .. 4 * half + 3 of the eight from 32 c + 8 g on, and of the next eight; each half gives one of them away)
      Words a = make(c, g), b = make(c, g + 1);
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(U)); ++w) {
        uint32_t const x = a[w], y = b[w];
        auto const both  = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        a[w]             = both[0];
        b[w]             = both[1];
      }
      typedef uint32_t Both __attribute__((ext_vector_type(2 * sizeof(U))));
      Both words;
#pragma unroll
      for (int w = 0; w < static_cast<int>(sizeof(U)); ++w) {
        words[w]             = a[w];
        words[w + sizeof(U)] = b[w];
      }
      Eight_t const eight = __builtin_bit_cast(Eight_t, words);
      int32_t const j     = 32 * c + 8 * g + 8 * half;
      if (width == 32 * COLUMNS || j + 8 <= width) {
        *reinterpret_cast<Eight_t*>(head + j) = eight;
      } else {
        for (int e = 0; e < 7; ++e)
          if (j + e < width) head[j + e] = eight[e];
      }
    }
}

template <typename T, int COLUMNS>
__device__ __forceinline__ void store_columns(T* head, f32x16_t const (&x)[COLUMNS], int half, int32_t width)
{
  store_eights<T, COLUMNS>(head, half, width, [&](int c, int g) {
    typedef T Four __attribute__((ext_vector_type(4)));
    Four const four = {static_cast<T>(x[c][4 * g]), static_cast<T>(x[c][4 * g + 1]), static_cast<T>(x[c][4 * g + 2]), static_cast<T>(x[c][4 * g + 3])};
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T))));
    return __builtin_bit_cast(Words, four);
  });
}

// The same for what rounding left off.
template <typename T, int COLUMNS>
__device__ __forceinline__ void store_rests(int8_t* head, f32x16_t const (&x)[COLUMNS], int half, int32_t width)
{
  store_eights<int8_t, COLUMNS>(head, half, width, [&](int c, int g) {
    uint32_t four = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) four |= static_cast<uint32_t>(static_cast<uint8_t>(rest_of(x[c][4 * g + e], static_cast<T>(x[c][4 * g + e])))) << 8 * e;
    typedef uint32_t Words __attribute__((ext_vector_type(1)));
    return Words{four};
  });
}

// ------------------------------------------------------------------ work
constexpr int kThreads = 256;
constexpr int kTileWaves = 4;  // wavefronts that share the tiles in LDS
// Of rows that have at most kShortRow tokens and keys on average, a wavefront alone: blocks of 32 tokens and tiles of 32 keys, so that nothing waits for what is not there.
// (60,000 tokens over their own keys, 8 heads, a step in bfloat16, us with four wavefronts and with one: rows of 12 tokens, heads of 64 1127 and 478, of 128 2547 and 1445; of 48 tokens
// 435 and 330, 945 and 841; of 100 367 and 352, 784 and 882.  Over more keys than that, four share them, forward: 16 rows of 48 tokens, 64 heads of 128 over 8, 2000 keys a row
// 142 and 162, 40000 keys 2440 and 2900; 1000 rows of 50 tokens, 8 heads of 64, 250 keys 153 and 173, 850 keys 437 and 540; of 20 tokens, 420 keys 294 and 291.)
constexpr int kShortRow = 64;
template <typename T>
bool is_short(Problem<T> const& p, int32_t most = kShortRow)
{
  return p.runs.rows > 0 && std::max(p.runs.tokens, p.key_runs.tokens) <= static_cast<int64_t>(p.runs.rows) * most;
}
template <typename T, int D, int WAVES>
constexpr int kTileOf = WAVES == 1 ? 32 : Tile<T, D>::kHeads;

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
// float32, for another launch to join.  A share has at least kLeastTiles, in which the first loads' wait is worth it: in how many shares `tiles` go, and what one of them has.
constexpr int kLeastTiles = 2;
__device__ __forceinline__ int32_t shares_of(int32_t tiles, int32_t splits) { return splits == 1 || tiles < 2 * kLeastTiles ? 1 : min(splits, tiles / kLeastTiles); }
__device__ __forceinline__ int32_t share_begin(int32_t tiles, int32_t share, int32_t shares) { return static_cast<int32_t>(static_cast<int64_t>(tiles) * share / shares); }

struct Split {
  int32_t splits;
  float* sums;
  float4* tops;  // (forward) [block][head][share][row]: top, the sum of the exponentials, and what out is divided by
  __device__ __forceinline__ int64_t slot(int64_t block, int32_t head, int32_t heads, int32_t share) const { return (block * heads + head) * splits + share; }
};

// A lane's part of a row of D values that a wavefront holds side by side: values first() .. first() + kEach - 1, of the lanes that have any.
template <int D>
struct Some {
  static constexpr int kEach = (D + kWave - 1) / kWave;
  float v[kEach] = {};
  __device__ __forceinline__ static int first() { return lane_id() * kEach; }
  __device__ __forceinline__ void add(const float* row, float weight)
  {
    if (first() < D) {
#pragma unroll
      for (int k = 0; k < kEach; ++k) v[k] = fmaf(row[first() + k], weight, v[k]);
    }
  }
  // whether the first `width` values of the row are all finite
  __device__ __forceinline__ bool finite(int32_t width) const
  {
    float check = 0.f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) check = first() + k < width ? fmaf(v[k], 0.f, check) : check;
    return __ballot(check != 0.f) == 0;
  }
};

// ------------------------------------------------------------------ launches
// Whether the tiles' loads can read heads as they lie: pieces of 16 bytes, lines of a tile within the 31 bits of their offsets, and tokens that do not overlap (unless all are one):
// what is loaded behind the last of them has to be zeros, or what the last one has in the same place.
template <typename T>
bool reads_as_it_lies(Heads<const T> const& x, int32_t width)
{
  constexpr int kEach = 16 / sizeof(T);
  return width % kEach == 0 && x.stride % kEach == 0 && x.head_stride % kEach == 0 && reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.stride < (int64_t{1} << 23) &&
         (x.stride == 0 || x.stride >= width);
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

// In how many shares a launch's tiles go: the number for which this time is least.  A tile takes PRODUCTS matrix products of 32 x 32 heads a wavefront, of 16-bit
// types 0.33 + 0.0031 D us each for 64 keys while a CU has one workgroup (of two, each takes 3/2 of that, as far as LDS has room for two), of float32, whose products are
// all that counts, 0.045 D.  Shares of a tile's rows are written and read again, at 2.5 TB/s, by another launch, 6 us.  Rows are taken to be alike, which is all the
// host knows; of causal ones the last blocks have twice as many tiles as the average.  (bfloat16, us without and with: two rows of 1536 tokens, 8 heads of
// 64 28 and 43, in 3 shares; one row of 8000, one head of 128 139 and 66, in 8; a step over one row of 2000, 12 heads of 64 117, 115 in 3, 144 in 6.)
constexpr int kMostShares = 16;
template <typename T, int D, int PRODUCTS>
int32_t splits_of(Problem<T> const& p, Runs const& blocks, int32_t heads, int shift, Runs const& other, int64_t times, int lds)
{
  constexpr int kTile  = Tile<T, D>::kHeads;
  int64_t const rows   = std::max(1, blocks.rows), length = (blocks.tokens + rows - 1) / rows, seen = (other.tokens + rows - 1) / rows;
  bool const half      = p.causal && other.tokens <= blocks.tokens;
  double const most    = static_cast<double>((seen + kTile - 1) / kTile * times), tiles = half ? (most + times) / 2 : most;
  double const tile    = PRODUCTS * (sizeof(T) == 2 ? 0.33 + 0.0031 * D : 0.045 * D) * kTile / 64;
  double const per_cu  = static_cast<double>(rows * ((length + (1 << shift) - 1) >> shift) * heads) / device_cus();
  double const bytes   = static_cast<double>(rows * length) * heads * D * sizeof(float) * (PRODUCTS > 3 ? 2 : 1);
  auto const at_once   = [&](double n) { return n <= 1 ? n : 2 * lds > 160 * 1024 ? 1. : std::min(1 + (n - 1) / 2, 1.5); };
  int32_t best         = 1;
  double least         = INFINITY;
  for (int32_t n = 1; n == 1 || (n <= kMostShares && n * kLeastTiles <= tiles); ++n) {
    double const time = tile * std::max(tiles * per_cu / at_once(per_cu * n), most / n) + (n > 1 ? 6 + 2 * n * bytes / 2.5e6 : 0);
    if (time < least) least = time, best = n;
  }
  return best;
}

// calls f with the width of the tiles that heads of `width` values go through
template <typename F>
nvtext_amd_status with_tiles(int32_t width, F&& f)
{
  if (width <= 64) return f(std::integral_constant<int, 64>{});
  if (width <= 96) return f(std::integral_constant<int, 96>{});
  if (width <= 128) return f(std::integral_constant<int, 128>{});
  if (width <= 192) return f(std::integral_constant<int, 192>{});
  return f(std::integral_constant<int, 256>{});
}

// What both directions ask of their arguments; nullptr if it holds.
inline const char* bad_attention(const nvtext_amd_heads* q, const nvtext_amd_heads* k, const nvtext_amd_heads* v, int32_t rows, const int32_t* offsets, const int32_t* key_offsets,
                          const int32_t* key_lengths, double scale)
{
  for (auto* x : {q, k, v})
    if (const char* bad = bad_heads(x)) return bad;
  if (k->type != q->type || v->type != q->type) return "q, k and v must be of one type";
  if (!is_like(v, k)) return "v must be of k's size";
  if (k->width != q->width) return "k and v must be of q's width";
  if (q->width > kMostWidth) return "heads may have 256 values at most";
  if (q->heads > 0 ? k->heads == 0 || q->heads % k->heads != 0 : k->heads != 0) return "the heads of k and v must be a divisor of q's";
  // (numbers of tiles are counted in 32 bits, and tokens up to a tile's end; launches in 64)
  if (q->tokens > kMostTokens || k->tokens > kMostTokens || q->heads > kMostHeads) return "there may be 2^31 - 1025 tokens and 65536 heads at most";
  if (k->heads > 0 && (q->tokens / 32 + 1) * (q->heads / k->heads) > INT32_MAX) return "too many tokens for so many heads that share keys";
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

}  // namespace nvtext_amd
