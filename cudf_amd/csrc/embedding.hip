// Embedding of a LIST<INT32> column of token ids, and the gradients of its tables.
#include "encoder.cuh"

#include <algorithm>

namespace nvtext_amd {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves   = kThreads / kWave;

struct Tokens {
  const int32_t* offsets;
  const int32_t* ids;
  int32_t rows;
  int32_t count;

  // where in its row token t is, or -1: it belongs to none.  (The last row that does not begin behind t: empty rows in front of it
  // begin where it does.)
  __device__ __forceinline__ int64_t place(int32_t t) const
  {
    if (rows == 0 || t >= offsets[rows]) return -1;
    int32_t lo = 0, hi = rows;  // offsets[lo - 1] <= t < offsets[hi]
    while (lo < hi) {
      int32_t const mid = lo + (hi - lo) / 2;
      if (offsets[mid] <= t)
        lo = mid + 1;
      else
        hi = mid;
    }
    return lo == 0 ? -1 : static_cast<int64_t>(t) - offsets[lo - 1];
  }
};

// A wavefront takes `each` consecutive tokens: a lane finds the place of one of them in its row, all at once (a search for each token
// on its own, a dozen reads one after the other, took 555 us of what is 294 now), then the rows of the tables are added up, kAtOnce
// tokens asked for at a time.  VEC = 8 columns a lane; the lanes behind the last column take the last eight once more.  (VEC = 1 for
// less than eight columns.)  Rows of up to 256 columns lie side by side in a wavefront, LANES lanes each: 1,276,351 tokens of 64
// columns took 185 us with one.  Bound by memory: 512,011 tokens of 1024 16-bit values take 294 us and move 1.44 GB, 4.9 TB/s, where a
// copy reaches 5 (1.18 GB are needed: some rows of the table are read again); the results are stored past the caches, which keep the
// table (372 us without that).
// With 8, 32 or 64 tokens a wavefront 308, 308 and 315 us, with 4 at a time 307.
constexpr int kAtOnce = 8, kMostEach = 16;

template <typename T, int VEC>
struct Some {
  typedef T type __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
};
template <typename T, int VEC>
using some_t = typename Some<T, VEC>::type;

template <int VEC, typename T>
__device__ __forceinline__ some_t<T, VEC> load_some(const T* p)
{
  return *reinterpret_cast<const some_t<T, VEC>*>(p);
}

template <int VEC, int LANES, typename T>
__global__ void __launch_bounds__(kThreads)
embedding_kernel(Tokens tokens, Rows<const T> table, int64_t vocabulary, Rows<const T> positions, int64_t places, int64_t cols, int32_t each, Rows<T> out)
{
  constexpr int kAcross = kWave / LANES;  // tokens side by side
  int const lane        = lane_id(), beside = lane / LANES;
  int64_t const first   = (static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave) * each;
  if (first >= tokens.count) return;
  int const count = static_cast<int>(tokens.count - first < each ? tokens.count - first : each);
  int32_t id = -1, at = -1;  // (-1: nothing)
  if (lane < count) {
    int64_t const place = tokens.place(static_cast<int32_t>(first + lane));
    id                  = tokens.ids[first + lane];
    id                  = place >= 0 && id < vocabulary ? id : -1;
    at                  = place < places ? static_cast<int32_t>(place) : -1;
  }
  for (int64_t slice = 0; slice < cols; slice += VEC * LANES) {
    int64_t const j = slice + lane % LANES * VEC + VEC <= cols ? slice + lane % LANES * VEC : cols - VEC;
    for (int base = 0; base < count; base += kAtOnce * kAcross) {
      some_t<T, VEC> e[kAtOnce], p[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        int const from = base + u * kAcross + beside;  // (behind the last there is nothing, or it is one before, not written)
        int32_t row, place;
        if constexpr (kAcross == 1) {
          row   = static_cast<int32_t>(wave_bcast(id, from % kWave));
          place = static_cast<int32_t>(wave_bcast(at, from % kWave));
        } else {
          row   = __shfl(id, from % kWave);
          place = __shfl(at, from % kWave);
        }
        e[u] = p[u] = some_t<T, VEC>{};
        if (row >= 0) e[u] = load_some<VEC>(table.row(row) + j);
        if (place >= 0) p[u] = load_some<VEC>(positions.row(place) + j);
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        int const from = base + u * kAcross + beside;
        if (from < count) {
          some_t<T, VEC> sum;
#pragma unroll
          for (int k = 0; k < VEC; ++k) sum[k] = static_cast<T>(static_cast<float>(e[u][k]) + static_cast<float>(p[u][k]));
          __builtin_nontemporal_store(sum, reinterpret_cast<some_t<T, VEC>*>(out.row(first + from) + j));
        }
      }
    }
  }
}

// ------------------------------------------------------------------ tokens in the order of their ids
// A stable sort: tokens of one id stay in their order, so that sums over them are added in one order at every call.  Least
// significant digit first, eight to ten bits a pass (as few passes as there can be: 218,375 tokens of 1000
// ids 26 us in two, 21 in one; 162,369 of 250,000 37 us in three, 31 in two): count the digits of every tile, then place, for which every workgroup adds up the
// counts that it needs (of more than kDirectTiles tiles, device_exclusive_scan does).  Up to kSmall tokens are sorted by one
// workgroup, in LDS: one launch.  Digits repeat as the words of a text do, so lanes with the same one are counted at once: with an
// atomic a lane the four launches over 262,139 tokens took 43 us.
constexpr int kSortThreads    = 1024;
constexpr int kSortWaves      = kSortThreads / kWave;
constexpr int kSmall          = 8192;  // tokens that one workgroup sorts
constexpr int kTile           = 2048;
constexpr int kRounds         = kTile / kSortThreads;
constexpr int kDirectTiles    = 256;

struct Sorted {
  uint32_t* keys;  // id, or the size of the vocabulary for what belongs to no entry
  uint32_t* tokens;
};

// Where a pass reads: the column itself at first.
struct Unsorted {
  Tokens column;
  uint32_t vocabulary;
  __device__ __forceinline__ uint32_t key(int64_t t) const
  {
    uint32_t const id = static_cast<uint32_t>(column.ids[t]);
    bool const inside = column.rows > 0 && t >= column.offsets[0] && t < column.offsets[column.rows];
    return inside && id < vocabulary ? id : vocabulary;
  }
  __device__ __forceinline__ uint32_t token(int64_t t) const { return static_cast<uint32_t>(t); }
};
struct Half {
  Sorted from;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return from.keys[i]; }
  __device__ __forceinline__ uint32_t token(int64_t i) const { return from.tokens[i]; }
};

// Of the wavefront's 64 keys (`here`: there is one): the lanes that have the same digit.
template <int BITS>
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool here)
{
  uint64_t same = ballot64(here);
#pragma unroll
  for (int bit = 0; bit < BITS; ++bit) {
    bool const set        = (digit >> bit) & 1u;
    uint64_t const others = ballot64(set);
    same &= set ? others : ~others;
  }
  return same;
}

// Counts the wavefront's keys in `counts`, digit by digit; returns how many with the same digit were counted before the lane's own.
template <int BITS>
__device__ __forceinline__ uint32_t count_digit(uint32_t* counts, uint32_t digit, bool here)
{
  uint64_t const same   = same_digit<BITS>(digit, here);
  uint32_t const below  = lanes_below(same);
  uint32_t const before = here ? counts[digit] : 0;
  wave_lds_fence();
  if (here && below == 0) counts[digit] = before + static_cast<uint32_t>(__builtin_popcountll(same));
  wave_lds_fence();
  return before + below;
}

// counts[tile][digit], or [digit][tile] for the scan
template <typename From, int BITS>
__global__ void __launch_bounds__(kSortThreads) digit_counts_kernel(From from, int32_t n, int shift, int32_t tiles, bool by_digit, uint32_t* counts)
{
  constexpr int kDigits = 1 << BITS;
  __shared__ uint32_t lds[kSortWaves][kDigits];
  int const wave = threadIdx.x / kWave;
  for (int w = threadIdx.x / kDigits; w < kSortWaves; w += kSortThreads / kDigits) lds[w][threadIdx.x % kDigits] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    int64_t const i = static_cast<int64_t>(blockIdx.x) * kTile + r * kSortThreads + threadIdx.x;
    bool const here = i < n;
    count_digit<BITS>(lds[wave], ((here ? from.key(i) : 0) >> shift) & (kDigits - 1), here);
  }
  __syncthreads();
  if (threadIdx.x >= kDigits) return;
  uint32_t sum = 0;
  for (int w = 0; w < kSortWaves; ++w) sum += lds[w][threadIdx.x];
  counts[by_digit ? static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x : static_cast<int64_t>(blockIdx.x) * kDigits + threadIdx.x] = sum;
}

// `summed`: counts[digit][tile] are places already.
template <typename From, int BITS>
__global__ void __launch_bounds__(kSortThreads) digit_place_kernel(From from, int32_t n, int shift, int32_t tiles, bool summed, const uint32_t* counts, Sorted out)
{
  constexpr int kDigits = 1 << BITS;
  __shared__ uint32_t lds[kSortWaves][kDigits];
  constexpr int kParts = kSortThreads / kDigits;
  __shared__ uint32_t before[kParts][kDigits], all[kParts][kDigits], scan[kSortWaves + 1];
  int const wave = threadIdx.x / kWave, lane = lane_id();
  for (int w = threadIdx.x / kDigits; w < kSortWaves; w += kSortThreads / kDigits) lds[w][threadIdx.x % kDigits] = 0;
  __syncthreads();
  // a wavefront's keys are consecutive, 64 a round
  uint32_t key[kRounds], token[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    int64_t const i = static_cast<int64_t>(blockIdx.x) * kTile + (wave * kRounds + r) * kWave + lane;
    key[r]          = i < n ? from.key(i) : 0;
    token[r]        = i < n ? from.token(i) : 0;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    rank[r] = count_digit<BITS>(lds[wave], (key[r] >> shift) & (kDigits - 1), static_cast<int64_t>(blockIdx.x) * kTile + (wave * kRounds + r) * kWave + lane < n);
  uint32_t place = 0;
  if (summed) {
    if (threadIdx.x < kDigits) place = counts[static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x];
    __syncthreads();
  } else {
    // kParts threads a digit add up the tiles' counts: those before this one, and all
    int const part = threadIdx.x / kDigits, digit = threadIdx.x % kDigits;
    uint32_t mine = 0, every = 0;
#pragma unroll 16
    for (int32_t t = part; t < tiles; t += kParts) {
      uint32_t const c = counts[static_cast<int64_t>(t) * kDigits + digit];
      every += c;
      mine += t < static_cast<int32_t>(blockIdx.x) ? c : 0;
    }
    before[part][digit] = mine;
    all[part][digit]    = every;
    __syncthreads();
    uint32_t total = 0, behind = 0;
    if (threadIdx.x < kDigits) {
      every = mine = 0;
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        every += all[p][digit];
        mine += before[p][digit];
      }
    }
    behind = block_exclusive_scan<kSortThreads>(threadIdx.x < kDigits ? every : 0, scan, &total);
    place  = behind + mine;
  }
  if (threadIdx.x < kDigits) {
    for (int w = 0; w < kSortWaves; ++w) {
      uint32_t const count = lds[w][threadIdx.x];
      lds[w][threadIdx.x]  = place;
      place += count;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    int64_t const i = static_cast<int64_t>(blockIdx.x) * kTile + (wave * kRounds + r) * kWave + lane;
    if (i < n) {
      uint32_t const at = lds[wave][(key[r] >> shift) & (kDigits - 1)] + rank[r];
      out.keys[at]      = key[r];
      out.tokens[at]    = token[r];
    }
  }
}

// All passes over up to kSmall tokens.
template <int BITS>
__global__ void __launch_bounds__(kSortThreads) small_sort_kernel(Unsorted from, int32_t n, Sorted out)
{
  constexpr int kDigits = 1 << BITS;
  __shared__ uint32_t lds[kSortWaves][kDigits];
  __shared__ uint32_t keys[kSmall];
  __shared__ uint16_t tokens[kSmall];
  __shared__ uint32_t scan[kSortWaves + 1];
  int const wave = threadIdx.x / kWave, lane = lane_id();
  // a wavefront's keys are consecutive, and shared evenly
  int const rounds = (n + kSortThreads - 1) / kSortThreads;
  constexpr int kMost = kSmall / kSortThreads;
  uint32_t key[kMost], token[kMost], rank[kMost];
#pragma unroll
  for (int r = 0; r < kMost; ++r) {
    int const i = (wave * rounds + r) * kWave + lane;
    key[r]      = r < rounds && i < n ? from.key(i) : 0;
    token[r]    = i;
  }
  for (int shift = 0; shift < 32 && (from.vocabulary >> shift) != 0; shift += BITS) {
    for (int w = threadIdx.x / kDigits; w < kSortWaves; w += kSortThreads / kDigits) lds[w][threadIdx.x % kDigits] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kMost; ++r)
      if (r < rounds) rank[r] = count_digit<BITS>(lds[wave], (key[r] >> shift) & (kDigits - 1), (wave * rounds + r) * kWave + lane < n);
    __syncthreads();
    uint32_t every = 0, total;
    if (threadIdx.x < kDigits)
      for (int w = 0; w < kSortWaves; ++w) every += lds[w][threadIdx.x];
    uint32_t place = block_exclusive_scan<kSortThreads>(every, scan, &total);
    if (threadIdx.x < kDigits)
      for (int w = 0; w < kSortWaves; ++w) {
        uint32_t const count = lds[w][threadIdx.x];
        lds[w][threadIdx.x]  = place;
        place += count;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kMost; ++r) {
      if (r < rounds && (wave * rounds + r) * kWave + lane < n) {
        uint32_t const at = lds[wave][(key[r] >> shift) & (kDigits - 1)] + rank[r];
        keys[at]          = key[r];
        tokens[at]        = static_cast<uint16_t>(token[r]);
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kMost; ++r) {
      int const i = (wave * rounds + r) * kWave + lane;
      if (r < rounds && i < n) {
        key[r]   = keys[i];
        token[r] = tokens[i];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kMost; ++r) {
    int const i = (wave * rounds + r) * kWave + lane;
    if (r < rounds && i < n) {
      out.keys[i]   = key[r];
      out.tokens[i] = token[r];
    }
  }
}

struct Counts {
  const uint32_t* counts;
  __device__ uint64_t operator()(int64_t i) const { return counts[i]; }
};

// ------------------------------------------------------------------ the tables' gradients
// Columns are taken 256 at a time, a slice: VEC = 4 values a lane, and the lanes behind the last column take the last four once more,
// so that no load has a condition.  (Of less than four columns, VEC = 1.)
constexpr int kAhead     = 16;  // rows of the gradient that a wavefront asks for before it adds the first
constexpr int kSumWaves  = 8;
constexpr int kSumThreads = kSumWaves * kWave;
// The sorted tokens are cut into chunks of kChunk, a token a lane, or of kSmallChunk, up to kFewTokens (which a wavefront reads at once,
// instead of four times one after the other: sums of 17,016 tokens of 192 columns 17 -> 13 us).  A wavefront adds up the gradients of a chunk, id by id; an id whose
// tokens all lie in the chunk is done then, the sums of others go to the chunk's two places: the first for an id that began in a
// chunk before, the second for one that begins here and goes on.
constexpr int kChunk = kWave, kSmallChunk = kAhead, kFewTokens = 32768;

template <typename T, int VEC>
__device__ __forceinline__ void add(float (&f)[VEC], some_t<T, VEC> const& v)
{
#pragma unroll
  for (int k = 0; k < VEC; ++k) f[k] += static_cast<float>(v[k]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_some(T* p, float const (&f)[VEC])
{
  some_t<T, VEC> v;
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = static_cast<T>(f[k]);
  *reinterpret_cast<some_t<T, VEC>*>(p) = v;
}

// What the sums are made from and where they go.
template <typename T, typename G>
struct Sums {
  Sorted sorted;
  int32_t n, chunk, chunks;  // tokens, of them a chunk, chunks
  uint32_t vocabulary;
  Tokens column;
  Rows<const T> grad;
  int64_t cols;
  Rows<G> tokens;
  float* token_parts;  // [chunk][2][cols]
  int32_t places, groups, group;  // positions, runs of rows, rows a run
  Rows<G> positions;
  float* position_parts;  // [run][place][cols], where there are several
};

// A wavefront a chunk.
template <int VEC, typename T, typename G>
__device__ __forceinline__ void add_chunk(Sums<T, G> const& s, int32_t chunk, int64_t j)
{
  int const lane      = lane_id();
  int64_t const first = static_cast<int64_t>(chunk) * s.chunk;
  int64_t const i     = first + lane;
  bool const here     = lane < s.chunk && i < s.n;
  uint32_t const none = 0xffffffffu;  // (no key)
  uint32_t const key = here ? s.sorted.keys[i] : none, token = here ? s.sorted.tokens[i] : 0;
  uint32_t const behind = here && i + 1 < s.n ? s.sorted.keys[i + 1] : none;
  uint64_t const ends   = ballot64(key != behind);
  int const count       = __builtin_popcountll(ballot64(key < s.vocabulary));  // (the lowest ones)
  bool begun            = first == 0 || s.sorted.keys[first - 1] != wave_bcast(key, 0);
  float f[VEC]          = {};
  for (int base = 0; base < count; base += kAhead) {
    some_t<T, VEC> g[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) g[u] = load_some<VEC>(s.grad.row(wave_bcast(token, base + u)) + j);  // (kAhead divides a chunk; what is not counted is some row all the same)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (base + u < count) {
        add<T, VEC>(f, g[u]);
        bool const end = (ends >> (base + u)) & 1u;
        if (end || base + u + 1 == count) {
          if (begun && end)
            store_some<G, VEC>(s.tokens.row(wave_bcast(key, base + u)) + j, f);
          else
            store_some<float, VEC>(s.token_parts + (2 * static_cast<int64_t>(chunk) + (begun ? 1 : 0)) * s.cols + j, f);
#pragma unroll
          for (int k = 0; k < VEC; ++k) f[k] = 0.f;
          begun = true;
        }
      }
    }
  }
}

// Zeros for the entries that do not occur: a wavefront looks 64 of them up in the sorted ids.
template <int VEC, typename T, typename G>
__device__ __forceinline__ void clear_absent(Sums<T, G> const& s, int64_t first, int64_t j)
{
  uint32_t const id = static_cast<uint32_t>(first) + lane_id();
  int32_t lo = 0, hi = s.n;
  while (lo < hi) {
    int32_t const mid = lo + (hi - lo) / 2;
    if (s.sorted.keys[mid] < id)
      lo = mid + 1;
    else
      hi = mid;
  }
  uint64_t absent       = ballot64(id < s.vocabulary && (lo >= s.n || s.sorted.keys[lo] != id));
  float const zero[VEC] = {};
  for (; absent; absent &= absent - 1) store_some<G, VEC>(s.tokens.row(first + __builtin_ctzll(absent)) + j, zero);
}

// A workgroup a place and a run of rows: its wavefronts share the rows that are long enough, and add up what they found in the end.
template <int VEC, typename T, typename G>
__device__ __forceinline__ void add_place(Sums<T, G> const& s, int32_t place, int32_t run, int64_t j, float (*lds)[VEC * kWave])
{
  int const wave = threadIdx.x / kWave, lane = lane_id();
  int64_t const first = static_cast<int64_t>(run) * s.group, last = first + s.group < s.column.rows ? first + s.group : s.column.rows;
  float f[VEC] = {};
  for (int64_t base = first + wave * kWave; base < last; base += kSumThreads) {
    int64_t const r = base + lane;
    int64_t const t = r < last ? static_cast<int64_t>(s.column.offsets[r]) + place : 0;
    uint64_t enough = ballot64(r < last && t >= 0 && t < s.column.offsets[r + 1] && t < s.n);
    while (enough) {
      some_t<T, VEC> g[kAhead];
      int const count = __builtin_popcountll(enough);
      int at          = 0;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (enough) at = __builtin_ctzll(enough);  // (else the last one again, which is not counted)
        enough &= enough - 1;
        g[u] = load_some<VEC>(s.grad.row(wave_bcast(static_cast<uint32_t>(t), at)) + j);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (u < count) add<T, VEC>(f, g[u]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) lds[wave][k * kWave + lane] = f[k];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int k = 0; k < VEC; ++k)
#pragma unroll
    for (int w = 1; w < kSumWaves; ++w) f[k] += lds[w][k * kWave + lane];
  if (s.groups == 1)
    store_some<G, VEC>(s.positions.row(place) + j, f);
  else
    store_some<float, VEC>(s.position_parts + (static_cast<int64_t>(run) * s.places + place) * s.cols + j, f);
}

// The first of a lane's columns in a slice.
template <int VEC>
__device__ __forceinline__ int64_t columns_of(int64_t slice, int64_t cols)
{
  int64_t const j = (slice * kWave + lane_id()) * VEC;
  return j + VEC <= cols ? j : cols - VEC;
}

// Slice after slice, so that what both sums read of a slice is read once from memory and once from the cache behind L2: places first,
// which take longest, then chunks, then what does not occur.
template <int VEC, typename T, typename G>
__global__ void __launch_bounds__(kSumThreads) embedding_sums_kernel(Sums<T, G> s)
{
  __shared__ float lds[kSumWaves][VEC * kWave];
  int64_t const of_places = static_cast<int64_t>(s.places) * s.groups, of_chunks = (s.chunks + kSumWaves - 1) / kSumWaves;
  int64_t const of_slice = of_places + of_chunks + (static_cast<int64_t>(s.vocabulary) + kSumThreads - 1) / kSumThreads;
  int64_t const block    = block_number();
  if (block / of_slice * kWave * VEC >= s.cols) return;
  int64_t const j = columns_of<VEC>(block / of_slice, s.cols);
  int64_t at      = block % of_slice;
  int const wave  = threadIdx.x / kWave;
  if (at < of_places) {
    add_place<VEC>(s, static_cast<int32_t>(at / s.groups), static_cast<int32_t>(at % s.groups), j, lds);
  } else if (at -= of_places; at < of_chunks) {
    int64_t const chunk = at * kSumWaves + wave;
    if (chunk < s.chunks) add_chunk<VEC>(s, static_cast<int32_t>(chunk), j);
  } else {
    int64_t const first = ((at - of_chunks) * kSumWaves + wave) * kWave;
    if (first < s.vocabulary) clear_absent<VEC>(s, first, j);
  }
}

// Adds up parts[0], parts[step], ... `count` (> 0) of them, kAhead asked for at a time.
template <int VEC>
__device__ __forceinline__ void add_rows(float (&f)[VEC], const float* parts, int64_t step, int64_t count)
{
  for (int64_t base = 0; base < count; base += kAhead) {
    some_t<float, VEC> g[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) g[u] = load_some<VEC>(parts + (base + u < count ? base + u : base) * step);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (base + u < count) add<float, VEC>(f, g[u]);
    }
  }
}

// Joins the parts: of an id that begins in a chunk and goes on into others, by a wavefront, or, where these are many, by all of the
// workgroup's; and of the places, where rows were cut into runs.
template <int VEC, typename T, typename G>
__global__ void __launch_bounds__(kSumThreads) embedding_join_kernel(Sums<T, G> s)
{
  __shared__ float lds[kSumWaves][VEC * kWave];
  __shared__ int32_t length[kSumWaves];
  constexpr int32_t kAlone = 32;  // parts that a wavefront adds up by itself
  int64_t const of_chunks = (s.chunks + kSumWaves - 1) / kSumWaves;
  int64_t const of_places = s.groups > 1 ? (s.places + kSumWaves - 1) / kSumWaves : 0;
  int const wave = threadIdx.x / kWave, lane = lane_id();
  int64_t const slice = block_number() / (of_chunks + of_places), at = block_number() % (of_chunks + of_places);
  if (slice * kWave * VEC >= s.cols) return;
  int64_t const j = columns_of<VEC>(slice, s.cols);
  float f[VEC]     = {};
  if (at >= of_chunks) {
    int64_t const place = (at - of_chunks) * kSumWaves + wave;
    if (place >= s.places) return;
    add_rows<VEC>(f, s.position_parts + place * s.cols + j, static_cast<int64_t>(s.places) * s.cols, s.groups);
    store_some<G, VEC>(s.positions.row(place) + j, f);
    return;
  }
  auto const parts_of = [&](int64_t chunk) { return s.token_parts + (2 * chunk + 1) * s.cols + j; };  // the second of its places, the first ones of the next lie behind
  int64_t const chunk = at * kSumWaves + wave;
  int64_t const first = chunk * s.chunk, last = first + s.chunk;
  int32_t more        = 0;  // chunks that the id goes on into
  uint32_t id         = 0;
  if (last < s.n) {
    id                 = s.sorted.keys[last];
    bool const goes_on = id < s.vocabulary && s.sorted.keys[last - 1] == id;
    if (goes_on && (first == 0 || s.sorted.keys[first] != id || s.sorted.keys[first - 1] != id)) {
      for (;;) {
        int64_t const next  = last + (static_cast<int64_t>(more) + lane) * s.chunk;
        uint64_t const same = ballot64(next < s.n && s.sorted.keys[next < s.n ? next : 0] == id);
        int const run       = same == ~0ull ? kWave : __builtin_ctzll(~same);
        more += run;
        if (run < kWave) break;
      }
    }
  }
  auto const begin = [&](const float* part) {
    auto const v = load_some<VEC>(part);
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = v[k];
  };
  if (more > 0 && more <= kAlone) {
    begin(parts_of(chunk));
    add_rows<VEC>(f, parts_of(chunk) + s.cols, 2 * s.cols, more);
    store_some<G, VEC>(s.tokens.row(id) + j, f);
  }
  if (lane == 0) length[wave] = more;
  __syncthreads();
  for (int w = 0; w < kSumWaves; ++w) {
    if (length[w] <= kAlone) continue;
    int64_t const from = at * kSumWaves + w, each = (length[w] + kSumWaves - 1) / kSumWaves, mine = wave * each;
    int64_t const here = mine + each < length[w] ? each : length[w] - mine;
#pragma unroll
    for (int k = 0; k < VEC; ++k) f[k] = 0.f;
    if (wave == 0) begin(parts_of(from));
    if (here > 0) add_rows<VEC>(f, parts_of(from) + s.cols + 2 * mine * s.cols, 2 * s.cols, here);
#pragma unroll
    for (int k = 0; k < VEC; ++k) lds[wave][k * kWave + lane] = f[k];
    __syncthreads();
    if (wave == w) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        f[k] = 0.f;
        for (int v = 0; v < kSumWaves; ++v) f[k] += lds[v][k * kWave + lane];
      }
      store_some<G, VEC>(s.tokens.row(id) + j, f);
    }
    __syncthreads();
  }
}

const char* bad_tokens(const nvtext_amd_list_column* t)
{
  if (t->child_type != NVTEXT_AMD_TYPE_INT32) return "tokens must be a LIST<INT32> column";
  if (t->size < 0 || t->child_size < 0) return "invalid column sizes";
  if ((t->size > 0 && !t->offsets) || (t->child_size > 0 && !t->child)) return "the column of tokens has no data";
  return nullptr;
}

Tokens view_of(const nvtext_amd_list_column* t)
{
  return Tokens{t->offsets, static_cast<const int32_t*>(t->child), t->size, static_cast<int32_t>(t->child_size)};
}

}  // namespace
}  // namespace nvtext_amd

extern "C" {

nvtext_amd_status nvtext_amd_embedding(const nvtext_amd_list_column* tokens, const nvtext_amd_matrix* token_table, const nvtext_amd_matrix* position_table,
                                       void* stream_, const nvtext_amd_matrix* out)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_embedding");
  if (!tokens || !token_table || !out) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_tokens(tokens)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (tokens->child_size > INT32_MAX) return fail(NVTEXT_AMD_OVERFLOW, "the column has too many tokens");
  for (auto* m : {token_table, position_table, out})
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (token_table->type != out->type || token_table->cols != out->cols || (position_table && (position_table->type != out->type || position_table->cols != out->cols)))
    return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the tables and out must be of one type and width");
  if (out->rows != tokens->child_size) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "out must have a row for every token");
  if (out->rows == 0 || out->cols == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  with_type(out->type, [&](auto zero) {
    using T = decltype(zero);
    ProfileScope const scope("embedding", stream);
    auto const launch = [&](auto kernel, int lanes) {
      // as many tokens a wavefront as leave every SIMD four wavefronts, and those that are side by side
      int64_t const across = kWave / lanes, most = std::min<int64_t>(kMostEach * across, kWave);
      int64_t const each   = std::max<int64_t>(across, std::min<int64_t>(most, out->rows / (16 * device_cus())));
      dim3 const grid(static_cast<unsigned>(((out->rows + each - 1) / each + kWaves - 1) / kWaves)), threads(kThreads);
      hipLaunchKernelGGL(kernel, grid, threads, 0, stream, view_of(tokens), rows_of<const T>(token_table), token_table->rows, rows_of<const T>(position_table),
                         position_table ? std::min<int64_t>(position_table->rows, INT32_MAX) : 0, out->cols, static_cast<int32_t>(each), rows_of<T>(out));
    };
    if (out->cols < 8)
      launch(embedding_kernel<1, 8, T>, 8);
    else if (out->cols <= 64)
      launch(embedding_kernel<8, 8, T>, 8);
    else if (out->cols <= 128)
      launch(embedding_kernel<8, 16, T>, 16);
    else if (out->cols <= 256)
      launch(embedding_kernel<8, 32, T>, 32);
    else
      launch(embedding_kernel<8, kWave, T>, kWave);
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

nvtext_amd_status nvtext_amd_embedding_backward(const nvtext_amd_list_column* tokens, const nvtext_amd_matrix* grad, void* stream_, const nvtext_amd_allocator* mr_,
                                                const nvtext_amd_matrix* token_grad, const nvtext_amd_matrix* position_grad)
{
  using namespace nvtext_amd;
  EntryScope const entry("nvtext_amd_embedding_backward");
  if (!tokens || !grad || !token_grad) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "null argument");
  if (const char* bad = bad_tokens(tokens)) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (tokens->child_size > INT32_MAX) return fail(NVTEXT_AMD_OVERFLOW, "the column has too many tokens");
  for (auto* m : {grad, token_grad, position_grad})
    if (const char* bad = m ? bad_matrix(m) : nullptr) return fail(NVTEXT_AMD_INVALID_ARGUMENT, bad);
  if (grad->rows != tokens->child_size) return fail(NVTEXT_AMD_INVALID_ARGUMENT, "grad must have a row for every token");
  for (auto* m : {token_grad, position_grad})
    if (m && (m->cols != grad->cols || (m->type != grad->type && m->type != NVTEXT_AMD_TYPE_FLOAT32) || m->type != token_grad->type))
      return fail(NVTEXT_AMD_INVALID_ARGUMENT, "the tables' gradients must be of grad's width, both of its type or both FLOAT32");
  if (token_grad->rows > INT32_MAX || (position_grad && position_grad->rows > INT32_MAX)) return fail(NVTEXT_AMD_OVERFLOW, "a table has too many rows");
  if (grad->cols == 0) return NVTEXT_AMD_SUCCESS;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Mr const mr{mr_, stream};
  Tokens const view         = view_of(tokens);
  uint32_t const vocabulary = static_cast<uint32_t>(token_grad->rows);
  int32_t const n           = view.count;
  int64_t const cols        = grad->cols;
  bool const small          = n <= kSmall;
  int32_t const tiles       = static_cast<int32_t>((static_cast<int64_t>(n) + kTile - 1) / kTile);
  bool const direct         = tiles <= kDirectTiles;
  int32_t const chunk       = n <= kFewTokens ? kSmallChunk : kChunk;
  int32_t const chunks      = vocabulary > 0 ? static_cast<int32_t>((static_cast<int64_t>(n) + chunk - 1) / chunk) : 0;
  // the bits of a digit: as many as make few passes over the bits of an id
  int id_bits = 1;
  while (id_bits < 32 && (vocabulary >> id_bits) != 0) ++id_bits;
  int const passes          = (id_bits + 9) / 10, bits = std::max(8, (id_bits + passes - 1) / passes);
  int64_t const counts      = static_cast<int64_t>(tiles) << bits;
  int64_t const vec         = cols >= 4 ? 4 : 1, slices = (cols + vec * kWave - 1) / (vec * kWave);
  // Rows in runs of 2,048 or, if these were more than 16, in 16 runs: a place's rows are read by one workgroup a run, 30 us for 2,048.  Of
  // few places in runs of 512 (128 places of 5199 rows, 320 columns: 65 -> 60 us; 512 places of 2048, 768 columns: 146 -> 164).
  int32_t const places = position_grad ? static_cast<int32_t>(position_grad->rows) : 0;
  int32_t const least  = places * slices <= 2 * device_cus() ? 512 : 2048;
  int32_t const group  = std::max<int32_t>(least, static_cast<int32_t>((static_cast<int64_t>(view.rows) + 15) / 16));
  int32_t const groups = std::max<int32_t>(1, static_cast<int32_t>((static_cast<int64_t>(view.rows) + group - 1) / group));
  size_t const list    = static_cast<size_t>(n) * sizeof(uint32_t);
  TempParts<8> const temp(mr, {list, list, small ? 0 : list, small ? 0 : list, small ? 0 : static_cast<size_t>(counts + 1) * sizeof(uint32_t), direct ? 0 : scan_temp_bytes(counts),
                               static_cast<size_t>(2 * cols) * static_cast<size_t>(chunks > 1 ? chunks : 0) * sizeof(float),
                               groups > 1 ? static_cast<size_t>(groups) * static_cast<size_t>(places * cols) * sizeof(float) : 0});
  if (!temp.ok()) return fail(NVTEXT_AMD_ALLOC_FAILED, "temporary allocation failed");
  Sorted sorted{temp.part<uint32_t>(0), temp.part<uint32_t>(1)}, other{temp.part<uint32_t>(2), temp.part<uint32_t>(3)};
  if (chunks > 0) {
    ProfileScope const scope("embedding_sort", stream);
    Unsorted const column{view, vocabulary};
    auto const sort = [&](auto bits_of) {
      constexpr int kBits = decltype(bits_of)::value;
      if (small) {
        hipLaunchKernelGGL(small_sort_kernel<kBits>, dim3(1), dim3(kSortThreads), 0, stream, column, n, sorted);
        return;
      }
      uint32_t* const places_of = temp.part<uint32_t>(4);
      auto const pass           = [&](auto from, int shift, Sorted to) {
        using From = decltype(from);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(digit_counts_kernel<From, kBits>), dim3(tiles), dim3(kSortThreads), 0, stream, from, n, shift, tiles, !direct, places_of);
        if (!direct) device_exclusive_scan(Counts{places_of}, counts, places_of, temp.part<uint64_t>(5), stream, TellNobody{});
        hipLaunchKernelGGL(HIP_KERNEL_NAME(digit_place_kernel<From, kBits>), dim3(tiles), dim3(kSortThreads), 0, stream, from, n, shift, tiles, !direct, places_of, to);
      };
      pass(column, 0, sorted);
      for (int shift = kBits; shift < 32 && (vocabulary >> shift) != 0; shift += kBits) {
        pass(Half{sorted}, shift, other);
        std::swap(sorted, other);
      }
    };
    if (bits == 8)
      sort(std::integral_constant<int, 8>{});
    else if (bits == 9)
      sort(std::integral_constant<int, 9>{});
    else
      sort(std::integral_constant<int, 10>{});
    NVTEXT_HIP_TRY(hipGetLastError());  // (what comes next takes the sorted tokens for rows of grad)
  }
  with_type(grad->type, [&](auto zero) {
    using T         = decltype(zero);
    auto const sums = [&](auto result) {
      using G = decltype(result);
      Sums<T, G> const s{sorted, n, chunk, chunks, vocabulary, view, rows_of<const T>(grad), cols, rows_of<G>(token_grad), temp.part<float>(6), places, groups, group,
                         rows_of<G>(position_grad), temp.part<float>(7)};
      int64_t const of_chunks = (chunks + kSumWaves - 1) / kSumWaves;
      int64_t const all = slices * (static_cast<int64_t>(places) * groups + of_chunks + (static_cast<int64_t>(vocabulary) + kSumThreads - 1) / kSumThreads);
      if (all > 0) {
        ProfileScope const scope("embedding_sums", stream);
        dim3 const grid = grid_of(all, kSumThreads), threads(kSumThreads);
        if (vec == 4)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(embedding_sums_kernel<4, T, G>), grid, threads, 0, stream, s);
        else
          hipLaunchKernelGGL(HIP_KERNEL_NAME(embedding_sums_kernel<1, T, G>), grid, threads, 0, stream, s);
      }
      int64_t const joins = slices * ((chunks > 1 ? of_chunks : 0) + (groups > 1 ? (places + kSumWaves - 1) / kSumWaves : 0));
      if (joins > 0) {
        ProfileScope const scope("embedding_join", stream);
        Sums<T, G> some = s;
        if (chunks <= 1) some.chunks = 0;
        dim3 const grid = grid_of(joins, kSumThreads), threads(kSumThreads);
        if (vec == 4)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(embedding_join_kernel<4, T, G>), grid, threads, 0, stream, some);
        else
          hipLaunchKernelGGL(HIP_KERNEL_NAME(embedding_join_kernel<1, T, G>), grid, threads, 0, stream, some);
      }
    };
    if (token_grad->type == NVTEXT_AMD_TYPE_FLOAT32)
      sums(float{});
    else
      sums(zero);
  });
  NVTEXT_HIP_TRY(hipGetLastError());
  return NVTEXT_AMD_SUCCESS;
}

}  // extern "C"
