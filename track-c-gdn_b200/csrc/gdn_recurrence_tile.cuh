// gdn_recurrence_tile.cuh -- what the recurrence's forward and backward share
// beyond the arithmetic: sequences and their tables of starts and ends, pairs of
// channels, affine maps, and the words that chunks hand to one another.
#pragma once
#include <cuda.h>

#include <atomic>
#include <type_traits>

#include "gdn_context.cuh"
#include "gdn_recurrence.cuh"

namespace gdn {
namespace rec {

// Chunks joined through one published state: 8 where one sequence (or a few) has
// to be worked on by all CTAs at once -- a state then travels one link for 8
// chunks (65536 x 1024 bf16: 171 us with 128 links; groups of 4: 218 us, 0.85 for
// each of 256; of 16: 317 us, with more maps to fetch and apply for each tile) --
// and 1 where streams and
// tiles of channels together give most CTAs a tile of a chunk whose predecessor
// is done: then a state per chunk is all that is published.
constexpr int kGroupLen = 8;

constexpr int kTokW = 8;
constexpr int kSlots = 8;
constexpr int kRows = kTokW * kSlots;  // 64

// Sequences that start or end in a tile.
template <int kRows>
struct Table {
  int64_t chunk;  // -1: no more tiles
  int64_t valid;  // rows of the tile that belong to a sequence
  int64_t reach;  // chunks from here to where the sequence of the first row starts
  int64_t ahead;  // ... and to where that of the last row ends
  int d;
  int last;       // the last chunk
  int only_map;   // nothing but the tile's map is wanted
  int cut;        // the cut that goes through the chunk where states are updated in place, or -1
  uint32_t starts[kRows / 32], ends[kRows / 32];
  int start[kRows], end[kRows];  // the sequence, or -1
};

// What the consumers need of an ordinary tile: all rows belong to sequences that
// neither start nor end there, and all 64 channels of each half exist.
struct alignas(16) Tile {
  int64_t at;  // element of out where the tile begins
  int d;       // the tile's channels; -1: no more tiles
  int plain;
};

struct Seqs {
  const int64_t *cu;  // [N + 1], or null: N sequences of S tokens each
  int64_t N, T, S;
  const int32_t *slots;  // state row of a sequence, or null: its number
  int64_t pool;
  __device__ __forceinline__ int64_t at(int64_t n) const { return cu != nullptr ? cu[n] : n * S; }
  __device__ __forceinline__ int64_t row(int64_t n) const {
    GDN_DCHECK(n >= 0 && n < N);
    return slots != nullptr ? slots[n] : n;
  }
  __device__ __forceinline__ int64_t total() const { return cu != nullptr ? cu[N] : T; }
};

// The chunks are worked on as up to kStreams streams side by side, each a run of
// consecutive chunks cut where a sequence starts, so that a chunk's predecessor
// in the chain has usually long been finished when its turn comes; one sequence
// alone is one stream.  The cut may go through a chunk: that chunk belongs to
// the stream that ends with it, but its map is needed by the other from the
// start, and is worked out there once more (only_map).  Both publish the map in
// the same word, and neither waits for the other: they have to find the same
// bits whenever they run, so what they read must not change during the call
// (Prepared::aside).
constexpr int kStreams = 32;
struct Stream {
  int64_t from, to;  // chunks [from, to)
  uint32_t ticket;
  int only_map;      // 1: starts with the map of chunk from - 1 (backwards: to)
  int cut;           // forwards: the cut that goes through chunk to - 1, or -1
  int opens;         // forwards with only_map: the cut that goes through chunk from - 1
};
struct Header {
  uint32_t bad;      // cu_seqlens or slots are not valid: write nothing
  int streams;
  int group;         // chunks joined through one published state
  uint32_t pad;
  Stream stream[kStreams];
};
static_assert(sizeof(Header) <= 2048, "what follows starts 2048 bytes into the workspace");
constexpr size_t kHeaderBytes = 2048;

#ifdef GDN_DEBUG_CHECKS
// The debug build holds a map-only tile back (about 0.5 ms) before it reads the
// state that the last sequence of its chunk starts from: the others have by then
// usually finished that sequence, and a read of what they write shows.
constexpr long long kMapOnlyDelayCycles = 1ll << 20;
__device__ __forceinline__ void delay(long long cycles) {
  for (const long long t0 = clock64(); clock64() - t0 < cycles;) {
  }
}
#endif

// Checks cu_seqlens and slots with all threads of a CTA; returns the device
// status code of what is wrong, or 0.
__device__ __forceinline__ int check_seqs(const Seqs &s) {
  int bad_cu = 0, bad_slot = 0;
  if (s.cu != nullptr) {
    if (threadIdx.x == 0) bad_cu = s.cu[0] != 0 || s.cu[s.N] > s.T;
    for (int64_t n = threadIdx.x; n < s.N; n += blockDim.x) bad_cu |= s.cu[n] > s.cu[n + 1];
  }
  if (s.slots != nullptr)
    for (int64_t n = threadIdx.x; n < s.N; n += blockDim.x)
      bad_slot |= s.slots[n] < 0 || s.slots[n] >= s.pool;
  bad_cu = __syncthreads_or(bad_cu);
  bad_slot = __syncthreads_or(bad_slot);
  return bad_cu ? kDevStatusBadSeqlens : bad_slot ? kDevStatusBadSlot : 0;
}

// First n in [0, N] with at(n) >= v (N if none), by one thread.  Stays in [0, N]
// whatever cu_seqlens holds.
__device__ __forceinline__ int64_t first_by_halves(const Seqs &s, int64_t v) {
  if (s.cu == nullptr) return s.S > 0 ? min((v + s.S - 1) / s.S, s.N) : 0;
  int64_t lo = 0, hi = s.N;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (s.cu[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// What the init kernel prepares besides: the parameters of all channels (zeros up
// to a multiple of 128), and the first sequence that starts
// at or behind each chunk's first row.
struct Prepared {
  const float *A_log, *dt_bias;
  float *dt, *c;    // [D up to 128s] each
  int64_t D;
  int *first;       // [chunks + 1], or null
  int64_t chunks, rows;
  int streams;      // as many as wanted, at most kStreams
  int64_t tiles, ctas;  // of channels; that work at once
  bool backwards;   // the chain runs from the last chunk to the first
  // States that the call updates in place (else null): a sequence that starts
  // in a cut chunk and goes on behind it is finished by the stream that begins
  // there, perhaps before the stream before, or this one's own map of the chunk,
  // has read where it starts from.  That state is set aside, one row for each
  // cut, and both take it from there.
  const float *state;
  float *aside;     // [kStreams][D up to 128s]
};

// Forwards: the first chunk that begins where the first sequence does that starts
// from an even cut on, or after that.
__device__ __forceinline__ int64_t first_of_stream(const Seqs &s, int64_t chunks, int64_t rows, int i, int streams) {
  const int64_t n = first_by_halves(s, chunks * i / streams * rows);
  return i == 0 ? 0 : n < s.N ? (s.at(n) + rows - 1) / rows : chunks;
}

// Empties the words, prepares, and checks the sequences, before the tiles run.
__global__ void __launch_bounds__(1024) recurrence_init_kernel(Header *hdr, ulonglong2 *words, int64_t n,
                                                               const Seqs s, const Prepared q) {
  const ulonglong2 e = make_ulonglong2(kEmptyWord, kEmptyWord);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    words[i] = e;
  if (q.state != nullptr) {
    for (int i = 1 + blockIdx.x; i < q.streams; i += gridDim.x) {
      // the sequence that covers the first row behind the cut chunk
      const int64_t n = first_by_halves(s, first_of_stream(s, q.chunks, q.rows, i, q.streams) * q.rows) - 1;
      const int64_t row = n >= 0 ? s.row(n) : -1;
      if (row < 0 || (s.slots != nullptr && row >= s.pool)) continue;
      for (int64_t c = threadIdx.x; c < q.D; c += blockDim.x)
        q.aside[i * ((q.D + 127) / 128 * 128) + c] = q.state[row * q.D + c];
    }
  }
  const int64_t me = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t c = me; c < (q.D + 127) / 128 * 128; c += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    q.dt[c] = c < q.D ? param_dt(q.dt_bias[c]) : 0.f;
    q.c[c] = c < q.D ? param_c(q.A_log[c]) : 0.f;
  }
  if (q.first != nullptr) {
    for (int64_t k = me; k <= q.chunks; k += static_cast<int64_t>(gridDim.x) * blockDim.x)
      q.first[k] = static_cast<int>(first_by_halves(s, k * q.rows));
  }
  if (blockIdx.x == 0) {
    const int code = check_seqs(s);
    __shared__ int64_t from[kStreams];
    __shared__ int only_map[kStreams];
    const int i = threadIdx.x;
    if (i < q.streams) {
      // from an even cut on, where the next sequence starts: forwards the first
      // chunk that begins there or after it, backwards the last one to end there
      // or before it is the first of its stream
      const int64_t n = first_by_halves(s, q.chunks * i / q.streams * q.rows);
      const int64_t row = n < s.N ? s.at(n) : q.chunks * q.rows;
      from[i] = i == 0 ? 0 : (q.backwards ? row : row + q.rows - 1) / q.rows;
      // backwards: the chunk that the cut goes through belongs to the stream
      // above, and the one below needs its map.  Forwards: the same of the chunk
      // before, unless a sequence starts with the first row itself
      const int64_t first = from[i] * q.rows, m = first_by_halves(s, first);
      only_map[i] = i > 0 && (q.backwards ? row % q.rows != 0 : !(m < s.N && s.at(m) == first));
    }
    __syncthreads();
    if (i == 0) {
      int n = 1;
      int64_t prev = 0;
      hdr->stream[0] = Stream{0, q.chunks, 0, 0, -1, -1};
      for (int j = 1; j < q.streams; ++j)
        if (from[j] > prev && from[j] < q.chunks) {
          prev = from[j];
          hdr->stream[n - 1].to = from[j];
          if (q.backwards) hdr->stream[n - 1].only_map = only_map[j];
          if (!q.backwards && only_map[j]) hdr->stream[n - 1].cut = j;
          hdr->stream[n] = Stream{from[j], q.chunks, 0, q.backwards ? 0 : only_map[j], -1, j};
          ++n;
        }
      hdr->streams = n;
      hdr->group = 2 * n * q.tiles >= q.ctas ? 1 : kGroupLen;
      hdr->bad = code != 0;
      if (code) set_device_status(code);
    }
  }
}

// First n in [0, N] with at(n) >= v (N if none), by all lanes of a warp.
__device__ __forceinline__ int64_t first_at_or_after(const Seqs &s, int64_t v, int lane) {
  if (s.cu == nullptr) return s.S > 0 ? min((v + s.S - 1) / s.S, s.N) : 0;
  int64_t lo = 0, hi = s.N;
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, i = lo + (lane + 1) * step - 1;
    const int64_t k = __popc(__ballot_sync(0xffffffffu, i < hi && s.cu[i] < v));
    hi = min(hi, lo + (k + 1) * step - 1);
    lo += k * step;
  }
  return lo;
}

// Fills the table of the rows [base, base + kRows) with one warp; returns whether
// no sequence starts or ends there.  on_empty(n) is called by the whole warp for
// each sequence without tokens that lies there (the last chunk also has those
// behind the last token).  `first`: where the chunks' first sequences were
// prepared, else they are searched for.
template <int kRows, typename F>
__device__ __forceinline__ bool fill_table(const Seqs &s, Table<kRows> &t, int64_t base, bool last, int lane,
                                           const int *first, F on_empty) {
  const int64_t lo = first != nullptr ? first[base / kRows] : first_at_or_after(s, base, lane);
  GDN_DCHECK(base >= 0 && base < max(s.T, int64_t{1}) && lo >= 0 && lo <= s.N);
  // the sequence that covers the first row, if it does not start there
  if (lane == 0) t.reach = lo > 0 ? base / kRows - s.at(lo - 1) / kRows : 0;
  const int64_t next = lo < s.N ? s.at(lo) : s.total();
  if (!last && next > base + kRows) {
    if (lane == 0) t.ahead = (next - 1) / kRows - base / kRows;
    if (lane < kRows / 32) t.starts[lane] = t.ends[lane] = 0;
    return true;
  }
#pragma unroll
  for (int i = 0; i < kRows; i += 32) t.start[i + lane] = t.end[i + lane] = -1;
  const int64_t hi = last               ? s.N
                     : first != nullptr ? first[base / kRows + 1]
                                        : first_at_or_after(s, base + kRows, lane);
  GDN_DCHECK(hi >= lo && hi <= s.N && (last || hi < s.N || s.total() >= base + kRows));
  if (lane == 0) t.ahead = last ? 0 : (s.at(hi) - 1) / kRows - base / kRows;
  __syncwarp();
  for (int64_t n0 = max(lo - 1, int64_t{0}); n0 < hi; n0 += 32) {
    const int64_t n = n0 + lane;
    bool empty = false;
    if (n < hi) {
      const int64_t from = s.at(n), to = s.at(n + 1);
      empty = from == to && n >= lo;
      if (from < to) {
        if (from >= base && from < base + kRows) t.start[from - base] = static_cast<int>(n);
        if (to > base && to <= base + kRows) t.end[to - 1 - base] = static_cast<int>(n);
      }
    }
    unsigned m = __ballot_sync(0xffffffffu, empty);
    while (m) {
      on_empty(n0 + __ffs(m) - 1);
      m &= m - 1;
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kRows / 32; ++i) {
    const unsigned a = __ballot_sync(0xffffffffu, t.start[i * 32 + lane] >= 0);
    const unsigned b = __ballot_sync(0xffffffffu, t.end[i * 32 + lane] >= 0);
    if (lane == 0) t.starts[i] = a, t.ends[i] = b;
  }
  return false;
}
// the bits of rows [row, row + n) of a table's mask, n <= 16 and within one word
__device__ __forceinline__ unsigned mask_bits(const uint32_t *words, int row, int n) {
  return (words[row >> 5] >> (row & 31)) & ((1u << n) - 1u);
}

inline cudaError_t launch_init(Header *hdr, uint64_t *words, int64_t n, const Seqs &s, const Prepared &q,
                               cudaStream_t stream) {
  const int64_t blocks = min(int64_t{148 * 2}, (n / 2 + 1023) / 1024);
  recurrence_init_kernel<<<static_cast<unsigned>(max(blocks, int64_t{1})), 1024, 0, stream>>>(
      hdr, reinterpret_cast<ulonglong2 *>(words), n / 2, s, q);
  return cudaGetLastError();
}

// whether any bit from `row` on is set (row up to 64)
__device__ __forceinline__ bool last_bits(const uint32_t (&words)[2], int row) {
  const uint64_t m = static_cast<uint64_t>(words[1]) << 32 | words[0];
  return row < 64 && m >> row;
}

// ---- how inputs reach shared memory ------------------------------------------------
// kTmaTile: one tensor copy a plane, rows of 64 channels side by side.  It wants
// 16-byte rows.  kRowCopies: asynchronous copies of the 16-byte blocks that hold
// a row's 64 channels (blocks never leave the pages of the data that they hold,
// but hold up to 15 bytes before and behind it, perhaps of another buffer); the
// row then starts up to 15 bytes into its place.  A bulk copy a row instead
// took 49 cycles a row and was slower than loads without any stage (494 against
// 328 us, 47000 x 1021 fp16).  kDirect: none; the consumers load from global
// memory (4-byte types that are packed as well, whose rows with gaps do not fit).
enum Fetch { kDirect, kTmaTile, kRowCopies };
// arrivals that complete a stage: the producer's, and its lanes' copies
constexpr int fetch_arrivals(Fetch f) { return f == kRowCopies ? 33 : 1; }

// bytes from one row of a plane to the next
template <int kElement>
__host__ __device__ constexpr int row_pitch(Fetch f) {
  return 64 * kElement + (f == kRowCopies ? 16 : 0);
}

// Issues the copies of rows [t0, t0 + rows) x `left` channels of a plane by all
// lanes of a warp.
template <int kElement>
__device__ __forceinline__ void copy_rows(uint32_t dst, const void *base, int64_t stride, int64_t t0, int rows,
                                          int64_t c0, int left, int lane) {
  // 32 / kPieces rows at a time, a lane's piece of the row always the same
  constexpr int kPieces = row_pitch<kElement>(kRowCopies) / 16, kStep = 32 / kPieces;
  const int r0 = lane / kPieces, c = lane - r0 * kPieces;
  if (r0 >= kStep) return;
  uintptr_t at = reinterpret_cast<uintptr_t>(base) + ((t0 + r0) * stride + c0) * kElement;
  const int64_t step = kStep * stride * kElement;
  dst += 16 * lane;
  const int end = left * kElement - 16 * c;
#pragma unroll 1
  for (int r = r0; r < rows; r += kStep, at += step, dst += 16 * kStep * kPieces)
    if (static_cast<int>(at & 15) + end > 0)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"((at & ~uintptr_t{15}) + 16 * c)
                   : "memory");
}
// This lane's arrival on a stage's barrier when its copies so far are there.
__device__ __forceinline__ void arrive_after_copies(uint32_t mbar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(mbar) : "memory");
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// The byte at which row t starts in its place.
template <int kElement>
__device__ __forceinline__ uint32_t row_offset(const void *base, int64_t stride, int64_t t, int64_t c0) {
  return (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base)) +
          static_cast<uint32_t>(t * stride + c0) * static_cast<uint32_t>(kElement)) & 15u;
}

// ---- two channels of a lane -----------------------------------------------------
// With kVec neighbours (one access), else lane and lane + 32 of 64 channels.
template <typename E>
struct Raw2;
template <>
struct Raw2<__nv_bfloat16> {
  uint32_t v;
  // magnitudes as bits whose order is that of the values, the larger of two for
  // each half, and one as an fp32's bits
  __device__ __forceinline__ uint32_t magnitudes() const { return v & 0x7fff7fffu; }
  __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 m =
        __hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  }
  __device__ static __forceinline__ uint32_t magnitude(uint32_t m) { return m << 16; }
  __device__ __forceinline__ uint64_t pair() const { return f2_pack(bf16_lo(v), bf16_hi(v)); }
};
template <>
struct Raw2<__half> {
  uint32_t v;
  __device__ __forceinline__ uint32_t magnitudes() const { return v & 0x7fff7fffu; }
  __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 m = __hmax2_nan(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  }
  __device__ static __forceinline__ uint32_t magnitude(uint32_t m) {
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(m))));
  }
  __device__ __forceinline__ uint64_t pair() const {
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v));
    return f2_pack(a.x, a.y);
  }
};
template <>
struct Raw2<float> {
  float2 v;
  __device__ __forceinline__ uint32_t magnitudes() const {  // of both in one
    return max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu);
  }
  __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return max(a, b); }
  __device__ static __forceinline__ uint32_t magnitude(uint32_t m) { return m; }
  __device__ __forceinline__ uint64_t pair() const { return f2_pack(v.x, v.y); }
};

// The largest magnitude of row l % 8 over the warp's 64 channels, in lane l: each
// exchange halves the rows that a lane still holds, so 9 exchanges serve 8 rows
// where a redux per row takes 8 of a slower pipe.  8 x 4096 x 2048 bf16 with
// 8-bit copies: 202 -> 190 us, with the rows fetched once instead of twice.
template <typename E>
__device__ __forceinline__ uint32_t row_maximum(const Raw2<E> (&r)[kTokW], int lane) {
  static_assert(kTokW == 8, "three halvings");
  using R = Raw2<E>;
  uint32_t v[kTokW];
#pragma unroll
  for (int i = 0; i < kTokW; ++i) v[i] = r[i].magnitudes();
#pragma unroll
  for (int step = 4; step >= 1; step /= 2) {
    const bool high = lane & step;
#pragma unroll
    for (int j = 0; j < step; ++j) {
      const uint32_t given = __shfl_xor_sync(0xffffffffu, high ? v[j] : v[j + step], step);
      v[j] = R::larger(high ? v[j + step] : v[j], given);
    }
  }
#pragma unroll
  for (int step = 8; step <= 16; step *= 2) v[0] = R::larger(v[0], __shfl_xor_sync(0xffffffffu, v[0], step));
  if constexpr (sizeof(E) == 2) return R::larger(v[0], __byte_perm(v[0], v[0], 0x1032)) & 0xffffu;
  return v[0];
}

template <typename E, bool kVec>
__device__ __forceinline__ Raw2<E> load2(const E *p, int lane, int left) {
  Raw2<E> r;
  r.v = {};
  if constexpr (kVec) {
    if (2 * lane < left) r.v = __ldg(reinterpret_cast<const decltype(r.v) *>(p) + lane);
  } else {
    E e[2] = {E(0.f), E(0.f)};
    if (lane < left) e[0] = p[lane];
    if (lane + 32 < left) e[1] = p[lane + 32];
    memcpy(&r.v, e, sizeof(r.v));
  }
  return r;
}
template <typename E, bool kVec>
__device__ __forceinline__ void store2(E *p, int lane, int left, uint64_t a) {
  using V = decltype(Raw2<E>::v);
  V v;
  // the one rounding of a result: to nearest even
  if constexpr (std::is_same<E, float>::value) {
    v = make_float2(f2_lo(a), f2_hi(a));
  } else if constexpr (std::is_same<E, __half>::value) {
    const __half2 h = __floats2half2_rn(f2_lo(a), f2_hi(a));
    v = *reinterpret_cast<const uint32_t *>(&h);
  } else {
    v = pack_bf16x2(f2_lo(a), f2_hi(a));
  }
  if constexpr (kVec) {
    if (2 * lane < left) reinterpret_cast<V *>(p)[lane] = v;
  } else {
    E e[2];
    memcpy(e, &v, sizeof(v));
    if (lane < left) p[lane] = e[0];
    if (lane + 32 < left) p[lane + 32] = e[1];
  }
}
// fp32 rows (states, parameters); plain loads, since a state may be updated in place
template <bool kVec>
__device__ __forceinline__ uint64_t load2_f32(const float *p, int lane, int left) {
  if constexpr (kVec) {
    const float2 v = 2 * lane < left ? reinterpret_cast<const float2 *>(p)[lane] : make_float2(0.f, 0.f);
    return f2_pack(v.x, v.y);
  } else {
    return f2_pack(lane < left ? p[lane] : 0.f, lane + 32 < left ? p[lane + 32] : 0.f);
  }
}
template <bool kVec>
__device__ __forceinline__ void store2_f32(float *p, int lane, int left, uint64_t a) {
  if constexpr (kVec) {
    if (2 * lane < left) reinterpret_cast<float2 *>(p)[lane] = make_float2(f2_lo(a), f2_hi(a));
  } else {
    if (lane < left) p[lane] = f2_lo(a);
    if (lane + 32 < left) p[lane + 32] = f2_hi(a);
  }
}

// A lane's two channels of a row in shared memory: neighbours of an aligned row
// (kVec), else lane and lane + 32 of a row at `src` (aligned to an element).
template <typename E, bool kVec>
__device__ __forceinline__ Raw2<E> fetch2(const unsigned char *src, int lane) {
  Raw2<E> r;
  if constexpr (kVec) {
    r.v = reinterpret_cast<const decltype(r.v) *>(src)[lane];
  } else if constexpr (std::is_same<E, float>::value) {
    r.v = make_float2(reinterpret_cast<const float *>(src)[lane], reinterpret_cast<const float *>(src)[lane + 32]);
  } else {
    const uint16_t *p = reinterpret_cast<const uint16_t *>(src);
    r.v = static_cast<uint32_t>(p[lane]) | static_cast<uint32_t>(p[lane + 32]) << 16;
  }
  return r;
}

struct Params2 {
  uint64_t dt, c;
};
template <bool kVec>
__device__ __forceinline__ Params2 load_params2(const float *A_log, const float *dt_bias, int lane, int left) {
  const uint64_t a = load2_f32<kVec>(A_log, lane, left), d = load2_f32<kVec>(dt_bias, lane, left);
  return Params2{f2_pack(param_dt(f2_lo(d)), param_dt(f2_hi(d))), f2_pack(param_c(f2_lo(a)), param_c(f2_hi(a)))};
}

// ---- affine maps of two channels ---------------------------------------------------
struct Map2 {
  uint64_t A, H;
};
__device__ __forceinline__ uint64_t apply2(const Map2 &m, uint64_t h) {
  return f2_pack(apply(f2_lo(m.A), f2_lo(m.H), f2_lo(h)), apply(f2_hi(m.A), f2_hi(m.H), f2_hi(h)));
}
// `then` after `first`
__device__ __forceinline__ Map2 compose2(const Map2 &first, const Map2 &then) {
  const uint64_t A = f2_mul(then.A, first.A);
  return Map2{f2_pack(restarts(f2_lo(then.A)) ? f2_lo(then.A) : f2_lo(A),
                      restarts(f2_hi(then.A)) ? f2_hi(then.A) : f2_hi(A)),
              apply2(then, first.H)};
}
// in shared memory, a lane's two side by side as (A, A, H, H)
__device__ __forceinline__ void put_map2(float4 *row, int lane, const Map2 &m) {
  row[lane] = make_float4(f2_lo(m.A), f2_hi(m.A), f2_lo(m.H), f2_hi(m.H));
}
__device__ __forceinline__ Map2 get_map2(const float4 *row, int lane) {
  const float4 v = row[lane];
  return Map2{f2_pack(v.x, v.y), f2_pack(v.z, v.w)};
}

// ---- words of two channels -----------------------------------------------------------
__device__ __forceinline__ void put_words2(uint64_t *p, uint64_t lo, uint64_t hi) {
  const uint64_t a = keep_apart(f2_pack(f2_lo(lo), f2_lo(hi))), b = keep_apart(f2_pack(f2_hi(lo), f2_hi(hi)));
  asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(p), "l"(a), "l"(b) : "memory");
}
struct Words2 {
  uint64_t a, b;
  __device__ __forceinline__ bool there() const { return a != kEmptyWord && b != kEmptyWord; }
  __device__ __forceinline__ Map2 map() const {
    return Map2{f2_pack(f2_lo(a), f2_lo(b)), f2_pack(f2_hi(a), f2_hi(b))};
  }
};
__device__ __forceinline__ Words2 try_words2(const uint64_t *p) {
  Words2 w;
  asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(w.a), "=l"(w.b) : "l"(p) : "memory");
  return w;
}
// Asks again for those of a lane's words that are wanted and missing, all at
// once, until no lane of the warp misses any (bounded): one after the other each
// would cost a round trip to L2.  `src` gives the address of word j.  A wait
// that runs out records device status 2 and goes on with zeros, as do all later
// waits of the CTA.
template <int kMost, typename F>
__device__ __forceinline__ void await_words2(Words2 (&w)[kMost], F src, volatile int *broken) {
  const long long limit = wait_limit_cycles();
  long long t0 = 0;
  while (true) {
    bool missing = false;
#pragma unroll
    for (int j = 0; j < kMost; ++j) missing |= !w[j].there();
    if (!__any_sync(0xffffffffu, missing)) return;
    if (t0 == 0) t0 = clock64();
    if (__any_sync(0xffffffffu, *broken || clock64() - t0 > limit)) {
      if (!*broken) set_device_status(kDevStatusWaitTimeout);
      *broken = 1;
#pragma unroll
      for (int j = 0; j < kMost; ++j)
        if (!w[j].there()) w[j] = Words2{0, 0};
      return;
    }
#pragma unroll
    for (int j = 0; j < kMost; ++j)
      if (!w[j].there()) w[j] = try_words2(src(j));
  }
}

// Expects `bytes` more of asynchronous copies in the barrier's phase.
__device__ __forceinline__ void mbar_expect_tx(uint32_t mbar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(mbar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t mbar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(mbar) : "memory");
}

// Allows a kernel its dynamic shared memory.  That holds in the context it was
// asked for in: `last` is the one of the last call, which need not ask again.
template <typename K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<unsigned long long> &last) {
  const unsigned long long id = current_context_id();
  if (id != 0 && last.load(std::memory_order_acquire) == id) return cudaSuccess;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  last.store(id, std::memory_order_release);
  return cudaSuccess;
}

// ---- host ---------------------------------------------------------------------
template <typename E>
bool make_row_map(CUtensorMap *m, const void *base, int64_t channels, int64_t rows, int64_t stride, int box_x,
                  int box_y) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(channels), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * sizeof(E)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_x), static_cast<cuuint32_t>(box_y)};
  const cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType type = std::is_same<E, float>::value     ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<E, __half>::value  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                   : std::is_same<E, uint8_t>::value ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                                                     : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return enc(m, type, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The workspace: header, prepared parameters and first sequences, words (as
// many as the widest tiles need).
struct Places {
  float *dt, *c, *aside;
  int *first;
  uint64_t *words;
  size_t bytes;
};
inline int64_t tiles_of(int64_t D) { return (D + 127) / 128; }
inline int64_t chunks_of(int64_t T) { return T > 0 ? (T + kRows - 1) / kRows : 1; }
inline Places places(void *workspace, int64_t T, int64_t D) {
  const int64_t width = tiles_of(D) * 128, chunks = chunks_of(T);
  const size_t first = kHeaderBytes + (8 + 4 * kStreams) * width, words = first + (4 * (chunks + 1) + 15) / 16 * 16;
  char *w = static_cast<char *>(workspace);
  float *f = reinterpret_cast<float *>(w + kHeaderBytes);
  return Places{f, f + width, f + 2 * width, reinterpret_cast<int *>(w + first), reinterpret_cast<uint64_t *>(w + words),
                words + 8 * (chunks + (chunks + kGroupLen - 1) / kGroupLen) * width};
}

// Streams for nt tiles of channels on `ctas` CTAs: about two tiles of channels to a
// CTA of the stream, so that the chunk before is done when a tile's turn comes
// and there is a stream left to join for CTAs whose own has ended (1.1 M x 1024
// bf16 1951 us with half as many, 1897; backward of 47000 x 1024 294 and 272).
inline int streams_for(int64_t nt, int64_t ctas) {
  return static_cast<int>(max(int64_t{1}, min(int64_t{kStreams}, 2 * ctas / nt)));
}

}  // namespace rec
}  // namespace gdn
