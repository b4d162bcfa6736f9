// gdn_recurrence_forward.cu -- prefill of the channelwise gated linear
// recurrence (mathematics and look-back: gdn_recurrence.cu).
#include "gdn_recurrence_tile.cuh"

namespace gdn {
namespace rec {

// Shape of a tile: 64 rows x 64 channels for 8 consumer warps, or with kPack
// the 128 channels that share a scale for 16.  A lane has 2 channels of 8
// consecutive rows, a warp's slot.  A stage of shared memory holds one half (64
// channels) of x, a and b, and afterwards, in place of rows that the same warp
// has read, what the first pass left: 16 bytes for each lane and row.  A tensor
// copy brings a plane of all 64 rows at a time; row copies lay a slot's rows of
// the three planes side by side, which fits the 16 bytes exactly.
template <typename E, Fetch kFetch, bool kPack>
struct FwdShape {
  static constexpr int kHalves = kPack ? 2 : 1;
  static constexpr int kCh = 64 * kHalves;
  static constexpr int kWorkers = kSlots * kHalves;       // consumer warps
  static constexpr int kThreads = 32 * (kWorkers + 1 + kHalves);
  static constexpr int kPitch = row_pitch<static_cast<int>(sizeof(E))>(kFetch);
  static constexpr int kRead = kFetch == kDirect ? 0 : 3 * kTokW * kPitch, kLeft = kTokW * 512;  // bytes of a slot
  static constexpr int kSlotStep = kFetch == kTmaTile ? kTokW * kPitch : kRead > kLeft ? kRead : kLeft;
  static constexpr int kPlane = kFetch == kTmaTile ? kRows * kPitch : kTokW * kPitch;
  // where a lane's 16 bytes of row i lie: kPerPlane rows in the slot's part of each plane
  static constexpr int kPerPlane = kFetch != kTmaTile ? kTokW : sizeof(E) == 4 ? 4 : 2;
  static constexpr int kHalfStage = kSlots * (kRead > kLeft ? kRead : kLeft);
  static constexpr int kStage = kHalves * kHalfStage;
  static constexpr int kStages = kHalfStage > 32768 ? 2 : 3;
  // The second pass is put off by a tile (8 x 4096 x 2048 bf16: 136 -> 120 us),
  // also where tensor copies have two stages only (65536 x 1024 fp32: 279 -> 209
  // us), but not with two stages of row copies, which wait for a stage longer.
  static constexpr bool kDefer = kStages > 2 || kFetch == kTmaTile;
  static constexpr int kCtas = kPack || kStages * kStage > 98304 ? 1 : 2;             // of an SM
};

struct Forward {
  CUtensorMap tx, ta, tb;  // kTmaTile
  const void *x, *a, *b;
  int64_t x_stride, a_stride, b_stride;  // elements from one token to the next
  const float *A_log, *dt_bias;
  const float *state;  // rows of D, or null: zeros
  Seqs s;
  int64_t D;
  void *out;       // [T, D], or null
  float *final;    // rows of D, or null; may be `state`
  float *carries;  // [T / 64][D up to 128s] states before every 64th row, or null
  uint8_t *packed; // 8-bit x, a, b (kPack)
  uint32_t skew[3][kTokW];  // kRowCopies: the byte at which row i (mod 8) of x, a, b starts in its place
  int zero_behind; // write zeros to out behind the last sequence
  Header *hdr;     // kChain
  uint64_t *maps, *states;  // kChain
  const float *dt, *c;      // kChain: prepared
  const float *aside;       // ... or null: the states are not updated in place
  const int *first;
};

struct Next {
  int64_t chunk;  // -1: no more tiles
  int64_t d;
};

template <typename Shape, bool kPack>
struct FwdShared {
  // maps of the slots' rows (A, A, H, H of a lane's channels); the chain warp
  // replaces them by the states that enter the slots
  float4 own[Shape::kStages][Shape::kHalves][kSlots][32];
  float params[Shape::kStages][2][Shape::kCh];  // kChain: dt and c of the tile's channels
  Table<kRows> tables[Shape::kStages];
  Tile tiles[Shape::kStages];
  Next next[Shape::kStages];      // kRowCopies: the tile that comes into a stage
  uint64_t posted[Shape::kStages];  // ... is known
  uint64_t full[Shape::kStages], ready[Shape::kStages], empty[Shape::kStages];
  uint64_t mapped[Shape::kStages][Shape::kHalves];  // the slots' maps are there
  uint64_t taken[Shape::kStages][Shape::kHalves];   // ... and have been read for the tile's
  uint64_t pair[kPack ? kSlots : 1];
  uint32_t amax[kPack ? 2 * kSlots * 64 : 1];
  alignas(16) float inverse[kPack ? Shape::kWorkers : 1][3 * kTokW];
  int broken;
};

// Roles of the warps, joined by mbarriers alone:
//   producer   takes tiles by ticket, fills the table, has the inputs copied.
//              Row copies are issued by the consumers, each warp for its own
//              rows as soon as it is done with a stage: 66 a tile would keep one
//              warp busy for 4000 cycles (47000 x 1021 fp16: 227 against 203 us).
//   consumers  first pass: gates; per row the state y from a zero start and the
//              product P of the gates so far, left in shared memory; the map
//              (P, y) of the slot, and the tile's, which is published.  Second
//              pass, one tile later (kDefer): out = y + P h, with h the state
//              that enters the slot.
//   chain      (one per half) looks back and hands each slot its state.  It has
//              the time of a first pass for that.
// Without kChain (short inputs, one launch) a CTA walks all chunks of its
// channels and the chain warp keeps the state.
//
// What bounds it: instructions, not memory.  8 x 4096 x 2048 bf16 takes 120 us
// (4.5 TB/s; 82 us at the rate of a copy): 37 warp instructions for 32 values,
// 2.2 a cycle of 4, the exponentials' pipe half busy.  256 sequences, 1.15 M x
// 1024 bf16: 1.90 ms, 5.0 TB/s.  One sequence of 65536 x 1024: 171 us in bf16,
// where a copy takes 82 and 128 links in series 109 (0.85 us each, see kGroupLen);
// 209 to 223 us in fp32 (4.9 TB/s).  With 8-bit copies 190
// us for 8 x 4096 x 2048 (3.9 TB/s), bound by integer work on groups and bytes.
// Rows that no tensor copy fits, 47000 x 1021 fp16: 191 us, 2.0 TB/s, bound by
// instructions (two 16-bit accesses for each pair of values, copies by address).
template <typename E, Fetch kFetch, bool kPack, bool kChain>
__global__ void __launch_bounds__(FwdShape<E, kFetch, kPack>::kThreads, FwdShape<E, kFetch, kPack>::kCtas)
recurrence_forward_kernel(const __grid_constant__ Forward p) {
  using S = FwdShape<E, kFetch, kPack>;
  constexpr bool kVec = kFetch == kTmaTile;
  constexpr int kElement = sizeof(E);
  constexpr int kCh = S::kCh, kStages = S::kStages;
  extern __shared__ __align__(1024) unsigned char smem[];
  FwdShared<S, kPack> &sh = *reinterpret_cast<FwdShared<S, kPack> *>(smem + kStages * S::kStage);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nt = static_cast<int>((p.D + kCh - 1) / kCh);

  if constexpr (kChain) {
    if (p.hdr->bad) return;
  } else {
    const int code = check_seqs(p.s);
    if (code) {
      if (tid == 0) set_device_status(code);
      return;
    }
  }
  if (tid == 0) {
    sh.broken = 0;
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&sh.full[i]), kFetch == kRowCopies ? 1 + 32 * S::kWorkers : 1);
      mbar_init(smem_u32(&sh.posted[i]), 1);
      for (int w = 0; w < S::kHalves; ++w) {
        mbar_init(smem_u32(&sh.mapped[i][w]), kSlots);
        mbar_init(smem_u32(&sh.taken[i][w]), 1);
      }
      mbar_init(smem_u32(&sh.ready[i]), S::kHalves);
      mbar_init(smem_u32(&sh.empty[i]), S::kWorkers);
    }
    if (kPack)
      for (int i = 0; i < kSlots; ++i) mbar_init(smem_u32(&sh.pair[i]), 2);
    mbar_init_fence();
  }
  __syncthreads();
  const int64_t total = p.s.total();
  const int64_t last = total > 0 ? (total - 1) / kRows : 0;
  const int group_len = kChain ? p.hdr->group : 1;  // 1 or kGroupLen
  uint64_t *const states = group_len == 1 ? p.maps : p.states;  // no maps are published then

  if (warp == S::kWorkers) {
    // ---- producer ----
    int64_t next = 0;  // !kChain: the next chunk
    // kChain: the stream that tickets are taken from, and those left after it
    int stream = 0, left_streams = 0;
    Stream st{};
    uint32_t ticket = 0;
    if constexpr (kChain) {
      left_streams = p.hdr->streams;
      stream = blockIdx.x % left_streams;
      st = p.hdr->stream[stream];
      if (lane == 0) ticket = atomicAdd(&p.hdr->stream[stream].ticket, 1u);
    }
    int k = 0;
    while (true) {
      int64_t chunk = -1;
      int d = blockIdx.x;
      bool only_map = false;
      if constexpr (kChain) {
        const int64_t t = __shfl_sync(0xffffffffu, ticket, 0);
        if (left_streams > 0) {
          const int64_t tiles = (st.to - st.from + st.only_map) * nt;
          if (t < tiles) {
            if (lane == 0) ticket = atomicAdd(&p.hdr->stream[stream].ticket, 1u);  // the next one, early
            chunk = st.from - st.only_map + t / nt;
            only_map = chunk < st.from;
            d = static_cast<int>(t % nt);
          } else if (--left_streams > 0) {
            stream = stream + 1 == p.hdr->streams ? 0 : stream + 1;
            st = p.hdr->stream[stream];
            if (lane == 0) ticket = atomicAdd(&p.hdr->stream[stream].ticket, 1u);
            continue;
          }
        }
      } else {
        if (next * kRows < max(p.s.T, int64_t{1})) chunk = next++;
      }
      const int64_t c0 = static_cast<int64_t>(d) * kCh, base = chunk * kRows;
      GDN_DCHECK(chunk < 0 || (d >= 0 && d < nt && base < max(p.s.T, int64_t{1})));
      if (chunk >= 0 && p.zero_behind && !only_map) {
        for (int64_t t = max(base, total); t < min(base + kRows, p.s.T); ++t)
#pragma unroll
          for (int w = 0; w < S::kHalves; ++w)
            store2<E, kVec>(static_cast<E *>(p.out) + t * p.D + c0 + 64 * w, lane,
                            static_cast<int>(min(p.D - c0 - 64 * w, int64_t{64})), 0);
      }
      if (chunk > last) continue;
      const int s = k % kStages;
      if constexpr (kFetch == kRowCopies) {
        // Consumers read an entry before they leave the stage's tile before it, so
        // the wait for `empty` below has covered the entry that this one replaces
        // -- but for a stage's first entry, which has been read when its copies
        // are there.
        const bool read = k < kStages || k >= 2 * kStages || wait_phase(smem_u32(&sh.full[s]), 0, &sh.broken);
        if (!__all_sync(0xffffffffu, read)) break;
        if (lane == 0) {
          sh.next[s] = Next{chunk, d};
          mbar_arrive(smem_u32(&sh.posted[s]));
        }
      }
      const bool go = k < kStages || wait_phase(smem_u32(&sh.empty[s]), ((k / kStages) - 1) & 1, &sh.broken);
      if (!__all_sync(0xffffffffu, go)) break;
      Table<kRows> &t = sh.tables[s];
      const uint32_t full = smem_u32(&sh.full[s]);
      if (chunk < 0) {
        if (lane == 0) {
          t.chunk = -1;
          sh.tiles[s].d = -1;
          mbar_arrive(full);
        }
        break;
      }
      uint64_t dt[S::kHalves], c[S::kHalves];
      if constexpr (kChain && kFetch == kRowCopies) {
#pragma unroll
        for (int w = 0; w < S::kHalves; ++w) {
          dt[w] = load2_f32<true>(p.dt + c0 + 64 * w, lane, 64);
          c[w] = load2_f32<true>(p.c + c0 + 64 * w, lane, 64);
        }
      }
      if (kChain && kFetch != kRowCopies && lane == 0) {
        mbar_expect_tx(full, 2 * kCh * 4);
        bulk_load(smem_u32(sh.params[s][0]), p.dt + c0, kCh * 4, full);
        bulk_load(smem_u32(sh.params[s][1]), p.c + c0, kCh * 4, full);
      }
      if (kFetch == kTmaTile && lane == 0) {
        mbar_expect_tx(full, S::kHalves * 3 * S::kPlane);
#pragma unroll
        for (int w = 0; w < S::kHalves; ++w) {
          const uint32_t dst = smem_u32(smem + s * S::kStage + w * S::kHalfStage);
          const int x = static_cast<int>(c0) + 64 * w, y = static_cast<int>(base);
          tma_load_2d(dst, &p.tx, x, y, full);
          tma_load_2d(dst + S::kPlane, &p.ta, x, y, full);
          tma_load_2d(dst + 2 * S::kPlane, &p.tb, x, y, full);
        }
      }
      const bool inside = fill_table<kRows>(p.s, t, base, chunk == last, lane, kChain ? p.first : nullptr, [&](int64_t n) {
        if (p.final == nullptr || only_map) return;  // an empty sequence's final state is its initial state
#pragma unroll
        for (int w = 0; w < S::kHalves; ++w) {
          const int left = static_cast<int>(min(p.D - c0 - 64 * w, int64_t{64}));
          const int64_t row = p.s.row(n) * p.D + c0 + 64 * w;
          store2_f32<kVec>(p.final + row, lane, left,
                           p.state != nullptr ? load2_f32<kVec>(p.state + row, lane, left) : 0);
        }
      });
      if constexpr (kChain && kFetch == kRowCopies) {
#pragma unroll
        for (int w = 0; w < S::kHalves; ++w) {
          store2_f32<true>(sh.params[s][0] + 64 * w, lane, 64, dt[w]);
          store2_f32<true>(sh.params[s][1] + 64 * w, lane, 64, c[w]);
        }
      }
      if (lane == 0) {
        t.chunk = chunk;
        t.d = d;
        t.last = chunk == last;
        t.only_map = only_map;
        t.cut = !kChain || p.aside == nullptr ? -1 : only_map ? st.opens : chunk == st.to - 1 ? st.cut : -1;
        t.valid = min(total - base, int64_t{kRows});
        const bool plain = inside && !only_map && base + kRows <= total && c0 + kCh <= p.D && p.out != nullptr;
        sh.tiles[s] = Tile{base * p.D + c0, d, plain ? 1 : 0};
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
      ++k;
    }
    // after a wait that ran out: no copy may be in flight when the CTA ends
    if (kFetch != kRowCopies && (kFetch != kDirect || kChain) && *static_cast<volatile int *>(&sh.broken))
      for (int i = max(k - kStages, 0); i < k; ++i)
        mbar_wait(smem_u32(&sh.full[i % kStages]), (i / kStages) & 1);
    return;
  }

  if (warp > S::kWorkers) {
    // ---- chain ----
    const int half = warp - S::kWorkers - 1;
    uint64_t h = 0;
    for (int k = 0;; ++k) {
      const int s = k % kStages;
      const uint32_t parity = (k / kStages) & 1;
      if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.full[s]), parity, &sh.broken))) return;
      const Table<kRows> &tab = sh.tables[s];
      const int64_t chunk = tab.chunk;
      if (chunk < 0) return;
      const bool last_chunk = tab.last, enters = !(tab.starts[0] & 1), only_map = tab.only_map;
      const int64_t lane_ch = static_cast<int64_t>(tab.d) * kCh + 64 * half + 2 * lane;
      const int64_t row_ch = static_cast<int64_t>(nt) * kCh;
      const int64_t group = group_len == 1 ? chunk : chunk / kGroupLen;
      const int place = group_len == 1 ? 0 : static_cast<int>(chunk % kGroupLen);
      const bool from_state = tab.reach > place;  // the sequence started before the group did
      const int before = from_state ? place : static_cast<int>(tab.reach);
      // the words that are wanted, asked for before the first pass is done: maps
      // of the chunks before, and the state that enters the first of them
      const bool looks = kChain && enters && !only_map;
      const bool groups = kChain && group_len > 1;
      // the words that are looked at are those of chunks before this one
      GDN_DCHECK(!looks || tab.valid <= 0 ||
                 (before >= 0 && before < kGroupLen && (from_state ? group >= 1 : before >= 1) && chunk - before >= 0));
      Words2 w[kGroupLen];
      auto src = [&](int j) {
        return j > 0 ? p.maps + (chunk - before + j - 1) * row_ch + lane_ch : states + (group - 1) * row_ch + lane_ch;
      };
      if constexpr (kChain) {
        w[0] = looks && from_state ? try_words2(src(0)) : Words2{0, 0};
        if (groups) {
#pragma unroll
          for (int j = 1; j < kGroupLen; ++j) w[j] = looks && j <= before ? try_words2(src(j)) : Words2{0, 0};
        }
      }
      if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.mapped[s][half]), parity, &sh.broken) &&
                                       wait_phase(smem_u32(&sh.taken[s][half]), parity, &sh.broken)))
        return;
      float4 *own = &sh.own[s][half][0][lane];
      const bool publishes = kChain && !last_chunk && !only_map && place == group_len - 1;
      if (kChain && !groups) {
        h = 0;
        if (looks && from_state) {
          Words2 one[1] = {w[0]};
          await_words2<1>(one, src, &sh.broken);
          h = one[0].map().H;
        }
      } else if (kChain) {
        Map2 all = get_map2(own, 0);
        if (publishes) {
#pragma unroll
          for (int i = 1; i < kSlots; ++i) all = compose2(all, get_map2(own + 32 * i, 0));
        }
        h = 0;
        if (looks) {
          await_words2<kGroupLen>(w, src, &sh.broken);
          if (from_state) h = w[0].map().H;
#pragma unroll
          for (int j = 1; j < kGroupLen; ++j)
            if (j <= before) h = apply2(w[j].map(), h);
        }
        // first what others wait for
        if (publishes) put_words2(states + group * row_ch + lane_ch, 0, apply2(all, h));
      }
      const uint64_t h_in = h;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        const Map2 m = get_map2(own + 32 * i, 0);
        *reinterpret_cast<uint64_t *>(own + 32 * i) = h;
        h = apply2(m, h);
      }
      if (publishes && !groups) put_words2(states + group * row_ch + lane_ch, 0, h);
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.ready[s]));
      if (p.carries != nullptr && !only_map)  // the table may hold another tile by now
        store2_f32<kVec>(p.carries + chunk * ((p.D + 127) / 128 * 128) + lane_ch - 2 * lane, lane, 64, h_in);
    }
  }

  // ---- consumers ----
  const int slot = warp / S::kHalves, half = warp % S::kHalves;
  const int row0 = slot * kTokW;
  unsigned char *const stage0 = smem + half * S::kHalfStage + slot * S::kSlotStep;
  Params2 par{};
  // kRowCopies: this warp's rows of the tile that comes into stage s next
  bool ended = kFetch != kRowCopies;
  Next next{};
  auto await_next = [&](int s, uint32_t parity) {
    if (ended) return true;
    if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.posted[s]), parity, &sh.broken))) return false;
    next = sh.next[s];
    return true;
  };
  auto copy_next = [&](int s) {
    if (ended) return;
    ended = next.chunk < 0;
    if (!ended) {
      const int64_t base = next.chunk * kRows + row0, c0 = next.d * kCh + 64 * half;
      const int rows = static_cast<int>(min(total - base, int64_t{kTokW}));
      const int left = static_cast<int>(min(p.D - c0, int64_t{64}));
      const uint32_t dst = smem_u32(stage0 + s * S::kStage);
      if (left > 0) {
        copy_rows<kElement>(dst, p.x, p.x_stride, base, rows, c0, left, lane);
        copy_rows<kElement>(dst + S::kPlane, p.a, p.a_stride, base, rows, c0, left, lane);
        copy_rows<kElement>(dst + 2 * S::kPlane, p.b, p.b_stride, base, rows, c0, left, lane);
      }
    }
    arrive_after_copies(smem_u32(&sh.full[s]));
  };
  // after a wait that ran out: no copy may be in flight when the CTA ends
  auto leave = [] {
    if (kFetch == kRowCopies) wait_copies();
  };
  // second pass over the tile of a stage; false if its wait ran out
  auto second_pass = [&](int s1, uint32_t parity1) {
    if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.ready[s1]), parity1, &sh.broken))) return false;
    const unsigned char *const src = stage0 + s1 * S::kStage + lane * 16;
    const uint64_t h = *reinterpret_cast<const uint64_t *>(&sh.own[s1][half][slot][lane]);
    auto kept = [&](int i) {
      return *reinterpret_cast<const ulonglong2 *>(src + i / S::kPerPlane * S::kPlane + i % S::kPerPlane * 512);
    };
    const Tile before = sh.tiles[s1];
    E *out = static_cast<E *>(p.out) + before.at + row0 * p.D + 64 * half;
    GDN_DCHECK(!before.plain || (before.at >= 0 && before.at + (kRows - 1) * p.D + kCh <= total * p.D));
    if (before.plain) {
#pragma unroll
      for (int i = 0; i < kTokW; ++i) {
        const ulonglong2 v = kept(i);
        store2<E, kVec>(out, lane, 64, f2_fma(v.y, h, v.x));
        out += p.D;
      }
    } else if (!sh.tables[s1].only_map) {
      const Table<kRows> &tab = sh.tables[s1];
      const int64_t c0 = static_cast<int64_t>(before.d) * kCh + 64 * half;
      const int left = static_cast<int>(min(p.D - c0, int64_t{64}));
      const int valid = static_cast<int>(max(int64_t{0}, min(int64_t{kTokW}, tab.valid - row0)));
      const unsigned starts = mask_bits(tab.starts, row0, kTokW), ends = mask_bits(tab.ends, row0, kTokW);
      const int first = starts ? __ffs(starts) - 1 : kTokW;
#pragma unroll
      for (int i = 0; i < kTokW; ++i) {
        const ulonglong2 v = kept(i);
        const uint64_t r = i < first ? f2_fma(v.y, h, v.x) : v.x;
        GDN_DCHECK(i >= valid || (tab.chunk * kRows + row0 + i < total && c0 < p.D + 64));
        GDN_DCHECK(!((ends >> i) & 1) || (i < valid && tab.end[row0 + i] >= 0 && tab.end[row0 + i] < p.s.N));
        if (p.out != nullptr && i < valid) store2<E, kVec>(out + i * p.D, lane, left, r);
        if (((ends >> i) & 1) && p.final != nullptr)
          store2_f32<kVec>(p.final + p.s.row(tab.end[row0 + i]) * p.D + c0, lane, left, r);
      }
    }
    if (kFetch == kTmaTile) fence_async_smem();  // this stage was written here; the next copy into it comes after
    if (!await_next(s1, parity1 ^ 1)) return false;
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.empty[s1]));
    copy_next(s1);
    return true;
  };
  if (!await_next(0, 0)) return leave();
  copy_next(0);
  int s = 0, s1 = 0, turn = 0;         // stages of this tile and the one before; whose turn to publish
  uint32_t parity = 0, parity1 = 0;    // ... and the phases of their barriers
  for (int k = 0;; ++k) {
    if (k + 1 < kStages) {
      if (!await_next(k + 1, 0)) return leave();
      copy_next(k + 1);
    }
    if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.full[s]), parity, &sh.broken))) return leave();
    const Tile tile = sh.tiles[s];
    if (tile.d >= 0) {
      // first pass
      const Table<kRows> &tab = sh.tables[s];
      const int64_t c0 = static_cast<int64_t>(tile.d) * kCh + 64 * half;
      if (kChain) {
        par = Params2{load2_f32<kVec>(sh.params[s][0] + 64 * half, lane, 64),
                      load2_f32<kVec>(sh.params[s][1] + 64 * half, lane, 64)};
      } else if (k == 0) {
        par = load_params2<kVec>(p.A_log + c0, p.dt_bias + c0, lane, static_cast<int>(min(p.D - c0, int64_t{64})));
      }
      unsigned char *const stage = stage0 + s * S::kStage;
      int valid = kTokW;
      unsigned starts = 0;
      if (!tile.plain) {
        valid = static_cast<int>(max(int64_t{0}, min(int64_t{kTokW}, tab.valid - row0)));
        starts = mask_bits(tab.starts, row0, kTokW);
      }
      Raw2<E> raw[3][kTokW];
      // row i of x, a or b
      auto fetch_row = [&](int w, int i) {
        const void *base = w == 0 ? p.x : w == 1 ? p.a : p.b;
        const int64_t stride = w == 0 ? p.x_stride : w == 1 ? p.a_stride : p.b_stride;
        if constexpr (kFetch == kDirect) {
          Raw2<E> r;
          r.v = {};
          if (i < valid)
            r = load2<E, kVec>(static_cast<const E *>(base) + (tab.chunk * kRows + row0 + i) * stride + c0, lane,
                               static_cast<int>(min(p.D - c0, int64_t{64})));
          return r;
        } else {
          const unsigned char *src = stage + w * S::kPlane + i * S::kPitch;
          if constexpr (kFetch == kRowCopies) src += p.skew[w][i];
          Raw2<E> r = fetch2<E, kVec>(src, lane);
          if constexpr (kPack && kFetch == kRowCopies) {  // what lies behind the row's end is no part of its group
            const int64_t left = p.D - c0;
            if (left < 64) r.v = (lane < left ? r.v & 0xffffu : 0u) | (lane + 32 < left ? r.v & 0xffff0000u : 0u);
          }
          return r;
        }
      };
#pragma unroll
      for (int w = 0; w < 3; ++w)
#pragma unroll
        for (int i = 0; i < kTokW; ++i) raw[w][i] = fetch_row(w, i);
      if constexpr (kPack) {
        // The groups' largest magnitudes: each half by one warp, joined through
        // shared memory.  Lane 8 w + i holds what belongs to row i of x, a or b.
        uint32_t mine = 0;
#pragma unroll
        for (int w = 0; w < 3; ++w) {
          const uint32_t m = row_maximum(raw[w], lane);
          if (lane / kTokW == w) mine = m;
        }
        uint32_t *amax = sh.amax + ((k & 1) * kSlots + slot) * 64;
        amax[32 * half + lane] = mine;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.pair[slot]));
        if (!__all_sync(0xffffffffu, wait_phase(smem_u32(&sh.pair[slot]), k & 1, &sh.broken))) return leave();
        asm volatile("" ::: "memory");
        const uint32_t ex =
            group_exponent(Raw2<E>::magnitude(max(mine, amax[32 * (half ^ 1) + lane])), exp_cap<E>());
        const int64_t t0 = tab.chunk * kRows + row0;
        GDN_DCHECK(t0 + valid <= p.s.T || valid == 0);
        const int left = static_cast<int>(min(p.D - c0, int64_t{64}));
        if (half == 0 && lane < 3 * kTokW && lane % kTokW < valid)
          p.packed[3 * p.s.T * p.D + (lane / kTokW * p.s.T + t0 + lane % kTokW) * nt + tile.d] =
              static_cast<uint8_t>(ex);
        if (tile.plain && __all_sync(0xffffffffu, ex < exp_cap<E>())) {
          // ordinary groups: one multiplication by the inverse scales, which
          // the lanes hand around through shared memory
          float *inv = sh.inverse[warp];
          if (lane < 3 * kTokW) inv[lane] = group_inverse(ex);
          __syncwarp();
#pragma unroll
          for (int w = 0; w < 3; ++w) {
            uint16_t *dst = reinterpret_cast<uint16_t *>(p.packed + (w * p.s.T + t0) * p.D + c0) + lane;
            float f[kTokW];
#pragma unroll
            for (int i = 0; i < kTokW; i += 4)
              *reinterpret_cast<float4 *>(f + i) = *reinterpret_cast<const float4 *>(inv + kTokW * w + i);
#pragma unroll
            for (int i = 0; i < kTokW; ++i) {
              const uint32_t q = quantise2(raw[w][i].pair(), f[i]);
              if constexpr (kVec) {
                *dst = static_cast<uint16_t>(q);
              } else {
                reinterpret_cast<uint8_t *>(dst - lane)[lane] = static_cast<uint8_t>(q);
                reinterpret_cast<uint8_t *>(dst - lane)[lane + 32] = static_cast<uint8_t>(q >> 8);
              }
              dst = reinterpret_cast<uint16_t *>(reinterpret_cast<uint8_t *>(dst) + p.D);
            }
          }
        } else {
#pragma unroll 1
          for (int w = 0; w < 3; ++w) {
            uint8_t *dst = p.packed + (w * p.s.T + t0) * p.D + c0;
#pragma unroll 1
            for (int i = 0; i < valid; ++i, dst += p.D) {
              const Raw2<E> r = fetch_row(w, i);
              const uint32_t q = quantise2(r.pair(), __shfl_sync(0xffffffffu, ex, kTokW * w + i), exp_cap<E>());
              if constexpr (kVec) {
                if (2 * lane < left) reinterpret_cast<uint16_t *>(dst)[lane] = static_cast<uint16_t>(q);
              } else {
                if (lane < left) dst[lane] = static_cast<uint8_t>(q);
                if (lane + 32 < left) dst[lane + 32] = static_cast<uint8_t>(q >> 8);
              }
            }
          }
        }
      }
      __syncwarp();  // the warp's rows are overwritten from here on
      auto keep = [&](int i, uint64_t y, uint64_t P) {
        *reinterpret_cast<ulonglong2 *>(stage + i / S::kPerPlane * S::kPlane + i % S::kPerPlane * 512 +
                                        lane * 16) = make_ulonglong2(y, P);
      };
      uint64_t P = f2_dup(1.f), y = 0;
      if (starts == 0 && valid == kTokW) {
#pragma unroll
        for (int i = 0; i < kTokW; ++i) {
          uint64_t g, u;
          gate_pair(raw[0][i].pair(), raw[1][i].pair(), raw[2][i].pair(), par.dt, par.c, g, u);
          P = f2_mul(P, g);
          y = f2_fma(g, y, u);
          keep(i, y, P);
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kTokW; ++i) {
          Raw2<E> r[3] = {raw[0][0], raw[1][0], raw[2][0]};
#pragma unroll
          for (int j = 1; j < kTokW; ++j)
            if (i == j) r[0] = raw[0][j], r[1] = raw[1][j], r[2] = raw[2][j];
          uint64_t g, u;
          gate_pair(r[0].pair(), r[1].pair(), r[2].pair(), par.dt, par.c, g, u);
          if (i >= valid) g = f2_dup(1.f), u = 0;
          if ((starts >> i) & 1) {  // y is the state itself from here on
            GDN_DCHECK(tab.start[row0 + i] >= 0 && tab.start[row0 + i] < p.s.N && tab.cut < kStreams);
            const int left = static_cast<int>(min(p.D - c0, int64_t{64}));
            const int row = row0 + i;
            // of a cut chunk the last sequence's was set aside if it goes on
            const bool goes_on = tab.cut >= 0 && !last_bits(tab.starts, row + 1) && !last_bits(tab.ends, row);
#ifdef GDN_DEBUG_CHECKS
            if (tab.only_map && !last_bits(tab.starts, row + 1)) delay(kMapOnlyDelayCycles);
#endif
            y = p.state == nullptr ? 0
                : goes_on          ? load2_f32<kVec>(p.aside + tab.cut * ((p.D + 127) / 128 * 128) + c0, lane, left)
                                   : load2_f32<kVec>(p.state + p.s.row(tab.start[row]) * p.D + c0, lane, left);
            P = f2_dup(-1.f);
          }
          P = f2_mul(P, g);
          y = f2_fma(g, y, u);
          keep(i, y, P);
        }
      }
      put_map2(&sh.own[s][half][slot][0], lane, Map2{P, y});
      __syncwarp();
      const uint32_t mapped = smem_u32(&sh.mapped[s][half]);
      if (lane == 0) mbar_arrive(mapped);
      if (slot == turn) {
        // the tile's map is published by the consumers, each warp in its turn,
        // so that it does not wait for the look-back of the tile before
        const bool group_end = group_len == 1 || tab.chunk % kGroupLen == kGroupLen - 1;
        if (kChain && !tab.last && (!group_end || tab.only_map)) {
          if (!__all_sync(0xffffffffu, wait_phase(mapped, parity, &sh.broken))) return leave();
          Map2 all = get_map2(&sh.own[s][half][0][0], lane);
#pragma unroll
          for (int i = 1; i < kSlots; ++i) all = compose2(all, get_map2(&sh.own[s][half][i][0], lane));
          const int64_t at = tile.d * kCh + 64 * half + 2 * lane;
          if (group_end)  // only_map: a sequence starts here, so the map is the state after it
            put_words2(states + (group_len == 1 ? tab.chunk : tab.chunk / kGroupLen) * nt * kCh + at, 0, all.H);
          else
            put_words2(p.maps + tab.chunk * nt * kCh + at, all.A, all.H);
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(smem_u32(&sh.taken[s][half]));
      }
      turn = turn + 1 == kSlots ? 0 : turn + 1;
    }
    if constexpr (S::kDefer) {
      if (k > 0 && !second_pass(s1, parity1)) return leave();
    } else {
      if (tile.d >= 0 && !second_pass(s, parity)) return leave();
    }
    if (tile.d < 0) return;
    s1 = s;
    parity1 = parity;
    if (++s == kStages) s = 0, parity ^= 1;
  }
}

// ---- launch ---------------------------------------------------------------------
// Inputs of up to this many chunks are walked by one CTA per 64 or 128 channels, in
// one launch without a look-back.  What that costs grows with the chunks, the more
// so where a chunk takes long; two launches take 20 to 30 us whatever they are.
// A call alone, inputs not in L2, 1024 channels (1021 where rows are copied), us in
// one launch and in two at the largest number of chunks that takes one, and at the
// next:
//                         one sequence                   four
//   2-byte                8  20.8, 21.0                  7  21.1, 23.4  8  25.1, 21.5
//   4-byte                5  21.1, 21.5  6  23.5, 21.4   4  21.0, 21.4  5  24.2, 23.5
//   2-byte, row by row    5  22.1, 21.5  6  24.9, 21.5   5  22.8, 25.5  6  26.1, 25.1
//   4-byte, row by row    3  17.9, 21.5  4  20.9, 19.4   3  19.1, 25.6  4  22.9, 23.6
// and with 8-bit copies
//   2-byte                3  24.3, 25.6  4  27.0, 27.0   3  27.1, 30.2  4  34.5, 25.6
//   4-byte                2  21.1, 27.1  3  26.9, 25.5   2  23.0, 25.6  3  30.3, 30.7
//   2-byte, row by row    2  25.0, 27.6  3  32.6, 29.2   2  26.2, 27.6  3  33.3, 35.8
//   4-byte, directly      1  21.2, 31.7  2  33.2, 31.0   1  22.7, 31.7  2  34.2, 34.7
// (2-byte, one sequence of 16 chunks, with both in L2: 26.7 against 17.8.)
// From 64 to 4096 channels both sides change by at most a few us.
template <typename E, Fetch kFetch, bool kPack>
constexpr int64_t serial_chunks(bool one_sequence) {
  constexpr bool kTwo = sizeof(E) == 2;
  if (kPack) return kFetch == kTmaTile ? (kTwo ? 3 : 2) : (kTwo ? 2 : 1);
  if (kFetch != kTmaTile) return kTwo ? 5 : 3;
  return (kTwo ? 7 : 4) + (one_sequence ? 1 : 0);
}
constexpr int64_t kSerialSeqs = 1024;  // each CTA checks all of cu_seqlens then

template <typename E, Fetch kFetch, bool kPack>
cudaError_t launch_forward_t(Forward p, void *workspace, int sms, cudaStream_t stream) {
  using S = FwdShape<E, kFetch, kPack>;
  const int64_t nt = (p.D + S::kCh - 1) / S::kCh, chunks = (max(p.s.T, int64_t{1}) - 1) / kRows + 1;
  constexpr int smem = S::kStages * S::kStage + static_cast<int>(sizeof(FwdShared<S, kPack>));
  static_assert(smem * S::kCtas <= 227 * 1024 - 1024 * (S::kCtas - 1), "CTAs of an SM share 228 KiB");
  if constexpr (kFetch == kRowCopies) {
    static_assert(kTokW * sizeof(E) % 16 == 0 && 64 * sizeof(E) % 16 == 0, "the same for all slots and tiles");
    const void *const base[3] = {p.x, p.a, p.b};
    const int64_t stride[3] = {p.x_stride, p.a_stride, p.b_stride};
    for (int w = 0; w < 3; ++w)
      for (int i = 0; i < kTokW; ++i)
        p.skew[w][i] = static_cast<uint32_t>(
            (reinterpret_cast<uintptr_t>(base[w]) + static_cast<uintptr_t>(i * stride[w]) * sizeof(E)) & 15);
  }
  if constexpr (kFetch == kTmaTile) {
    if (!make_row_map<E>(&p.tx, p.x, p.D, p.s.T, p.x_stride, 64, kRows) ||
        !make_row_map<E>(&p.ta, p.a, p.D, p.s.T, p.a_stride, 64, kRows) ||
        !make_row_map<E>(&p.tb, p.b, p.D, p.s.T, p.b_stride, 64, kRows))
      return cudaErrorInvalidValue;
  }
  const bool serial =
      chunks <= serial_chunks<E, kFetch, kPack>(p.s.N == 1) && (p.s.cu == nullptr || p.s.N <= kSerialSeqs);
  auto kernel = serial ? recurrence_forward_kernel<E, kFetch, kPack, false>
                       : recurrence_forward_kernel<E, kFetch, kPack, true>;
  static std::atomic<unsigned long long> allowed[2];
  if (cudaError_t e = allow_shared(kernel, smem, allowed[serial])) return e;
  int64_t blocks = nt;
  if (!serial) {
    p.hdr = static_cast<Header *>(workspace);
    const Places w = places(workspace, p.s.T, p.D);
    p.maps = w.words;
    p.states = p.maps + chunks * nt * S::kCh;
    p.dt = w.dt, p.c = w.c;
    p.aside = p.state != nullptr && p.state == p.final ? w.aside : nullptr;
    p.first = w.first;
    const int64_t words = (chunks + (chunks + kGroupLen - 1) / kGroupLen) * nt * S::kCh;
    const Prepared q{p.A_log,     p.dt_bias, w.dt,  w.c, p.D, w.first, chunks, kRows,
                     streams_for(nt, int64_t{sms} * S::kCtas), nt, int64_t{sms} * S::kCtas, false,
                     p.aside != nullptr ? p.state : nullptr, w.aside};
    if (cudaError_t e = launch_init(p.hdr, p.maps, words, p.s, q, stream)) return e;
    blocks = min(chunks * nt, int64_t{sms} * S::kCtas);
  }
  kernel<<<static_cast<unsigned>(blocks), S::kThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

template <typename E>
cudaError_t launch_forward_e(const Forward &p, bool tma, void *workspace, int sms, cudaStream_t stream) {
  constexpr Fetch kOther = sizeof(E) == 4 ? kDirect : kRowCopies;
  if (p.packed != nullptr)
    return tma ? launch_forward_t<E, kTmaTile, true>(p, workspace, sms, stream)
               : launch_forward_t<E, kOther, true>(p, workspace, sms, stream);
  return tma ? launch_forward_t<E, kTmaTile, false>(p, workspace, sms, stream)
             : launch_forward_t<E, kRowCopies, false>(p, workspace, sms, stream);
}

}  // namespace rec
}  // namespace gdn
