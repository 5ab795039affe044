// Gated linear recurrence for gfx950: h[t] = a[t] h[t-1] + x[t] for every channel, its gradient, and
// the step of single tokens against a cache of states.
//
// Mathematics.  Row t is the affine map m_t(h) = a_t h + x_t; the maps of consecutive rows compose to
// a map of the same form, (A, H) after (A', H') = (A A', A H' + H), and composition is associative, so
// the recurrence is a scan along the rows, independent for every channel.  The gradient is the same
// scan from the last row to the first: with c the gradient of the state that enters row t + 1,
//   g_t = dout_t + c,  dx_t = g_t,  da_t = g_t h_{t-1} (times a_t when the gate is a logarithm),
//   c <- a_t g_t,
// starting from the gradient of the final state and ending in the gradient of the initial one.
//
// What bounds it: memory.  Each kernel reads and writes every array once, 6 to 20 bytes a value (a large
// copy reaches 6.0 TB/s on MI355X).  Measured: 131072 rows of 2048 channels, all 16-bit, 320 us, 5.0 TB/s;
// 8 x 4096 x 2560 with 32-bit logarithms as gates 159 us, 4.2 TB/s, and its gradient 249 us, 4.7 TB/s.  A
// short call is bound by the trips to memory one behind the other: 8192 rows of 4096 channels 56 us,
// 3.6 TB/s.
//
// Split.  A workgroup of 8 wavefronts takes a tile of 8 S rows by 64 VEC channels; wavefront w holds S
// consecutive rows of it in registers, a lane holds VEC neighbouring channels of each.  One pass over
// the registers gives the wavefront's map, LDS combines the wavefronts, a second pass replays the rows
// from the state that enters them and stores.  The rows of a sequence that span tiles are joined by
// tile descriptors: every tile publishes its map, the 8th of a group of 8 tiles the map of the group,
// the 64th of a super-group the state itself.  A tile reads at most one state, 7 group maps and 7 tile
// maps and folds them in the order of the rows: what is combined with what depends on the sizes alone,
// so results do not vary from run to run.
//
// The tile.  S is 16 rows for 16-bit arrays and 8 otherwise: 64 registers of a lane, which leaves two
// workgroups to a compute unit (128 registers at most).  Half the rows in twice the workgroups take 415 us
// instead of 336 for the long sequence (uniform gates): every halving of the rows doubles the tiles that
// wait for one another.  Measured in an earlier build, whose first passes took exp of every 16-bit gate and
// which took 408 us for the same rows: twice as many channels in half the rows 816; 80 registers, for three
// workgroups, spill: 491; a look-back that met in LDS, group maps behind tile maps: 459.
//
// Descriptors.  A map is one 64-bit word (A's bits << 32 | H's bits), stored inverted in a single
// relaxed agent-scope atomic; NaNs are stored as the canonical one, so no map is the word 0, which
// means "not there yet" and is what the clearing kernel leaves.
//
// Range.  A is a product of up to 1024 gates and leaves 32 bits where the states do not, so products have
// exponents of their own; plain ones took 313.5 us instead of 322 for the long sequence, 380 instead of
// 391 for the dense training pass.
//
// Sequences.  A row that begins a sequence takes its initial state by selection, never by a product
// with zero, so infinities and NaNs of one sequence stay in it.  Which predecessors a tile needs
// follows from the offsets alone, as does whether a published map begins anew.
#include "lm_types.h"

namespace tcd {

constexpr int kLinWaves = 8;
constexpr int kLinBlock = kLinWaves * kWave;
constexpr int kLinGroup = 8;   // tiles of a group, groups of a super-group
constexpr int kLinTicketWords = 32;
constexpr int kLinSuper = kLinGroup * kLinGroup;
constexpr int kLinChunk = THRUST_CDNA4_LINEAR_SCAN_CHUNK;
constexpr int64_t kLinMaxChannels = int64_t(1) << 28;  // a lane's offset in a row of maps is 32 bits of bytes

struct LinArgs {
  const void* gate;
  const void* x;
  void* out;               // backward: grad_x
  const void* grad_out;    // backward
  void* grad_gate;         // backward
  const float* init;
  float* final_state;      // backward: grad_init
  const float* grad_final; // backward
  float* states;
  const void* offsets;
  int64_t gate_bs, gate_rs, x_bs, x_rs, out_bs, out_rs, grad_bs, grad_rs, grad_gate_bs, grad_gate_rs;
  int64_t rows, channels;
  int sequences, offsets64, log_gate, clear_outside;
  int batch, ntiles, ncb;
  uint32_t* tickets;    // [batch][channel blocks], a cache line each
  uint64_t* tile_map;   // [batch][ntiles][channels]
  uint64_t* group_map;  // [batch][groups][channels]
  uint32_t* super_state;  // [batch][super-groups][channels]
  uint32_t* timeouts;     // waits that were given up
  uint32_t spin_limit;    // polls after which they are; seconds
  int publish_delay;
};

// ---------------------------------------------------------------------------------------
// Published maps
// ---------------------------------------------------------------------------------------
__device__ inline uint32_t canonical_bits(float v) { return v != v ? 0x7fc00000u : bit_cast<uint32_t>(v); }

// A product of factors, m 2^e, |m| < 1.  The product leaves the range of 32 bits where the states that it
// takes one to the other do not (160 gates of one half and a state of 1e30), so it has an exponent of its own;
// m is 0, infinite or NaN where a factor is.
struct Product {
  float m;
  int e;
};
__device__ inline void times(Product& p, float a) {
  p.m *= __builtin_amdgcn_frexp_mantf(a);  // of [1/2, 1): 16 of them, and 24 that are normalised, stay in range
  p.e += __builtin_amdgcn_frexp_expf(a);
}
__device__ inline Product normalised(Product p) {
  return Product{__builtin_amdgcn_frexp_mantf(p.m), p.e + __builtin_amdgcn_frexp_expf(p.m)};
}
// An exponent out of [kLowest + 1, kHighest - 1] takes every finite state but 0 to 0, or to infinity, and
// whatever follows leaves it there.
constexpr int kLowest = -511, kHighest = 510;
__device__ inline bool out_of_range(int e) { return (uint32_t)(e - kLowest - 1) >= (uint32_t)(kHighest - kLowest - 1); }
// b after a
__device__ inline Product join(Product a, Product b) { return Product{a.m * b.m, out_of_range(a.e) ? a.e : out_of_range(b.e) ? b.e : a.e + b.e}; }
// a h + x for a normalised product a
__device__ inline float apply(Product a, float h, float x) { return __builtin_amdgcn_ldexpf(a.m * h, a.e) + x; }

// A published product has 32 bits: a sign, 10 of the exponent, 21 of the mantissa behind its leading 1.  The
// two bits that a float has more go to the exponent; that costs 2^-22 relative, as much as four roundings of 32
// bits, for a hop of 64 rows or more, each of which rounds twice.
__device__ inline uint32_t product_bits(Product p) {
  p = normalised(p);
  const uint32_t u = bit_cast<uint32_t>(p.m), sign = u & 0x80000000u;
  const uint32_t r = ((u & 0x7fffffffu) + 1u + (u >> 2 & 1u)) >> 2;  // to nearest, ties to even: 126 << 21 and on, or 127 << 21
  int e = p.e + (int)(r >> 21) - 126;
  e = e < kLowest ? kLowest : e > kHighest ? kHighest : e;
  uint32_t v = (uint32_t)(e + 512) << 21 | (r & 0x1fffffu);  // 1 .. 1022 in the exponent's place
  if (p.m == 0.f) v = 0;
  if (!(__builtin_fabsf(p.m) < 1.f)) v = 1023u << 21 | (p.m != p.m ? 1u : 0u);
  return sign | v;
}
__device__ inline Product product_of(uint32_t v) {
  const uint32_t code = v >> 21 & 1023u;
  const uint32_t exponent = code == 0 ? 0u : code == 1023 ? 255u << 23 : 126u << 23;
  return Product{bit_cast<float>((v & 0x80000000u) | exponent | (v & 0x1fffffu) << 2), (int)code - 512};
}

struct Map {
  Product a;
  float h;
};
__device__ inline void publish_map(uint64_t* p, Map m) { st_agent(p, ~(((uint64_t)product_bits(m.a) << 32) | canonical_bits(m.h))); }

// ---------------------------------------------------------------------------------------
// Sequences of packed rows.  Everything here is the same in all lanes of a wavefront.  Offsets that
// do not ascend give meaningless results but no access outside the arrays.
// ---------------------------------------------------------------------------------------
__device__ inline int64_t offset_at(const LinArgs& p, int64_t j) {
  return p.offsets64 ? static_cast<const int64_t*>(p.offsets)[j] : (int64_t) static_cast<const int32_t*>(p.offsets)[j];
}

__device__ inline int64_t first_lane(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// The last sequence that begins at or before `row` (not empty if `row` is inside one), or -1.  64 offsets a step.
__device__ inline int sequence_of(const LinArgs& p, int64_t row) {
  const int lane = lane_id();
  int lo = 0, n = p.sequences + 1;  // the answer + 1 is the number of offsets <= row among lo .. lo + n - 1, plus lo
  while (n > kWave) {
    const int step = (n + kWave - 1) / kWave;
    const int at = lane * step;
    const bool below = at < n && offset_at(p, lo + at) <= row;
    const int full = __popcll(__ballot(below));
    if (full == 0) return lo - 1;
    const int skip = (full - 1) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  const bool below = lane < n && offset_at(p, lo + lane) <= row;
  return __builtin_amdgcn_readfirstlane(lo + __popcll(__ballot(below)) - 1);
}

// What a wavefront needs to know of its S rows: which of them are inside a sequence, begin one or end
// one (bit k: row r0 + k) and the sequence of the first of them.  In begins[l], of the wavefront's own in
// LDS, the row in which the l-th sequence from that one begins, from r0, in 32 bits, which hold it
// wherever it matters; a wavefront that sees more than 64 sequences searches.
struct RowSpan {
  uint32_t inside, heads, ends;
  int first_sequence;
  int64_t since;  // the row in which the first sequence begins
};
constexpr int kFarRow = 1 << 30;

__device__ inline int clamp_sequence(const LinArgs& p, int s) { return s >= p.sequences ? p.sequences - 1 : s < 0 ? 0 : s; }

template <int S, bool PACKED>
__device__ inline RowSpan row_span(const LinArgs& p, int b, int64_t r0, int* own) {
  RowSpan r{0, 0, 0, b, 0};
  const int64_t left = p.rows - r0;
  const int n = left <= 0 ? 0 : left < S ? (int)left : S;
  if (n == 0) return r;
  if constexpr (!PACKED) {
    r.inside = (uint32_t)((uint64_t(1) << n) - 1);
    r.heads = r0 == 0;
    r.ends = left <= S ? 1u << (n - 1) : 0u;
  } else {
    if (p.sequences == 0) return r;
    const int64_t end = first_lane(offset_at(p, p.sequences)) - r0;  // of the last sequence
    const int s = clamp_sequence(p, sequence_of(p, r0));
    r.first_sequence = s;
    const int hi = end < n ? (int)(end < 0 ? 0 : end) : n;
    int lo = 0;
    for (int64_t base = s; base <= p.sequences; base += kWave) {
      const int64_t j = base + lane_id();
      const int64_t row = j <= p.sequences ? offset_at(p, j) : INT64_MAX;
      const int64_t from = row - r0;
      const int begins = row >= r0 + kFarRow ? kFarRow : from < -1 ? -1 : (int)from;
      if (base == s) {
        own[lane_id()] = begins;
        r.since = first_lane(row);
        lo = __builtin_amdgcn_readfirstlane(begins) < 0 ? 0 : __builtin_amdgcn_readfirstlane(begins);
        if (lo >= hi) return r;
        r.inside = (uint32_t)((uint64_t(1) << hi) - 1) & ~(uint32_t)((uint64_t(1) << lo) - 1);
      }
      uint64_t edges = __ballot(begins >= lo && begins <= hi);
      while (edges) {
        const int k = __builtin_amdgcn_readlane(begins, __builtin_ctzll(edges));
        edges &= edges - 1;
        if (k < hi) r.heads |= 1u << k;
        if (k > lo) r.ends |= 1u << (k - 1);
      }
      if (__builtin_amdgcn_readlane(begins, kWave - 1) > hi) break;
    }
  }
  return r;
}
// the sequence that row r0 + k, which is inside one, belongs to; all lanes of the wavefront call
template <bool PACKED>
__device__ inline void to_sequence(const LinArgs& p, const RowSpan& span, const int* own, int64_t r0, int k, int& s) {
  if constexpr (PACKED) {
    const int n = __popcll(__ballot(own[lane_id()] <= k));
    s = clamp_sequence(p, n < kWave ? span.first_sequence + n - 1 : sequence_of(p, r0 + k));
  }
}

// A row's element c of this lane: the row's address is the same in all lanes and stays in scalar
// registers, what differs is 32 bits of offset.
template <class T>
__device__ inline T* at(T* row, uint32_t c) {
  using Byte = typename std::conditional<std::is_const<T>::value, const char, char>::type;
  return reinterpret_cast<T*>(reinterpret_cast<Byte*>(row) + c * (uint32_t)sizeof(T));
}

template <int VEC>
__device__ inline void load_state(const float* p, int64_t row, uint32_t c, float (&h)[VEC]) {
  if (p) {
    p = at(p + row, c);
#pragma unroll
    for (int j = 0; j < VEC; j++) h[j] = p[j];
  } else {
#pragma unroll
    for (int j = 0; j < VEC; j++) h[j] = 0.f;
  }
}
template <int VEC>
__device__ inline void store_state(float* p, int64_t row, uint32_t c, const float (&h)[VEC]) {
  p = at(p + row, c);
#pragma unroll
  for (int j = 0; j < VEC; j++) p[j] = h[j];
}

// ---------------------------------------------------------------------------------------
// The state that enters a tile.  "Logical" tiles and wavefronts are numbered in the direction of the
// scan: as the rows for the recurrence, from the last one for its gradient.
// ---------------------------------------------------------------------------------------
template <int CH>
struct LinShared {
  float m[kLinWaves][CH], h[kLinWaves][CH];  // maps of the tile's wavefronts, the factors normalised
  int e[kLinWaves][CH];
  float map_m[CH], map_h[CH];                // the map of the group's earlier tiles, likewise
  int map_e[CH];
  float carry[CH];                           // the state before them
  int in_group;                              // the sequence begins among them: map_h is a state, and all there is
  int anew[kLinWaves];  // wavefront: a sequence begins in it (its h is then a state)
  int64_t since;        // logical row in which the sequence of the tile's first row begins; -1: none comes in
  uint32_t ticket;
};

// One channel: the maps of the wavefronts w0, w0 + 1 .. w1 - 1 after (A, H)
template <int CH>
__device__ inline void fold(const LinShared<CH>& sm, int w0, int w1, int ch, Product& A, float& H) {
  for (int w = w0; w < w1; w++) {
    const Product a{sm.m[w][ch], sm.e[w][ch]};
    H = apply(a, H, sm.h[w][ch]);
    A.m *= a.m;
    A.e += a.e;
  }
}
__device__ inline Product map_factor(uint64_t word) { return product_of((uint32_t)(~word >> 32)); }
__device__ inline float map_shift(uint64_t word) { return bit_cast<float>((uint32_t)~word); }

// The state behind the group's earlier tiles
template <int CH>
__device__ inline float group_state(const LinShared<CH>& sm, int ch) {
  return sm.in_group ? sm.map_h[ch] : apply(Product{sm.map_m[ch], sm.map_e[ch]}, sm.carry[ch], sm.map_h[ch]);
}

// Waits until n words that start `stride` elements apart are published; they have been asked for once.
template <int N, class W>
__device__ inline void wait_words(const LinArgs& args, const W* p, int64_t stride, uint32_t c, W (&v)[N]) {
  // The ticket order makes every predecessor a running workgroup, so these waits end; the limit keeps a
  // mistake from hanging the device, and is counted (thrust_cdna4_lookback_timeouts); what was waited for
  // then reads as NaN.
  for (uint32_t spins = 0;; spins++) {
    bool all = true;
#pragma unroll
    for (int k = 0; k < N; k++) all = all && v[k] != 0;
    if (all) return;
    if (spins >= args.spin_limit) break;
    __builtin_amdgcn_s_sleep(1);
#pragma unroll
    for (int k = 0; k < N; k++)
      if (v[k] == 0) v[k] = ld_agent(at(p + k * stride, c));
  }
  atomicAdd(args.timeouts, 1u);
}

// Called by the whole workgroup after sm.m, sm.e, sm.h, sm.anew and sm.since are written and a barrier.
// `i`: logical tile of `nt`; `rows`: rows of a tile.  Leaves the map of the group's earlier tiles in
// sm.map_m, sm.map_e and sm.map_h and the state before them in sm.carry.  One half of the workgroup deals with the
// tiles of the group and the other with what lies before it, a thread for each channel; what a thread
// may wait for it asks for at once, so that maps which are there cost one trip to memory.
template <int VEC>
__device__ inline void tile_carry(LinShared<kWave * VEC>& sm, const LinArgs& p, int b, int64_t i, int64_t nt, int rows, int64_t block_c0) {
  constexpr int CH = kWave * VEC, N = kLinGroup - 1;
  const int ch = threadIdx.x % CH, role = __builtin_amdgcn_readfirstlane((int)threadIdx.x / CH);
  const int64_t C = p.channels, groups = ceil_div(nt, kLinGroup), supers = ceil_div(nt, kLinSuper);
  const bool publishes = i + 1 < nt;
  const int64_t since = first_lane(sm.since);
  const bool needs = since >= 0;                   // a sequence comes in from earlier tiles
  const int64_t first = needs ? since / rows : i;  // the tile it begins in
  const int64_t g = i / kLinGroup, base = g * kLinGroup, sg = g / kLinGroup, gbase = sg * kLinGroup, gfirst = first / kLinGroup;
  const bool in_group = needs && first >= base;
  const int64_t from = block_c0 + ch / VEC * VEC;
  const uint32_t chan = (uint32_t)((from + VEC > C ? C - VEC : from) + ch % VEC);
  int last_anew = -1;
#pragma unroll
  for (int v = 0; v < kLinWaves; v++)
    if (sm.anew[v]) last_anew = v;
  last_anew = __builtin_amdgcn_readfirstlane(last_anew);
  // the tile's own map after (A, H); folded again where it is needed again, which is rare, rather than
  // kept in registers over the waits
  auto tile_after = [&](Product A, float H) {
    Product own{1.f, 0};
    if (last_anew >= 0) H = sm.h[last_anew][ch];
    fold<CH>(sm, last_anew + 1, kLinWaves, ch, own, H);
    return Map{join(A, own), H};
  };
  const Product one{1.f, 0};
  if (role == 0 && from < C) {
    if (i == 0)
      for (int k = 0; k < p.publish_delay; k++) __builtin_amdgcn_s_sleep(127);  // test knob, 0 in normal use
    if (publishes) publish_map(at(p.tile_map + ((int64_t)b * nt + i) * C, chan), tile_after(one, 0.f));
    __builtin_amdgcn_sched_barrier(0);  // the folded maps' registers are free for the words that follow
    const uint64_t* maps = p.tile_map + ((int64_t)b * nt + base) * C;
    const int k0 = needs ? (int)(in_group ? first - base : 0) : N, k1 = (int)(i - base);
    uint64_t v[N];
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = k >= k0 && k < k1 ? ld_agent(at(maps + k * C, chan)) : ~uint64_t(0);
    wait_words(p, maps, C, chan, v);
    // (GA, GH): the map of the group's earlier tiles, or GH a state where the sequence begins among them
    Product GA = one;
    float GH = 0.f;
#pragma unroll
    for (int k = 0; k < N; k++) {
      if (k >= k0 && k < k1) {
        const Product a = map_factor(v[k]);
        const float h = map_shift(v[k]);
        GH = in_group && k == k0 ? h : apply(a, GH, h);
        GA = join(GA, a);
      }
    }
    if (publishes && i - base == N)
      publish_map(at(p.group_map + ((int64_t)b * groups + g) * C, chan), tile_after(GA, GH));
    GA = normalised(GA);
    sm.map_m[ch] = GA.m;
    sm.map_e[ch] = GA.e;
    sm.map_h[ch] = GH;
  } else if (role == 1 && from < C) {
    float H = 0.f;
    if (needs && !in_group) {
      const uint64_t* maps = p.group_map + ((int64_t)b * groups + gbase) * C;
      const uint32_t* states = p.super_state + ((int64_t)b * supers + sg - 1) * C;
      const bool from_super = gfirst < gbase;
      const int k0 = from_super ? 0 : (int)(gfirst - gbase), k1 = (int)(g - gbase);
      uint64_t v[N];
      uint32_t state[1] = {~0u};
#pragma unroll
      for (int k = 0; k < N; k++) v[k] = k >= k0 && k < k1 ? ld_agent(at(maps + k * C, chan)) : ~uint64_t(0);
      if (from_super) state[0] = ld_agent(at(states, chan));
      wait_words(p, maps, C, chan, v);
      wait_words(p, states, 0, chan, state);
      H = bit_cast<float>(~state[0]);
#pragma unroll
      for (int k = 0; k < N; k++) {
        if (k >= k0 && k < k1) {
          const float h = map_shift(v[k]);
          H = !from_super && k == k0 ? h : apply(map_factor(v[k]), H, h);
        }
      }
    }
    sm.carry[ch] = H;
  }
  if (threadIdx.x == 0) sm.in_group = in_group;
  __syncthreads();
  if (role == 0 && from < C && publishes && i % kLinSuper == kLinSuper - 1) {
    const float H = group_state(sm, ch);
    st_agent(at(p.super_state + ((int64_t)b * supers + sg) * C, chan), ~canonical_bits(tile_after(one, H).h));
  }
}

// The state that enters logical wavefront `lw` of the tile
template <int VEC>
__device__ inline void wave_carry(const LinShared<kWave * VEC>& sm, int lw, int lane, float (&h)[VEC]) {
  int last_anew = -1;
  for (int v = 0; v < lw; v++)
    if (sm.anew[v]) last_anew = v;
  last_anew = __builtin_amdgcn_readfirstlane(last_anew);
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    const int ch = lane * VEC + j;
    Product A{1.f, 0};
    h[j] = last_anew >= 0 ? sm.h[last_anew][ch] : group_state(sm, ch);
    fold<kWave * VEC>(sm, last_anew + 1, lw, ch, A, h[j]);
  }
}

// Which tile this workgroup takes.  Tiles wait for one another along the rows only, so every chain of
// tiles (a batch's block of channels) has a ticket of its own: a tile then only waits for running ones,
// and the tickets of a first generation of 512 workgroups, 14 ns each where they all take the same one,
// are taken side by side.  Without anything to wait for there are no tickets.
__device__ inline void take_lin_tile(const LinArgs& p, uint32_t* shared, int64_t& i, int& b, int& cb) {
  const uint32_t across = (uint32_t)p.batch * (uint32_t)p.ncb;
  // each row of workgroups serves every chain once, shifted by one from row to row, so that no chain
  // stays with one XCD (workgroup k runs on XCD k mod 8) and ends when the slowest of them does
  const uint32_t chain = (blockIdx.x + blockIdx.x / across) % across;
  cb = (int)(chain % (uint32_t)p.ncb);
  b = (int)(chain / (uint32_t)p.ncb);
  i = blockIdx.x / across;
  if (p.tickets) {
    if (threadIdx.x == 0) *shared = atomicAdd(p.tickets + (size_t)chain * kLinTicketWords, 1u);
    __syncthreads();
    i = (uint32_t)__builtin_amdgcn_readfirstlane((int)*shared);
  }
}

// States of sequences without rows: the final state is the initial one (the gradients likewise).
template <int VEC>
__device__ inline void empty_sequences(const LinArgs& p, int64_t i, const float* from, float* to, uint32_t c0, bool active) {
  const int w = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  for (int64_t s0 = (i * kLinWaves + w) * kWave; s0 < p.sequences; s0 += (int64_t)p.ntiles * kLinWaves * kWave) {
    const int64_t s = s0 + lane;
    uint64_t none = __ballot(s < p.sequences && offset_at(p, s) >= offset_at(p, s + 1));
    while (none) {
      const int64_t row = (s0 + __builtin_ctzll(none)) * p.channels;
      none &= none - 1;
      float h[VEC];
      load_state<VEC>(from, row, c0, h);
      if (active) store_state<VEC>(to, row, c0, h);
    }
  }
}

// 32-bit gates that are logarithms are replaced once, where they are; 16-bit ones, whose factors do not
// fit their place, are taken through exp in each pass of kernels of their own (LOG16; left to a test at
// run time the exponentials were computed for every gate and cost as much as the memory traffic).
template <class TG, int VEC, int S>
__device__ inline void gates_of_logarithms(const LinArgs& p, Pack<TG, VEC> (&gate)[S]) {
  if constexpr (sizeof(TG) == 4) {
    if (p.log_gate) {
#pragma unroll
      for (int k = 0; k < S; k++)
#pragma unroll
        for (int j = 0; j < VEC; j++) gate[k].w[j] = bit_cast<uint32_t>(expf(gate[k].value(j)));
    }
  }
}

// ---------------------------------------------------------------------------------------
// The recurrence
// ---------------------------------------------------------------------------------------
template <class TG, class TX, int VEC, int S, bool PACKED, bool LOG16>
__global__ __launch_bounds__(kLinBlock) void linear_scan_kernel(LinArgs p) {
  constexpr int CH = kWave * VEC, R = S * kLinWaves;
  __shared__ LinShared<CH> sm;
  __shared__ int begins[PACKED ? kLinWaves : 1][kWave];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  int64_t i;
  int b, cb;
  take_lin_tile(p, &sm.ticket, i, b, cb);
  const int64_t C = p.channels, block_c0 = (int64_t)cb * CH;
  // the last lane's vector ends with the last channel: it may repeat channels of the lane before it,
  // and stores the same values
  const int64_t from = block_c0 + lane * VEC;
  const bool active = from < C;
  const uint32_t c0 = (uint32_t)(from + VEC > C ? C - VEC : from);
  const int64_t r0 = i * R + w * S;
  const int64_t rows_left = p.rows - r0;
  const int left = rows_left < 0 ? 0 : rows_left < S ? (int)rows_left : S;  // of this wavefront's S

  const RowSpan span = row_span<S, PACKED>(p, b, r0, begins[PACKED ? w : 0]);  // before the loads of rows: a load that follows them waits for them
  Pack<TG, VEC> gate[S];
  Pack<TX, VEC> x[S];
  if (left > 0) {
    const TG* gp = static_cast<const TG*>(p.gate) + b * p.gate_bs + r0 * p.gate_rs;
    const TX* xp = static_cast<const TX*>(p.x) + b * p.x_bs + r0 * p.x_rs;
#pragma unroll
    for (int k = 0; k < S; k++) {
      gate[k] = load_pack<TG, VEC>(at(gp, c0));
      x[k] = load_pack<TX, VEC>(at(xp, c0));
      if (k + 1 < left) gp += p.gate_rs, xp += p.x_rs;  // behind the last row, that one again
    }
    gates_of_logarithms<TG, VEC, S>(p, gate);
  }
  auto gate_value = [&](const Pack<TG, VEC>& g, int j) { return LOG16 ? expf(g.value(j)) : g.value(j); };
  auto step = [&](int k, float (&h)[VEC], Product (&A)[VEC], int& s) {
    if (span.heads >> k & 1) {
      to_sequence<PACKED>(p, span, begins[PACKED ? w : 0], r0, k, s);
      load_state<VEC>(p.init, (int64_t)s * C, c0, h);
    }
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      const float a = gate_value(gate[k], j);
      h[j] = a * h[j] + x[k].value(j);
      times(A[j], a);
    }
  };
  float h[VEC];
  Product A[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) h[j] = 0.f, A[j] = Product{1.f, 0};
  int s = span.first_sequence;
#pragma unroll
  for (int k = 0; k < S; k++)
    if (span.inside >> k & 1) step(k, h, A, s);
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    const Product a = normalised(A[j]);
    sm.m[w][lane * VEC + j] = a.m;
    sm.e[w][lane * VEC + j] = a.e;
    sm.h[w][lane * VEC + j] = h[j];
  }
  if (lane == 0) sm.anew[w] = span.heads != 0;
  if (w == 0) {
    int64_t since = -1;
    if (!(span.heads & 1) && (span.inside & 1)) since = PACKED ? span.since : 0;
    if (lane == 0) sm.since = since < 0 || since > r0 ? -1 : since;
  }
  __syncthreads();
  if (p.ntiles > 1) {
    tile_carry<VEC>(sm, p, b, i, p.ntiles, R, block_c0);
  } else {
    if (tid < CH) sm.map_h[tid] = 0.f;
    if (tid == 0) sm.in_group = 1;
    __syncthreads();
  }

  wave_carry<VEC>(sm, w, lane, h);
  s = span.first_sequence;
  if (p.states && left > 0 && r0 % kLinChunk == 0 && active) {
    float first[VEC];
    if (span.heads & 1) load_state<VEC>(p.init, (int64_t)s * C, c0, first);
    store_state<VEC>(p.states, (b * ceil_div(p.rows, (int64_t)kLinChunk) + r0 / kLinChunk) * C, c0, span.heads & 1 ? first : h);
  }
  TX* out = static_cast<TX*>(p.out) + b * p.out_bs + r0 * p.out_rs;
#pragma unroll
  for (int k = 0; k < S; k++) forget(gate[k]), forget(x[k]);
#pragma unroll
  for (int k = 0; k < S; k++) {
    if (span.inside >> k & 1) {
      step(k, h, A, s);
      if (active) {
        store_pack<TX, VEC>(at(out + k * p.out_rs, c0), Pack<TX, VEC>::of(h));
        if (p.final_state && span.ends >> k & 1) store_state<VEC>(p.final_state, (int64_t)s * C, c0, h);
      }
    } else if (PACKED && p.clear_outside && k < left && active) {
      store_pack<TX, VEC>(at(out + k * p.out_rs, c0), Pack<TX, VEC>{});
    }
  }
  if (p.final_state) {
    if constexpr (PACKED) {
      empty_sequences<VEC>(p, i, p.init, p.final_state, c0, active);
    } else if (p.rows == 0 && w == 0) {
      load_state<VEC>(p.init, (int64_t)b * C, c0, h);
      if (active) store_state<VEC>(p.final_state, (int64_t)b * C, c0, h);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Its gradient.  A tile is one chunk: the state that enters it was kept by the recurrence, so the
// states of its rows are computed again, in 32 bits, from the gates and inputs, which costs no more
// memory traffic than reading the outputs would and does not differentiate their rounding.
// ---------------------------------------------------------------------------------------
template <class TG, class TX, int VEC, bool PACKED, bool LOG16>
__global__ __launch_bounds__(kLinBlock) __attribute__((amdgpu_waves_per_eu(4))) void linear_scan_backward_kernel(LinArgs p) {
  constexpr int S = kLinChunk / kLinWaves, CH = kWave * VEC, R = kLinChunk;
  __shared__ LinShared<CH> sm;
  __shared__ int begins[PACKED ? kLinWaves : 1][kWave];
  __shared__ float fwd[kLinWaves][CH], entering[CH];
  __shared__ int fwd_anew[kLinWaves];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int lw = kLinWaves - 1 - w;
  int64_t i;  // from the last tile
  int b, cb;
  take_lin_tile(p, &sm.ticket, i, b, cb);
  const int64_t tile = p.ntiles - 1 - i;
  const int64_t C = p.channels, block_c0 = (int64_t)cb * CH;
  const int64_t from = block_c0 + lane * VEC;
  const bool active = from < C;
  const uint32_t c0 = (uint32_t)(from + VEC > C ? C - VEC : from);
  const int64_t r0 = tile * R + w * S;
  const int64_t rows_left = p.rows - r0;
  const int left = rows_left < 0 ? 0 : rows_left < S ? (int)rows_left : S;  // of this wavefront's S

  const RowSpan span = row_span<S, PACKED>(p, b, r0, begins[PACKED ? w : 0]);  // before the loads of rows: a load that follows them waits for them
  Pack<TG, VEC> gate[S];
  Pack<TX, VEC> x[S], d[S];
  float h[VEC], enter[VEC] = {};
  if (left > 0) {
    const TG* gp = static_cast<const TG*>(p.gate) + b * p.gate_bs + r0 * p.gate_rs;
    const TX* xp = static_cast<const TX*>(p.x) + b * p.x_bs + r0 * p.x_rs;
    const TX* dp = static_cast<const TX*>(p.grad_out) + b * p.grad_bs + r0 * p.grad_rs;
#pragma unroll
    for (int k = 0; k < S; k++) {
      gate[k] = load_pack<TG, VEC>(at(gp, c0));
      x[k] = load_pack<TX, VEC>(at(xp, c0));
      d[k] = load_pack<TX, VEC>(at(dp, c0));
      if (k + 1 < left) gp += p.gate_rs, xp += p.x_rs, dp += p.grad_rs;
    }
    gates_of_logarithms<TG, VEC, S>(p, gate);
    if (w == 0) load_state<VEC>(p.states, (b * ceil_div(p.rows, (int64_t)kLinChunk) + tile) * C, c0, enter);
  }
  auto gate_value = [&](const Pack<TG, VEC>& g, int j) { return LOG16 ? expf(g.value(j)) : g.value(j); };
  // one row of the recurrence, and one of its gradient (c: in the gradient of the state after the row, out that of the one before)
  auto step = [&](int k, float (&hh)[VEC], int& s) {
    if (span.heads >> k & 1) {
      to_sequence<PACKED>(p, span, begins[PACKED ? w : 0], r0, k, s);
      load_state<VEC>(p.init, (int64_t)s * C, c0, hh);
    }
  };
  auto turn = [&](int k, float (&c)[VEC], int& s) {
    if (span.ends >> k & 1) {
      to_sequence<PACKED>(p, span, begins[PACKED ? w : 0], r0, k, s);
      load_state<VEC>(p.grad_final, (int64_t)s * C, c0, c);
    }
  };
  Product A[VEC];
  float c[VEC];
#pragma unroll
  for (int j = 0; j < VEC; j++) h[j] = 0.f, A[j] = Product{1.f, 0}, c[j] = 0.f;
  int s = span.first_sequence;
#pragma unroll
  for (int k = 0; k < S; k++) {
    if (span.inside >> k & 1) {
      step(k, h, s);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float a = gate_value(gate[k], j);
        h[j] = a * h[j] + x[k].value(j);
        times(A[j], a);
      }
    }
  }
  const int last_sequence = s;
#pragma unroll
  for (int k = S - 1; k >= 0; k--) {
    if (span.inside >> k & 1) {
      turn(k, c, s);
#pragma unroll
      for (int j = 0; j < VEC; j++) c[j] = gate_value(gate[k], j) * (d[k].value(j) + c[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < VEC; j++) {
    const Product a = normalised(A[j]);
    sm.m[lw][lane * VEC + j] = a.m;
    sm.e[lw][lane * VEC + j] = a.e;
    sm.h[lw][lane * VEC + j] = c[j];
    fwd[w][lane * VEC + j] = h[j];
    if (w == 0) entering[lane * VEC + j] = enter[j];
  }
  if (lane == 0) {
    sm.anew[lw] = span.ends != 0;
    fwd_anew[w] = span.heads != 0;
  }
  // the sequence of the tile's last row: in how many logical rows before this tile it begins (that is, ends)
  if (w == kLinWaves - 1) {
    int64_t since = -1;
    const int64_t logical = (int64_t)p.ntiles * R - 1;
    if (!(span.ends >> (S - 1) & 1) && (span.inside >> (S - 1) & 1)) {
      int64_t end = p.rows;
      if constexpr (PACKED) end = offset_at(p, last_sequence + 1);
      since = end > p.rows ? -1 : logical - (end - 1);
    }
    if (lane == 0) sm.since = since < 0 || since >= i * R ? -1 : since;
  }
  __syncthreads();
  if (p.ntiles > 1) {
    tile_carry<VEC>(sm, p, b, i, p.ntiles, R, block_c0);
  } else {
    if (tid < CH) sm.map_h[tid] = 0.f;
    if (tid == 0) sm.in_group = 1;
    __syncthreads();
  }

#pragma unroll
  for (int k = 0; k < S; k++) forget(gate[k]), forget(x[k]), forget(d[k]);
  // states before each row
  int last_anew = -1;
  for (int v = 0; v < w; v++)
    if (fwd_anew[v]) last_anew = v;
  last_anew = __builtin_amdgcn_readfirstlane(last_anew);
  if (left > 0) {
#pragma unroll
    for (int j = 0; j < VEC; j++) {
      const int ch = lane * VEC + j;
      h[j] = last_anew >= 0 ? fwd[last_anew][ch] : entering[ch];
      for (int v = last_anew + 1; v < w; v++) h[j] = apply(Product{sm.m[kLinWaves - 1 - v][ch], sm.e[kLinWaves - 1 - v][ch]}, h[j], fwd[v][ch]);
    }
  }
  float before[S][VEC];
  s = span.first_sequence;
#pragma unroll
  for (int k = 0; k < S; k++) {
    if (span.inside >> k & 1) {
      step(k, h, s);
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        before[k][j] = h[j];
        h[j] = gate_value(gate[k], j) * h[j] + x[k].value(j);
      }
    }
  }
  wave_carry<VEC>(sm, lw, lane, c);
  TG* grad_gate = static_cast<TG*>(p.grad_gate) + b * p.grad_gate_bs + r0 * p.grad_gate_rs;
  TX* grad_x = static_cast<TX*>(p.out) + b * p.out_bs + r0 * p.out_rs;
#pragma unroll
  for (int k = S - 1; k >= 0; k--) {
    if (span.inside >> k & 1) {
      turn(k, c, s);
      float dg[VEC], dx[VEC];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        const float a = gate_value(gate[k], j);
        const float g = d[k].value(j) + c[j];
        const float da = g * before[k][j];
        c[j] = a * g;
        dx[j] = g;
        dg[j] = p.log_gate ? da * a : da;
      }
      if (span.heads >> k & 1) to_sequence<PACKED>(p, span, begins[PACKED ? w : 0], r0, k, s);
      if (active) {
        store_pack<TX, VEC>(at(grad_x + k * p.out_rs, c0), Pack<TX, VEC>::of(dx));
        store_pack<TG, VEC>(at(grad_gate + k * p.grad_gate_rs, c0), Pack<TG, VEC>::of(dg));
        if (p.final_state && span.heads >> k & 1) store_state<VEC>(p.final_state, (int64_t)s * C, c0, c);
      }
    } else if (PACKED && p.clear_outside && k < left && active) {
      store_pack<TX, VEC>(at(grad_x + k * p.out_rs, c0), Pack<TX, VEC>{});
      store_pack<TG, VEC>(at(grad_gate + k * p.grad_gate_rs, c0), Pack<TG, VEC>{});
    }
  }
  if (p.final_state) {
    if constexpr (PACKED) {
      empty_sequences<VEC>(p, i, p.grad_final, p.final_state, c0, active);
    } else if (p.rows == 0 && w == 0) {
      load_state<VEC>(p.grad_final, (int64_t)b * C, c0, h);
      if (active) store_state<VEC>(p.final_state, (int64_t)b * C, c0, h);
    }
  }
}

// ---------------------------------------------------------------------------------------
// One token for each of a batch: state[slot] = a state[slot] + x, out = state.  Rows of one slot are
// taken in their order: the first of them does all, the others leave.  What bounds it is memory: 2048
// rows of 8192 16-bit channels take 46 us, 5.1 TB/s.  To know whether a row is the first of its slot a
// workgroup reads all slots, 16 bytes a thread; with one wavefront reading 4 bytes a lane, and four
// times as many workgroups, the same batch took 89 us.  So a thread takes UNITS = 4 vectors where that
// leaves two workgroups to a compute unit, and one in a small batch (8 x 1024: 3.7 us on the device).  The
// slots read grow with the square of the batch: 16384 rows of 1024 channels take 115 us, 53 without slots;
// 65536 rows 1027 and 174.
// ---------------------------------------------------------------------------------------
constexpr int kStepBlock = 256;
constexpr int kStepWide = 4;  // vectors a thread takes in a large batch

template <class TG, class TX, int UNITS, bool LOG>
__global__ __launch_bounds__(kStepBlock) void linear_scan_step_kernel(const TG* gate, int64_t gate_rs, const TX* x, int64_t x_rs, TX* out,
                                                                      int64_t out_rs, float* state, int64_t num_slots, const int32_t* slots,
                                                                      int batch, int64_t C, int ncb) {
  constexpr int VEC = 4;
  __shared__ int s_found[kStepBlock / kWave];  // bit 0: an earlier row of this slot, bit 1: a later one
  const int tid = threadIdx.x;
  const int row = (int)(blockIdx.x / (unsigned)ncb), cb = (int)(blockIdx.x % (unsigned)ncb);
  const int slot = slots ? slots[row] : row;
  uint32_t c0[UNITS];
  int n[UNITS];  // channels of each vector; 0: none
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    const int64_t from = (((int64_t)cb * UNITS + u) * kStepBlock + tid) * VEC;
    n[u] = C - from >= VEC ? VEC : C - from > 0 ? (int)(C - from) : 0;
    c0[u] = (uint32_t)from;
  }
  auto load = [&](auto* p, int u) {
    using T = typename std::remove_cv<typename std::remove_pointer<decltype(p)>::type>::type;
    if (n[u] == VEC) return load_pack<T, VEC>(at(p, c0[u]));
    return n[u] ? load_part<T, VEC>(at(p, c0[u]), n[u]) : Pack<T, VEC>{};
  };
  auto store = [&](auto* p, int u, const auto& v) {
    if (n[u] == VEC) store_pack(at(p, c0[u]), v);
    else if (n[u]) store_part(at(p, c0[u]), v, n[u]);
  };
  if (slot < 0 || slot >= num_slots) {  // a padded row
#pragma unroll
    for (int u = 0; u < UNITS; u++) store(out + (int64_t)row * out_rs, u, Pack<TX, VEC>{});
    return;
  }
  // Asked for before it is known that the row is the first of its slot: one that is not may read the state
  // while the first replaces it, and leaves without using what it read.
  float* own = state + (int64_t)slot * C;
  Pack<TG, VEC> g[UNITS];
  Pack<TX, VEC> v[UNITS];
  Pack<float, VEC> old[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    old[u] = load(own, u);
    g[u] = load(gate + (int64_t)row * gate_rs, u);
    v[u] = load(x + (int64_t)row * x_rs, u);
  }
  int found = 0;
  if (slots) {
    int mine = 0;
    auto look = [&](int q, int s) { mine |= s == slot ? (q < row ? 1 : q > row ? 2 : 0) : 0; };
    for (int q = tid * 4; q < batch; q += kStepBlock * 4) {
      if (q + 4 <= batch) {
        const tcd_v4u s = *reinterpret_cast<const tcd_v4u_anywhere*>(slots + q);
#pragma unroll
        for (int k = 0; k < 4; k++) look(q + k, (int)s[k]);
      } else {
        for (int k = q; k < batch; k++) look(k, slots[k]);
      }
    }
    const uint64_t earlier = __ballot(mine & 1), later = __ballot(mine & 2);
    if (tid % kWave == 0) s_found[tid / kWave] = (earlier != 0) | (later != 0) << 1;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStepBlock / kWave; w++) found |= s_found[w];
    if (found & 1) return;
  }
  float h[UNITS][VEC];
#pragma unroll
  for (int u = 0; u < UNITS; u++)
#pragma unroll
    for (int j = 0; j < VEC; j++) h[u][j] = old[u].value(j);
  auto one = [&](int q) {
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
#pragma unroll
      for (int j = 0; j < VEC; j++) h[u][j] = (LOG ? expf(g[u].value(j)) : g[u].value(j)) * h[u][j] + v[u].value(j);
      store(out + (int64_t)q * out_rs, u, Pack<TX, VEC>::of(h[u]));
    }
  };
  one(row);
  if (found & 2) {
    for (int q = row + 1; q < batch; q++) {
      if (slots[q] != slot) continue;
#pragma unroll
      for (int u = 0; u < UNITS; u++) {
        g[u] = load(gate + (int64_t)q * gate_rs, u);
        v[u] = load(x + (int64_t)q * x_rs, u);
      }
      one(q);
    }
  }
#pragma unroll
  for (int u = 0; u < UNITS; u++) store(own, u, Pack<float, VEC>::of(h[u]));
}

// ---------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------
// (gate, x) types: the same, or 32-bit gates with 16-bit inputs
template <class F>
inline bool dispatch_activation(int gate, int x, F&& f) {
  if (gate == THRUST_CDNA4_F32 && x == THRUST_CDNA4_F32) return f(float{}, float{}), true;
  if (gate == THRUST_CDNA4_F16 && x == THRUST_CDNA4_F16) return f(f16_t{}, f16_t{}), true;
  if (gate == THRUST_CDNA4_BF16 && x == THRUST_CDNA4_BF16) return f(bf16_t{}, bf16_t{}), true;
  if (gate == THRUST_CDNA4_F32 && x == THRUST_CDNA4_F16) return f(float{}, f16_t{}), true;
  if (gate == THRUST_CDNA4_F32 && x == THRUST_CDNA4_BF16) return f(float{}, bf16_t{}), true;
  return false;
}

struct LinPlan {
  int vec, ncb;
  int64_t ntiles;
  size_t tile_at, group_at, super_at, bytes, clear;
};

inline bool lin_plan(int64_t batch, int64_t rows, int64_t channels, int tile_rows, int vec, LinPlan& l) {
  l.vec = vec;
  const int64_t ncb = ceil_div(channels, (int64_t)kWave * l.vec);
  l.ntiles = rows > 0 ? ceil_div(rows, (int64_t)tile_rows) : 1;
  const double grid = (double)ncb * (double)batch * (double)l.ntiles;
  if (grid * kLinBlock >= 4294967296.0) return false;  // a launch counts its threads in 32 bits
  l.ncb = (int)ncb;
  l.bytes = 256;
  l.clear = 0;
  if (l.ntiles > 1) {
    const size_t across = (size_t)batch * (size_t)channels;
    l.tile_at = align_up((size_t)batch * (size_t)ncb * kLinTicketWords * 4, 256);
    l.group_at = l.tile_at + align_up(across * (size_t)l.ntiles * 8, 256);
    l.super_at = l.group_at + align_up(across * (size_t)ceil_div(l.ntiles, (int64_t)kLinGroup) * 8, 256);
    l.bytes = l.super_at + align_up(across * (size_t)ceil_div(l.ntiles, (int64_t)kLinSuper) * 4, 256);
    l.clear = l.bytes;
  }
  return true;
}

inline hipError_t lin_storage(LinArgs& p, const LinPlan& l, void* temp) {
  p.ntiles = (int)l.ntiles;
  p.ncb = l.ncb;
  p.tickets = nullptr;
  if (l.ntiles > 1) {
    char* t = static_cast<char*>(temp);
    p.tickets = reinterpret_cast<uint32_t*>(t);
    p.tile_map = reinterpret_cast<uint64_t*>(t + l.tile_at);
    p.group_map = reinterpret_cast<uint64_t*>(t + l.group_at);
    p.super_state = reinterpret_cast<uint32_t*>(t + l.super_at);
    p.spin_limit = lookback_spin_limit();
    p.publish_delay = lookback_test_publish_delay();
    return lookback_timeout_counter(&p.timeouts);
  }
  return hipSuccess;
}

// rows of the recurrence's tile: the payload of a lane is 64 registers at most
template <class TG, class TX>
constexpr int lin_rows_per_wave() { return sizeof(TG) == 2 && sizeof(TX) == 2 ? 16 : 8; }

inline bool valid_shape(int64_t batch, int64_t rows, int64_t channels, int64_t sequences, const void* offsets, int offset_bytes) {
  if (batch < 0 || rows < 0 || channels < 0 || channels > kLinMaxChannels || batch > 0x7fffffff) return false;
  if (offsets || offset_bytes) return batch == 1 && (offset_bytes == 4 || offset_bytes == 8) && sequences >= 0 && sequences < 0x7fffffff;
  return true;
}

// the bytes that rows of this shape and these strides span (strides are not negative)
inline size_t span_bytes(int64_t batch, int64_t rows, int64_t channels, int64_t bs, int64_t rs, int elem) {
  if (batch == 0 || rows == 0 || channels == 0) return 0;
  return (size_t)((batch - 1) * bs + (rows - 1) * rs + channels) * (size_t)elem;
}

// whether rows of `row` bytes, `pitch` >= 0 apart, meet [b, b + nb)
inline bool rows_meet(const void* a, int64_t rows, int64_t pitch, size_t row, const void* b, size_t nb) {
  const uintptr_t first = reinterpret_cast<uintptr_t>(a), lo = reinterpret_cast<uintptr_t>(b);
  if (rows <= 0 || row == 0 || nb == 0 || first >= lo + nb) return false;
  if (first + row > lo) return true;
  if (pitch <= 0) return false;
  const uintptr_t k = (lo - first - row) / (uintptr_t)pitch + 1;  // the first row that ends behind lo
  return k < (uintptr_t)rows && first + k * (uintptr_t)pitch < lo + nb;
}

// Four channels a lane where more than half of a wavefront's lanes find work, one otherwise.  Training pass
// of 60000 rows, us with one channel a lane and with four (two in the gradient of 32-bit arrays):
//   channels            64         128        160        192        256        512
//   16-bit            71,  87    86,  91   112,  93   111,  94   134,  99   232, 151
//   f32 gates, bf16   85,  98    94, 103   121, 106   122, 109   145, 120   263, 185
//   32-bit            92,  92    92, 102   111, 125   118, 129   151, 141   262, 239
// An output over an input allows four only where no vector reaches over a workgroup's channels: the
// neighbour may have replaced what it repeats.  32768 x 2047 in place takes 161 us so, into a new array 122;
// in 32 bits 245 and 185.
inline bool lin_narrow(int64_t channels, bool in_place) { return channels <= 128 || (in_place && channels % 4 != 0); }

}  // namespace tcd

extern "C" int thrust_cdna4_linear_scan(void* temp, size_t* temp_bytes, const thrust_cdna4_linear_scan_args* a, void* stream) {
  using namespace tcd;
  if (!temp_bytes || !a || temp_misaligned(temp)) return hipErrorInvalidValue;
  const bool packed = a->offset_bytes != 0;
  if (!valid_shape(a->batch, a->rows, a->channels, a->sequences, a->offsets, a->offset_bytes)) return hipErrorInvalidValue;
  if (!activation_size(a->gate_dtype) || !activation_size(a->x_dtype)) return hipErrorInvalidValue;
  const size_t span_x = span_bytes(a->batch, a->rows, a->channels, a->x_batch_stride, a->x_row_stride, activation_size(a->x_dtype));
  const size_t span_g = span_bytes(a->batch, a->rows, a->channels, a->gate_batch_stride, a->gate_row_stride, activation_size(a->gate_dtype));
  const size_t span_o = span_bytes(a->batch, a->rows, a->channels, a->out_batch_stride, a->out_row_stride, activation_size(a->x_dtype));
  const bool in_place = a->out && (ranges_overlap(a->out, span_o, a->x, span_x) || ranges_overlap(a->out, span_o, a->gate, span_g));
  hipError_t rc = hipErrorInvalidValue;
  dispatch_activation(a->gate_dtype, a->x_dtype, [&](auto tg, auto tx) {
    using TG = decltype(tg);
    using TX = decltype(tx);
    constexpr int S = lin_rows_per_wave<TG, TX>();
    LinPlan l;
    if (!lin_plan(a->batch, a->rows, a->channels, S * kLinWaves, lin_narrow(a->channels, in_place) ? 1 : 4, l)) return;
    if (temp == nullptr) {
      *temp_bytes = l.bytes;
      rc = hipSuccess;
      return;
    }
    const int64_t states = packed ? a->sequences : a->batch;
    if (a->channels == 0 || a->batch == 0) {
      rc = hipSuccess;
      return;
    }
    if (*temp_bytes < l.bytes || (packed && !a->offsets)) return;
    if (a->rows > 0 && (!a->gate || !a->x || !a->out)) return;
    const size_t state_bytes = (size_t)states * (size_t)a->channels * 4;
    if (a->init && a->final_state && ranges_overlap(a->init, state_bytes, a->final_state, state_bytes)) return;
    hipStream_t s = static_cast<hipStream_t>(stream);
    LinArgs p{};
    p.gate = a->gate, p.x = a->x, p.out = a->out;
    p.init = static_cast<const float*>(a->init);
    p.final_state = static_cast<float*>(a->final_state);
    p.states = static_cast<float*>(a->states);
    p.offsets = a->offsets, p.offsets64 = a->offset_bytes == 8, p.sequences = (int)a->sequences;
    p.gate_bs = a->gate_batch_stride, p.gate_rs = a->gate_row_stride;
    p.x_bs = a->x_batch_stride, p.x_rs = a->x_row_stride;
    p.out_bs = a->out_batch_stride, p.out_rs = a->out_row_stride;
    p.rows = a->rows, p.channels = a->channels, p.batch = (int)a->batch, p.log_gate = a->log_gate != 0, p.clear_outside = packed && a->clear_outside;
    rc = lin_storage(p, l, temp);
    if (rc != hipSuccess) return;
    if (l.clear) {
      rc = zero_async(temp, l.clear, s);
      if (rc != hipSuccess) return;
    }
    const dim3 grid((unsigned)((int64_t)l.ncb * a->batch * l.ntiles));
    auto launch = [&](auto vec, auto pk, auto log16) {
      TCD_LAUNCH("linear_scan_kernel", (linear_scan_kernel<TG, TX, decltype(vec)::value, S, decltype(pk)::value, decltype(log16)::value>), grid,
                 dim3(kLinBlock), s, p);
    };
    auto go = [&](auto vec, auto pk) {
      if constexpr (sizeof(TG) == 2) {
        if (p.log_gate) return launch(vec, pk, std::true_type{});
      }
      launch(vec, pk, std::false_type{});
    };
    using One = std::integral_constant<int, 1>;
    using Four = std::integral_constant<int, 4>;
    if (l.vec == 1) packed ? go(One{}, std::true_type{}) : go(One{}, std::false_type{});
    else packed ? go(Four{}, std::true_type{}) : go(Four{}, std::false_type{});
    rc = hipGetLastError();
  });
  return (int)rc;
}

extern "C" int thrust_cdna4_linear_scan_backward(void* temp, size_t* temp_bytes, const thrust_cdna4_linear_scan_backward_args* a, void* stream) {
  using namespace tcd;
  if (!temp_bytes || !a || temp_misaligned(temp)) return hipErrorInvalidValue;
  const bool packed = a->offset_bytes != 0;
  if (!valid_shape(a->batch, a->rows, a->channels, a->sequences, a->offsets, a->offset_bytes)) return hipErrorInvalidValue;
  if (!activation_size(a->gate_dtype) || !activation_size(a->x_dtype)) return hipErrorInvalidValue;
  hipError_t rc = hipErrorInvalidValue;
  dispatch_activation(a->gate_dtype, a->x_dtype, [&](auto tg, auto tx) {
    using TG = decltype(tg);
    using TX = decltype(tx);
    LinPlan l;
    // the payload of a lane, three arrays of 8 rows: 8 x 4096 x 2560 in 32 bits, both ways, 533 us with two
    // channels, 548 with one, 607 with four, which spill
    constexpr int kWide = sizeof(TX) == 4 ? 2 : 4;
    if (!lin_plan(a->batch, a->rows, a->channels, kLinChunk, lin_narrow(a->channels, false) ? 1 : kWide, l)) return;
    if (temp == nullptr) {
      *temp_bytes = l.bytes;
      rc = hipSuccess;
      return;
    }
    const int64_t states = packed ? a->sequences : a->batch;
    if (a->channels == 0 || a->batch == 0) {
      rc = hipSuccess;
      return;
    }
    if (*temp_bytes < l.bytes || (packed && !a->offsets)) return;
    if (a->rows > 0 && (!a->gate || !a->x || !a->grad_out || !a->grad_x || !a->grad_gate || !a->states)) return;
    const size_t state_bytes = (size_t)states * (size_t)a->channels * 4;
    if (a->grad_init && ((a->grad_final && ranges_overlap(a->grad_init, state_bytes, a->grad_final, state_bytes)) ||
                         (a->init && ranges_overlap(a->grad_init, state_bytes, a->init, state_bytes))))
      return;
    hipStream_t s = static_cast<hipStream_t>(stream);
    LinArgs p{};
    p.gate = a->gate, p.x = a->x, p.grad_out = a->grad_out, p.out = a->grad_x, p.grad_gate = a->grad_gate;
    p.init = static_cast<const float*>(a->init);
    p.grad_final = static_cast<const float*>(a->grad_final);
    p.final_state = static_cast<float*>(a->grad_init);
    p.states = const_cast<float*>(static_cast<const float*>(a->states));
    p.offsets = a->offsets, p.offsets64 = a->offset_bytes == 8, p.sequences = (int)a->sequences;
    p.gate_bs = a->gate_batch_stride, p.gate_rs = a->gate_row_stride;
    p.x_bs = a->x_batch_stride, p.x_rs = a->x_row_stride;
    p.out_bs = a->grad_x_batch_stride, p.out_rs = a->grad_x_row_stride;
    p.grad_bs = a->grad_out_batch_stride, p.grad_rs = a->grad_out_row_stride;
    p.grad_gate_bs = a->grad_gate_batch_stride, p.grad_gate_rs = a->grad_gate_row_stride;
    p.rows = a->rows, p.channels = a->channels, p.batch = (int)a->batch, p.log_gate = a->log_gate != 0, p.clear_outside = packed && a->clear_outside;
    rc = lin_storage(p, l, temp);
    if (rc != hipSuccess) return;
    if (l.clear) {
      rc = zero_async(temp, l.clear, s);
      if (rc != hipSuccess) return;
    }
    const dim3 grid((unsigned)((int64_t)l.ncb * a->batch * l.ntiles));
    auto launch = [&](auto vec, auto pk, auto log16) {
      TCD_LAUNCH("linear_scan_backward_kernel", (linear_scan_backward_kernel<TG, TX, decltype(vec)::value, decltype(pk)::value, decltype(log16)::value>),
                 grid, dim3(kLinBlock), s, p);
    };
    auto go = [&](auto vec, auto pk) {
      if constexpr (sizeof(TG) == 2) {
        if (p.log_gate) return launch(vec, pk, std::true_type{});
      }
      launch(vec, pk, std::false_type{});
    };
    using One = std::integral_constant<int, 1>;
    using Wide = std::integral_constant<int, kWide>;
    if (l.vec == 1) packed ? go(One{}, std::true_type{}) : go(One{}, std::false_type{});
    else packed ? go(Wide{}, std::true_type{}) : go(Wide{}, std::false_type{});
    rc = hipGetLastError();
  });
  return (int)rc;
}

extern "C" int thrust_cdna4_linear_scan_step(int gate_dtype, int x_dtype, int log_gate, const void* gate, int64_t gate_row_stride,
                                             const void* x, int64_t x_row_stride, void* out, int64_t out_row_stride, void* state,
                                             int64_t num_slots, const int32_t* slots, int64_t batch, int64_t channels, void* stream) {
  using namespace tcd;
  if (batch < 0 || channels < 0 || num_slots < 0 || batch > 0x7fffffff || channels > kLinMaxChannels) return hipErrorInvalidValue;
  if (!activation_size(gate_dtype) || !activation_size(x_dtype)) return hipErrorInvalidValue;
  if (!slots && batch > num_slots) return hipErrorInvalidValue;
  hipError_t rc = hipErrorInvalidValue;
  dispatch_activation(gate_dtype, x_dtype, [&](auto tg, auto tx) {
    using TG = decltype(tg);
    using TX = decltype(tx);
    if (batch == 0 || channels == 0) {
      rc = hipSuccess;
      return;
    }
    if (!gate || !x || !out || (!state && num_slots > 0)) return;
    const size_t state_bytes = (size_t)num_slots * (size_t)channels * 4;
    auto meets_state = [&](const void* p, int64_t stride, int elem) {
      return rows_meet(p, batch, stride * elem, (size_t)channels * (size_t)elem, state, state_bytes);
    };
    if (meets_state(gate, gate_row_stride, (int)sizeof(TG)) || meets_state(x, x_row_stride, (int)sizeof(TX)) || meets_state(out, out_row_stride, (int)sizeof(TX))) return;
    const int64_t vectors = ceil_div(channels, (int64_t)4), few = ceil_div(vectors, (int64_t)kStepBlock);
    const int64_t wide = ceil_div(vectors, (int64_t)kStepBlock * kStepWide);
    const bool many = batch * wide >= 2 * (int64_t)device_cu_count();
    const int64_t ncb = many ? wide : few;
    if ((double)ncb * (double)batch * kStepBlock >= 4294967296.0) return;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const dim3 grid((unsigned)(ncb * batch));
    auto go = [&](auto units, auto log) {
      TCD_LAUNCH("linear_scan_step_kernel", (linear_scan_step_kernel<TG, TX, decltype(units)::value, decltype(log)::value>), grid, dim3(kStepBlock),
                 s, static_cast<const TG*>(gate), gate_row_stride, static_cast<const TX*>(x), x_row_stride, static_cast<TX*>(out), out_row_stride,
                 static_cast<float*>(state), num_slots, slots, (int)batch, channels, (int)ncb);
    };
    using One = std::integral_constant<int, 1>;
    using Wide = std::integral_constant<int, kStepWide>;
    if (many) log_gate ? go(Wide{}, std::true_type{}) : go(Wide{}, std::false_type{});
    else log_gate ? go(One{}, std::true_type{}) : go(One{}, std::false_type{});
    rc = hipGetLastError();
  });
  return (int)rc;
}
