// Operators of a decoding step over a paged key / value cache (gfx950 / CDNA4, wave64): rotary positions, the append to
// the cache, attention of new tokens over it, and products of a few rows with 4-bit weights.  Part of the generated
// translation unit of modules that call them (custom calls `mononn$...`); each function is one unit of a stage of the
// monolithic kernel.
//
// Run-time indices come from device memory and are never trusted: offsets of sequences are clamped to the token count,
// lengths to what the page table can hold, page numbers to the pool (reads) or skipped (writes), so that every address
// is in range whatever the data.
#pragma once

#ifndef MONONN_LDS_READ_TR16
// 4 x 16 elements of 16 bits per group of 16 lanes: lane i gives the address of 4 elements, elements 4 (i % 4) .. of row
// i / 4, and receives column i of the four rows
typedef short mononn_short4 __attribute__((ext_vector_type(4)));
#define MONONN_LDS_READ_TR16(p) __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) mononn_short4*)(p))
#endif

// an empty statement after which the compiler has the constant `v` in a vector register (and may still share or move it)
#ifndef MONONN_KEEP_IN_VGPR
#define MONONN_KEEP_IN_VGPR(v) asm("" : "+v"(v))
#endif

namespace mononn_dev {

template <class T>
struct IsBf16 { static constexpr bool value = false; };
template <>
struct IsBf16<__bf16> { static constexpr bool value = true; };

// stores of a result: written through where a later stage of the kernel reads it, ordinary otherwise
template <bool COHERENT, class T, int N>
__device__ __forceinline__ void store_run(T* p, const T (&v)[N]) {
  constexpr int BYTES = N * (int)sizeof(T);
  if constexpr (BYTES == 2 || BYTES == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (COHERENT) st1(p + i, v[i]);
      else st1_plain(p + i, v[i]);
    }
  } else {
    if constexpr (COHERENT) stN<T, N>(p, v);
    else stN_plain<T, N>(p, v);
  }
}
template <class T, int N>
__device__ __forceinline__ void load_run(const T* p, T (&v)[N]) {
  struct alignas(N * sizeof(T)) Run { T e[N]; };
  const Run r = *reinterpret_cast<const Run*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = r.e[i];
}

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// ---------------------------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------------------------
// Pair i of a head turns by position * inv_freq[i].  The angle is reduced to a fraction of a turn in 64 bits: at
// position 10^6 a 32-bit angle is off by 0.03 rad.  The functions themselves take 32 bits of it; what those leave, up to
// 9e-8 rad, turns their results further (to first order: its square is 10^-14), and the amplitude goes on before they are
// rounded to f32 again.
__device__ __forceinline__ void rotation_of(int position, float inv_freq, double amplitude, float& c, float& s) {
  double half_turns = (double)position * (double)inv_freq * 0.31830988618379067154;
  half_turns -= 2.0 * __builtin_rint(0.5 * half_turns);
  const float near = (float)half_turns;
  const float rest = (float)((half_turns - (double)near) * 3.14159265358979323846);
  float sn, cs;
  sincospif(near, &sn, &cs);
  // the amplitude in two f32 values (constants of the call): products in 64 bits would cost 10122 appended tokens 1 us of 16
  const float a = (float)amplitude, a_rest = (float)(amplitude - (double)a), turn = rest * a;
  c = __builtin_fmaf(cs, a, __builtin_fmaf(-sn, turn, cs * a_rest));
  s = __builtin_fmaf(sn, a, __builtin_fmaf(cs, turn, sn * a_rest));
}

// A head of D elements, the first R of them rotated, cut into pieces a thread handles: VEC pairs (two runs of VEC
// elements) of the rotated part, or VEC elements that are copied.  Pairs are (i, i + R / 2), or (2 i, 2 i + 1) when
// INTERLEAVED.
template <class T, int D, int R, bool INTERLEAVED, int VEC>
struct RotaryHead {
  static constexpr int kTurned = R / 2 / VEC;
  static constexpr int kPieces = kTurned + (D - R) / VEC;
  static constexpr int kRuns = R > 0 ? 2 : 1;
  float c[VEC], s[VEC];
  int first, second;   // element offsets of the piece's runs; second < 0: a copied piece

  __device__ __forceinline__ RotaryHead(int piece, int position, const float* inv_freq, double amplitude) {
    if (piece < kTurned) {
      first = INTERLEAVED ? 2 * piece * VEC : piece * VEC;
      second = INTERLEAVED ? first + VEC : first + R / 2;
#pragma unroll
      for (int i = 0; i < VEC; ++i) rotation_of(position, inv_freq[piece * VEC + i], amplitude, c[i], s[i]);
    } else {
      first = R + (piece - kTurned) * VEC;
      second = -1;
    }
  }
  __device__ __forceinline__ bool turned() const { return second >= 0; }
  __device__ __forceinline__ void load(const T* head, T (&x)[2][VEC]) const {
    load_run<T, VEC>(head + first, x[0]);
    if (turned()) load_run<T, VEC>(head + second, x[1]);
  }
  // rounded once, to the element type
  __device__ __forceinline__ void turn(T (&x)[2][VEC]) const {
    if (!turned()) return;
    T y[2][VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      // element i of the two runs read as pair number: pair i is (run 0, run 1)[i], or consecutive elements
      const float a = (float)(INTERLEAVED ? x[2 * i / VEC][2 * i % VEC] : x[0][i]);
      const float b = (float)(INTERLEAVED ? x[(2 * i + 1) / VEC][(2 * i + 1) % VEC] : x[1][i]);
      const T u = (T)(a * c[i] - b * s[i]), v = (T)(a * s[i] + b * c[i]);
      if constexpr (INTERLEAVED) {
        y[2 * i / VEC][2 * i % VEC] = u;
        y[(2 * i + 1) / VEC][(2 * i + 1) % VEC] = v;
      } else {
        y[0][i] = u;
        y[1][i] = v;
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[0][i] = y[0][i], x[1][i] = y[1][i];
  }
  template <bool COHERENT>
  __device__ __forceinline__ void store(T* head, const T (&x)[2][VEC]) const {
    store_run<COHERENT, T, VEC>(head + first, x[0]);
    if (turned()) store_run<COHERENT, T, VEC>(head + second, x[1]);
  }
};

// y[t, h] = x[t, h] turned by positions[t].  A thread keeps the sines of one piece and takes HEADS heads of a token.
// Bound by reading x and writing y: every byte once, in 16-byte runs of neighbouring threads; sines and cosines in 64-bit
// reduction cost more than the rotation, hence several heads per thread once there are threads enough (one head each: 26
// us where eight take 21).  8192 tokens of 32 heads of 128 in bf16: 21.3 us (134 MB, 6.3 TB/s while the input is in the
// last-level cache, 5.4 TB/s from memory); a single token: 2.5 us, the launch.
template <class T, int TOKENS, int H, int D, int R, bool INTERLEAVED, int VEC, int HEADS, bool COHERENT>
__device__ __forceinline__ void rope_unit(int unit, const T* x, const int* positions, const float* inv_freq, T* y, double amplitude) {
  using Head = RotaryHead<T, D, R, INTERLEAVED, VEC>;
  constexpr int STRIDE = (H + HEADS - 1) / HEADS;   // neighbouring threads take neighbouring heads
  const long item = (long)unit * MONONN_BLOCK_SIZE + thread_id();
  if (item >= (long)TOKENS * STRIDE * Head::kPieces) return;
  const int piece = (int)(item % Head::kPieces), h0 = (int)(item / Head::kPieces % STRIDE), t = (int)(item / Head::kPieces / STRIDE);
  T v[HEADS][2][VEC];
  const T* row = x + (long)t * H * D;
  const Head head(piece, positions[t], inv_freq, amplitude);
#pragma unroll
  for (int k = 0; k < HEADS; ++k)
    if (h0 + k * STRIDE < H) head.load(row + (h0 + k * STRIDE) * D, v[k]);
#pragma unroll
  for (int k = 0; k < HEADS; ++k)
    if (h0 + k * STRIDE < H) {
      head.turn(v[k]);
      head.template store<COHERENT>(y + ((long)t * H + h0 + k * STRIDE) * D, v[k]);
    }
}

// ---------------------------------------------------------------------------------------------
// sequences of a batch
// ---------------------------------------------------------------------------------------------
struct Sequence {
  int start, len;   // its tokens among the call's tokens
  int ctx;          // keys of the sequence, the new tokens among them
};
template <int TOKENS, int MAX_KEYS>
__device__ __forceinline__ Sequence sequence_at(const int* query_start, const int* context_len, int b) {
  Sequence s;
  s.start = clamp_int(query_start[b], 0, TOKENS);
  s.len = clamp_int(query_start[b + 1], s.start, TOKENS) - s.start;
  s.ctx = clamp_int(context_len[b], 0, MAX_KEYS);
  return s;
}
// the sequence that holds token t, or -1: the last b with query_start[b] <= t, if its tokens reach t
template <int SEQS>
__device__ __forceinline__ int sequence_of(const int* query_start, int t) {
  int lo = 0, hi = SEQS;   // query_start[lo] <= t < query_start[hi], if at all
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (query_start[mid] <= t) lo = mid;
    else hi = mid;
  }
  return query_start[lo] <= t && t < query_start[lo + 1] ? lo : -1;
}

// ---------------------------------------------------------------------------------------------
// append to the paged cache
// ---------------------------------------------------------------------------------------------
// Token i of sequence b has position context_len[b] - new tokens + i and goes to row position % PAGE of page
// page_table[b, position / PAGE]; the key is turned by its position on the way.  Positions outside the table and
// pages outside the pool are left out.  10122 tokens of 9 sequences, 8 heads of 128 in bf16: 15.8 us while k and v are in the
// last-level cache (83 MB, 5.2 TB/s: the bytes, read once and written once, as in the rotation), 22 from memory, where their
// loads stand behind a chain of small ones (the token's sequence, its lengths, its page); 48 sequences of one token: 4.4
// us, that chain behind the launch.
template <class T, int TOKENS, int SEQS, int H, int D, int R, bool INTERLEAVED, int VEC, int HEADS, int PAGE, int PAGES, int WIDTH, bool COHERENT>
__device__ __forceinline__ void kv_append_unit(int unit, const T* k, const T* v, T* k_cache, T* v_cache, const int* page_table, const int* query_start, const int* context_len,
                                               const float* inv_freq, double amplitude) {
  using Head = RotaryHead<T, D, R, INTERLEAVED, VEC>;
  constexpr int STRIDE = (H + HEADS - 1) / HEADS;
  const long item = (long)unit * MONONN_BLOCK_SIZE + thread_id();
  if (item >= (long)TOKENS * STRIDE * Head::kPieces) return;
  const int piece = (int)(item % Head::kPieces), h0 = (int)(item / Head::kPieces % STRIDE), t = (int)(item / Head::kPieces / STRIDE);
  const int b = sequence_of<SEQS>(query_start, t);
  if (b < 0) return;
  const Sequence s = sequence_at<TOKENS, WIDTH * PAGE>(query_start, context_len, b);
  const int position = s.ctx - s.len + (t - s.start);
  if (position < 0) return;   // position < WIDTH * PAGE follows from the clamped length
  const int page = page_table[(long)b * WIDTH + position / PAGE];
  if (page < 0 || page >= PAGES) return;
  const long to = ((long)page * PAGE + position % PAGE) * H * D, from = (long)t * H * D;
  const Head head(piece, position, inv_freq, amplitude);
  T kx[HEADS][2][VEC], vx[HEADS][2][VEC];
#pragma unroll
  for (int i = 0; i < HEADS; ++i)
    if (h0 + i * STRIDE < H) {
      head.load(k + from + (h0 + i * STRIDE) * D, kx[i]);
      head.load(v + from + (h0 + i * STRIDE) * D, vx[i]);
    }
#pragma unroll
  for (int i = 0; i < HEADS; ++i)
    if (h0 + i * STRIDE < H) {
      head.turn(kx[i]);
      head.template store<COHERENT>(k_cache + to + (h0 + i * STRIDE) * D, kx[i]);
      head.template store<COHERENT>(v_cache + to + (h0 + i * STRIDE) * D, vx[i]);
    }
}

// ---------------------------------------------------------------------------------------------
// attention over the paged cache
// ---------------------------------------------------------------------------------------------
// the larger of, and the sum of, a lane's value and that of the lane 32 further on (one swap of half waves)
__device__ __forceinline__ void half_waves(float v, float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  a = __builtin_bit_cast(float, (unsigned)r[0]), b = __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ __forceinline__ float half_waves_max(float v) {
  float a, b;
  half_waves(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float half_waves_sum(float v) {
  float a, b;
  half_waves(v, a, b);
  return a + b;
}
// the same for the lane 16 further on or back
__device__ __forceinline__ void quarter_waves(float v, float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  a = __builtin_bit_cast(float, (unsigned)r[0]), b = __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ __forceinline__ float quarter_waves_max(float v) {
  float a, b;
  quarter_waves(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float quarter_waves_sum(float v) {
  float a, b;
  quarter_waves(v, a, b);
  return a + b;
}

// The query rows of a sequence for one key / value head are its new tokens times the G = H / HKV query heads that
// share it (row = token * G + head of the group), in tiles: 32 rows per wave in a *wide* item, 16 in all in a
// *narrow* one (a sequence with at most 16 rows: decoding).  An item (sequence, key head, tile) works through its
// keys in steps: 64 keys that all waves share in a wide item, 32 keys per wave in a narrow one.
//
// The steps of all items, in order, are dealt to the workgroups in equal contiguous ranges, whatever the lengths of
// the sequences: every workgroup reads the same number of keys.  Items that end inside a range are written out by it;
// a range that begins or ends inside an item leaves the running maximum, sum and output of its part in memory, and
// the next stage (`join`) adds those up: the range in which an item begins owns it.
//
// Per step, with S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16 (narrow: 16x16x32): queries lie along the lanes in both products, so
// the maximum, the sum and the rescaling of a query stay in its lane (and those 32, or 16, further on), and the
// probabilities leave the first product in the lanes that feed the second (a lane's 8 accumulator rows are the 8 keys
// of one contraction step, in an order that the transposed reads of V follow).
template <class T, int TOKENS, int SEQS, int H, int HKV, int D, int PAGE, int PAGES, int WIDTH, int WINDOW, int GRID, bool COHERENT>
struct PagedAttention {
  static constexpr int NW = MONONN_BLOCK_SIZE / kWaveSize;
  static constexpr int G = H / HKV;
  static constexpr int MAX_KEYS = WIDTH * PAGE;
  static constexpr bool kBf16 = IsBf16<T>::value;
  static constexpr int CPR = D / 8;              // 16-byte pieces of a row
  static constexpr int DT = (D + 31) / 32;       // tiles of 32 output elements
  static constexpr int QS = D / 16;              // contraction steps of the first product
  // LDS rows: keys are read 16 bytes per lane down 32 rows (an odd number of 16-byte pieces spreads them over the
  // banks), values 32 bytes of 4 rows per 16 lanes (a pitch of 64 modulo 128 bytes keeps the rows apart; it covers
  // the last tile's 32 columns where D is not a multiple of 32)
  static constexpr int KP = D * 2 + 16;
  static constexpr int VP = (D * 2 + 63) / 128 * 128 + 64;
  static_assert(VP >= D * 2 && VP >= DT * 64, "value rows");
  static constexpr int kWideKeys = 64;
  // narrow items: values are read 32 bytes of 8 rows per 32 lanes; an odd multiple of 32 bytes keeps 8 rows apart
  static constexpr int VPN = (D / 16 | 1) * 32;
  static constexpr int kWaveBuffer = 32 * (KP + VPN);
  static constexpr int kTiles = D / 16;          // tiles of 16 output elements of a narrow item
  static constexpr int QN = (D + 31) / 32;       // its contraction steps of the first product
  static constexpr int kLdsLimit = 160 * 1024;
  static constexpr bool kSkew = NW >= 8 && kWideKeys * (2 * KP + 3 * VP) <= kLdsLimit;   // two waves per SIMD, and room: see wide()
  static constexpr int kValueBuffers = kSkew ? 3 : 2;
  static constexpr int narrow_waves(int n) { return n * kWaveBuffer <= kLdsLimit && n * (kTiles * 1024 + 128) <= kLdsLimit ? n : narrow_waves(n / 2); }
  static constexpr int NN = narrow_waves(NW);    // waves that take part in a narrow item
  static constexpr int kNarrowKeys = 32 * NN;
  static constexpr bool kAllNarrow = TOKENS * G <= 16;      // no sequence can have more rows
  static constexpr int kPartWave = DT * 1024 + 64;          // floats: output tiles as they lie in the registers, maxima, sums
  static constexpr int kPartNarrow = kTiles * 256 + 32;
  static constexpr long kMostRows = (long)TOKENS * G;       // no item has more
  static constexpr int kBlocks = kMostRows < 32 * NW ? (int)((kMostRows + 31) / 32) : NW;   // blocks of 32 rows of an item, at most
  static constexpr int kPart = kAllNarrow ? kPartNarrow : kBlocks * kPartWave;   // floats of one partial result; two per workgroup
  static constexpr int kMergeBytes = NN * (kTiles * 1024 + 128);
  static constexpr int lds_bytes() {
    int n = kAllNarrow ? 0 : kWideKeys * (2 * KP + kValueBuffers * VP);
    if (NN * kWaveBuffer > n) n = NN * kWaveBuffer;
    return kMergeBytes > n ? kMergeBytes : n;
  }

  static constexpr float kNothing = -3e38f;   // running maximum before the first key: below any finite score

  struct Item {
    int b, h, tile;
    Sequence s;
    int narrow;
    int first, steps;   // first step (a multiple of the step's keys) and how many
  };

  static __device__ __forceinline__ bool is_narrow(int len) { return kAllNarrow || len * G <= 16; }
  static __device__ __forceinline__ int tiles_of(int len) { return is_narrow(len) ? (len > 0 ? 1 : 0) : (len * G + 32 * NW - 1) / (32 * NW); }
  // keys [lo, hi) that some row of the tile sees
  static __device__ __forceinline__ void tile_keys(const Sequence& s, int tile, int& lo, int& hi) {
    const int rows = is_narrow(s.len) ? 16 : 32 * NW;
    const int t0 = tile * rows / G;
    int t1 = ((tile + 1) * rows - 1) / G;
    if (t1 > s.len - 1) t1 = s.len - 1;
    const int p0 = s.ctx - s.len + t0, p1 = s.ctx - s.len + t1;
    lo = WINDOW > 0 && p0 - WINDOW + 1 > 0 ? p0 - WINDOW + 1 : 0;
    hi = p1 + 1;   // <= ctx
  }
  // ... as steps; at least one step, so that empty rows are written too
  static __device__ __forceinline__ void tile_steps(const Sequence& s, int tile, int& first, int& steps) {
    const int keys = is_narrow(s.len) ? kNarrowKeys : kWideKeys;
    int lo, hi;
    tile_keys(s, tile, lo, hi);
    first = lo / keys;
    steps = hi > lo ? (hi + keys - 1) / keys - first : 0;
    if (steps < 1) steps = 1;
  }
  static __device__ __forceinline__ int head_steps(const Sequence& s) {
    int n = 0, f, k;
    const int tiles = tiles_of(s.len);
    for (int i = 0; i < tiles; ++i) {
      tile_steps(s, i, f, k);
      n += k;
    }
    return n;
  }
  static __device__ __forceinline__ Sequence sequence(const int* qs, const int* cl, int b) { return sequence_at<TOKENS, MAX_KEYS>(qs, cl, b); }
  // of the same sequence in all lanes: in scalar registers, and so what is decided by it
  static __device__ __forceinline__ Sequence uniform(const Sequence& s) {
    return {__builtin_amdgcn_readfirstlane(s.start), __builtin_amdgcn_readfirstlane(s.len), __builtin_amdgcn_readfirstlane(s.ctx)};
  }

  // Steps up to and with every sequence: lane l of a wave holds those of sequence l; behind the first 64 sequences
  // they are added up again where they are needed.
  struct Plan {
    int total;          // steps of the call
    int steps, upto;    // of the lane's sequence; of all sequences up to it
    Sequence mine;      // the lane's sequence
    bool whole;         // counted in items instead: every range is an item, or none
  };
  static __device__ __forceinline__ int steps_of(const int* qs, const int* cl, int b) { return b < SEQS ? HKV * head_steps(sequence(qs, cl, b)) : 0; }
  // Where there are no more items than ranges, an item may be a range, uncut: as long as the longest takes no more steps
  // than an equal share and what the parts would cost.  In steps, that is two for the barrier and the join, and one for
  // 256 blocks of 32 rows in parts, written and read (a wide block of 128 elements is 17 KB).
  //   32 / 8 heads of 128 elements in bf16, us uncut and cut: one prompt of 256 tokens 19 and 21, of 1024 43 and 50, of
  //   2048 79 and 110; 32 tokens each behind two caches of 1200 keys 40 and 19 (cut, by the rule)
  //   12 heads of 64 elements, single tokens of 4 sequences of 210 .. 505 keys: 8.7 and 9.2
  struct Uncut {   // what a sequence adds to the decision
    int items, steps, longest, blocks;
  };
  static __device__ __forceinline__ Uncut uncut(const Sequence& s, int tiles) {
    Uncut u = {HKV * tiles, 0, 0, 0};
    if (tiles > 0) {
      int first, shortest;
      tile_steps(s, 0, first, shortest);
      tile_steps(s, tiles - 1, first, u.longest);
      shortest = shortest < 1 << 18 ? shortest : 1 << 18, u.longest = u.longest < 1 << 18 ? u.longest : 1 << 18;   // sums stay below 2^31
      u.steps = (int)((unsigned)(HKV * tiles) * (unsigned)(shortest + u.longest) / 2);   // taken where there are at most GRID items
      u.blocks = is_narrow(s.len) ? 0 : clamp_int((s.len * G + 31) / 32, 0, NW);
    }
    return u;
  }
  static __device__ __forceinline__ bool cuts_cost_more(const Uncut& all) {
    const int parts = all.steps < GRID + all.items ? all.steps : GRID + all.items;
    return all.longest <= all.steps / GRID + 2 + parts * all.blocks / 256;
  }
#ifndef MONONN_ONE_THREAD
  // Sums and maxima over the lanes of the first 64 sequences: moves inside rows of 16 lanes on the vector unit, then the
  // rows' results through scalar registers.  (Six exchanges through the LDS take half a microsecond, which a call of single
  // tokens has twice.)
  static constexpr int kRows = SEQS >= kWaveSize ? 4 : (SEQS + 15) / 16;
  template <int SHIFT>
  static __device__ __forceinline__ int lanes_before(int v) { return __builtin_amdgcn_update_dpp(0, v, 0x110 + SHIFT, 0xf, 0xf, false); }   // 0 where the row begins
  static __device__ __forceinline__ int sum_upto(int v) {
    v += lanes_before<1>(v);
    v += lanes_before<2>(v);
    v += lanes_before<4>(v);
    v += lanes_before<8>(v);
    const int row = lane_id() >> 4;
    int before = 0;   // of the rows in front
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int of_row = __builtin_amdgcn_readlane(v, i * 16 + 15);
      before += row > i ? of_row : 0;
    }
    v += before;
    return v;
  }
  template <class Op>
  static __device__ __forceinline__ int over_sequences(int v, Op op) {   // lanes behind the last sequence hold 0
    v = op(v, dpp_move<0xB1>(v));    // quad_perm [1,0,3,2]
    v = op(v, dpp_move<0x4E>(v));    // quad_perm [2,3,0,1]
    v = op(v, dpp_move<0x141>(v));   // row_half_mirror
    v = op(v, dpp_move<0x140>(v));   // row_mirror
    int r = __builtin_amdgcn_readlane(v, 0);
#pragma unroll
    for (int row = 1; row < kRows; ++row) r = op(r, __builtin_amdgcn_readlane(v, row * 16));
    return r;
  }
  static __device__ __forceinline__ bool fewer_without_cuts(const Sequence& s, int tiles) {
    Uncut u = uncut(s, tiles);
    if constexpr (kAllNarrow) return SEQS * HKV <= GRID && __all(u.longest <= 2);
    const auto sum = [](int a, int b) { return a + b; };
    const auto larger = [](int a, int b) { return a > b ? a : b; };
    u.items = over_sequences(u.items, sum);
    if (u.items > GRID) return false;
    u.steps = over_sequences(u.steps, sum), u.longest = over_sequences(u.longest, larger);
    u.blocks = over_sequences(u.blocks, larger);
    return cuts_cost_more(u);
  }
  static __device__ __forceinline__ Plan plan(const int* qs, const int* cl) {
    Plan p;
    p.mine = sequence(qs, cl, lane_id() < SEQS ? lane_id() : SEQS - 1);
    const int tiles = lane_id() < SEQS ? tiles_of(p.mine.len) : 0;
    p.whole = SEQS <= kWaveSize && fewer_without_cuts(p.mine, tiles);
    p.steps = HKV * (p.whole || tiles == 0 ? tiles : head_steps(p.mine));
    p.upto = sum_upto(p.steps);
    p.total = __builtin_amdgcn_readlane(p.upto, kWaveSize - 1);
    for (int base = kWaveSize; base < SEQS; base += kWaveSize)
      p.total += __builtin_amdgcn_readfirstlane(wave_all_reduce(steps_of(qs, cl, base + lane_id()), [](int a, int c) { return a + c; }));
    return p;
  }
  // the sequence that holds step `rem` of the call; `rem` becomes the step inside it
  static __device__ __forceinline__ int sequence_with_step(const Plan& p, const int* qs, const int* cl, int& rem) {
    int steps = p.steps, upto = p.upto, base = 0;
    for (;;) {
      const unsigned long long behind = __ballot(upto > rem);
      if (behind != 0) {
        const int l = __builtin_ctzll(behind);
        rem -= __builtin_amdgcn_readlane(upto - steps, l);
        return base + l < SEQS ? base + l : SEQS - 1;
      }
      rem -= __builtin_amdgcn_readlane(upto, kWaveSize - 1);
      base += kWaveSize;
      if (base >= SEQS) return SEQS - 1;
      steps = steps_of(qs, cl, base + lane_id());
      upto = sum_upto(steps);
    }
  }
  static __device__ __forceinline__ Sequence planned(const Plan& p, const int* qs, const int* cl, int b) {   // b is the same in all lanes
    if (b >= kWaveSize) return uniform(sequence(qs, cl, b));
    return {__builtin_amdgcn_readlane(p.mine.start, b), __builtin_amdgcn_readlane(p.mine.len, b), __builtin_amdgcn_readlane(p.mine.ctx, b)};
  }
#else   // for a host build that runs one thread at a time
  static __device__ __forceinline__ Sequence planned(const Plan&, const int* qs, const int* cl, int b) { return sequence(qs, cl, b); }
  static __device__ __forceinline__ bool fewer_without_cuts(const int* qs, const int* cl) {
    Uncut all = {0, 0, 0, 0};
    for (int b = 0; b < SEQS; ++b) {
      const Sequence s = sequence(qs, cl, b);
      const Uncut u = uncut(s, tiles_of(s.len));
      all.items += u.items;
      if (all.items > GRID || (kAllNarrow && u.longest > 2)) return false;
      all.steps += u.steps;
      all.longest = u.longest > all.longest ? u.longest : all.longest, all.blocks = u.blocks > all.blocks ? u.blocks : all.blocks;
    }
    return kAllNarrow ? SEQS * HKV <= GRID : cuts_cost_more(all);
  }
  static __device__ __forceinline__ int counted(const Plan& p, const int* qs, const int* cl, int b) { return p.whole ? HKV * tiles_of(sequence(qs, cl, b).len) : steps_of(qs, cl, b); }
  static __device__ __forceinline__ Plan plan(const int* qs, const int* cl) {
    Plan p = {0, 0, 0, {0, 0, 0}, SEQS <= kWaveSize && fewer_without_cuts(qs, cl)};
    for (int b = 0; b < SEQS; ++b) p.total += counted(p, qs, cl, b);
    return p;
  }
  static __device__ __forceinline__ int sequence_with_step(const Plan& p, const int* qs, const int* cl, int& rem) {
    for (int b = 0; b < SEQS; ++b) {
      if (rem < counted(p, qs, cl, b)) return b;
      rem -= counted(p, qs, cl, b);
    }
    return SEQS - 1;
  }
#endif
  // the item that holds step `at` of the call (0 <= at < total_steps) and the step inside it
  static __device__ __forceinline__ Item locate(const Plan& p, const int* qs, const int* cl, int at, int& inside) {
    Item it;
    int rem = at;
    it.b = sequence_with_step(p, qs, cl, rem);
    it.s = planned(p, qs, cl, it.b);
    it.narrow = is_narrow(it.s.len);
    const int tiles = tiles_of(it.s.len);
    int per_head = p.whole ? tiles : head_steps(it.s);
    if (per_head < 1) per_head = 1;
    it.h = clamp_int(rem / per_head, 0, HKV - 1);
    rem -= it.h * per_head;
    it.tile = p.whole ? rem : 0;
    tile_steps(it.s, it.tile, it.first, it.steps);
    if (p.whole) {
      inside = 0;
      return it;
    }
    while (rem >= it.steps && it.tile + 1 < tiles) {
      rem -= it.steps;
      ++it.tile;
      tile_steps(it.s, it.tile, it.first, it.steps);
    }
    inside = clamp_int(rem, 0, it.steps - 1);
    return it;
  }
  // the item behind `it`
  static __device__ __forceinline__ void next_item(const int* qs, const int* cl, Item& it) {
    if (it.tile + 1 < tiles_of(it.s.len)) ++it.tile;
    else {
      it.tile = 0;
      if (it.h + 1 < HKV) ++it.h;
      else {
        it.h = 0;
        do {
          if (it.b + 1 >= SEQS) return;
          ++it.b;
          it.s = uniform(sequence(qs, cl, it.b));
        } while (it.s.len == 0);
        it.narrow = is_narrow(it.s.len);
      }
    }
    tile_steps(it.s, it.tile, it.first, it.steps);
  }
  // Ranges follow each other inside an XCD (workgroup u runs on XCD u % 8 of an even deal): the tiles of one key head
  // then read its keys through the same L2.
  static __device__ __forceinline__ int range_of(int unit) { return GRID % kXcds == 0 ? unit % kXcds * (GRID / kXcds) + unit / kXcds : unit; }
  static __device__ __forceinline__ int range_begin(int total, int range) { return (int)((long)total * range / GRID); }
  static __device__ __forceinline__ int range_with_step(int total, int step) {
    if (total < 0x7fffffff / GRID) return (int)((((unsigned)step + 1) * GRID + total - 1) / (unsigned)total) - 1;   // a division in 64 bits takes ten times as long
    return (int)((((long)step + 1) * GRID + total - 1) / total) - 1;
  }

  // ---- loads -----------------------------------------------------------------------------------------------------
  // The pieces of consecutive rows are dealt to the lanes in order.  Lane l fetches the page of row l of a step (one
  // load, a step ahead); where the 64 / CPR rows of an instruction lie in one page its number is the same for the
  // whole wave, and the rows' addresses are a scalar base and a lane offset that never changes.
  // What a lane's part in that comes to is worked out once per item, not per step (Lane).
  static constexpr bool kWholeRows = kWaveSize % CPR == 0;
  static constexpr bool kUniformRows = kWholeRows && PAGE % (kWholeRows ? kWaveSize / CPR : 1) == 0;
  struct Lane {
    int lane, wave;
    unsigned cell;   // element offset of the lane's piece from its run's first row in the cache
    int row, piece;  // row and piece of the lane in a run that begins with a row
    __device__ __forceinline__ Lane() {
      lane = lane_id();
      wave = __builtin_amdgcn_readfirstlane(wave_id());
      row = lane / CPR, piece = lane % CPR;
      cell = (unsigned)row * (HKV * D) + (unsigned)piece * 8;
    }
    // LDS byte offset of piece (first + lane) in rows of `pitch` bytes; `mine`: row * pitch + piece * 16
    __device__ __forceinline__ int lds(int first, int pitch, int mine) const {
      if constexpr (kWholeRows) return first / CPR * pitch + mine;
      else return (first + lane) / CPR * pitch + (first + lane) % CPR * 16;
    }
    __device__ __forceinline__ int row_of(int first) const {
      if constexpr (kWholeRows) return first / CPR + row;
      else return (first + lane) / CPR;
    }
  };
  static __device__ __forceinline__ int lane_page(const Lane& l, const int* table, int b, int key0) {
    const int key = clamp_int(key0 + l.lane, 0, MAX_KEYS - 1);
    return table[(long)b * WIDTH + (unsigned)key / PAGE];   // clamped to the pool where it is used: nothing waits for it here
  }
  static __device__ __forceinline__ half8_t load_piece(const T* p) { return *reinterpret_cast<const half8_t*>(p); }
  static __device__ __forceinline__ int in_pool(int pages) { return clamp_int(pages, 0, PAGES - 1); }
  // Element offset, in either cache, of piece (first + lane) of the cells from key0 on: a scalar part, and the lane's.
  // `pages`: in_pool(lane_page of key0).
  struct Cell {
    unsigned long base;
    unsigned mine;
  };
  static __device__ __forceinline__ Cell cell_of(const Lane& l, int pages, int key0, int first, int h) {
    Cell c;
    if constexpr (kUniformRows) {
      const int row0 = first / CPR;
      const unsigned page = __builtin_amdgcn_readlane(pages, row0 & (kWaveSize - 1));
      c.base = (unsigned long)page * ((unsigned)PAGE * HKV * D) + ((unsigned)(key0 + row0) % PAGE * (HKV * D) + (unsigned)h * D);
      c.mine = l.cell;
    } else {
      const int row = l.row_of(first);
      const unsigned page = __shfl(pages, row & (kWaveSize - 1), kWaveSize);
      c.base = (unsigned long)page * ((unsigned)PAGE * HKV * D);
      c.mine = (unsigned)(key0 + row) % PAGE * (HKV * D) + (unsigned)h * D + (kWholeRows ? l.piece : (first + l.lane) % CPR) * 8;
    }
    return c;
  }
  static __device__ __forceinline__ half8_t load_cell(const T* cache, const Cell& c) { return load_piece(cache + c.base + c.mine); }

  // the lane's query row: operand of the first product, and the keys it sees, [lo, hi]
  struct Rows {
    half8_t q[QS];
    int lo, hi;
    bool valid;
    long out;   // element offset of the row
  };
  static __device__ __forceinline__ long row_element(const Item& it, int row) {
    return ((long)clamp_int(it.s.start + row / G, 0, TOKENS - 1) * H + it.h * G + row % G) * D;
  }
  static __device__ __forceinline__ void load_rows(const T* q, const Item& it, int row0, Rows& r) {
    const int lane = lane_id(), count = it.s.len * G;
    int row = row0 + (lane & 31);
    r.valid = row < count;
    if (!r.valid) row = count > 0 ? count - 1 : 0;
    const int t = row / G;
    r.out = row_element(it, row);
#pragma unroll
    for (int i = 0; i < QS; ++i) r.q[i] = load_piece(q + r.out + i * 16 + (lane >> 5) * 8);
    r.hi = it.s.ctx - it.s.len + t;
    r.lo = WINDOW > 0 ? r.hi - WINDOW + 1 : 0;
  }

  struct State {
    float16_t o[DT];
    float m, l;   // of the lane's query; l of the lane's half of the keys until finish()
    __device__ __forceinline__ void clear() {
      m = kNothing;
      l = 0.0f;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    }
    __device__ __forceinline__ void finish() { l = half_waves_sum(l); }
  };

  // The three parts of a step: 64 keys on the wave's 32 query rows.  Left to itself the compiler reads every operand of a
  // product right in front of it and waits; here operands are read in batches of four products, a batch ahead, and nothing
  // moves across the marks between them.
  static constexpr int kBatch = 4;
  typedef float16_t Scores[2];
  // Rounded to the element type, probabilities would cost a result as much as its own rounding does (its error against 64
  // bits grows by 25 to 45 %), so each goes into the second product as two values of that type: its leading bits, and what
  // they leave.  Together they hold 16 bits of it in bf16, 22 in f16.  Single tokens, bound by the reads, take the same time
  // (2 % more at most); 6830 prompt tokens, bound by the products, take 612 us instead of 476.
  struct Probabilities {
    half8_t lead[4], rest[4];   // 16 keys each
  };
  static __device__ __forceinline__ void split(float e, half_t& lead, half_t& rest) {
    if constexpr (kBf16) {
      const unsigned top = __builtin_bit_cast(unsigned, e) & 0xffff0000u;   // cut, not rounded: the remainder is exact
      lead = __builtin_bit_cast(half_t, (unsigned short)(top >> 16));
      rest = __builtin_bit_cast(half_t, (T)(e - __builtin_bit_cast(float, top)));
    } else {
      lead = (half_t)e;
      rest = (half_t)(e - (float)lead);
    }
  }
  // The reference of a query's exponentials only has to stay near its maximum: it moves, and what has been added up
  // is rescaled, when some query of the wave has outgrown its own by 2^6, which after the first steps is rare.  In f16 it
  // is set 2^9 below the maximum: exponentials up to 2^15 are in range, and keys count that lie 2^34 below the maximum
  // (without it those 2^25 below would vanish from the product, but not from the sum: 131071 of them are 0.4 % of it).  In
  // bf16 it is set 2^32 above: values up to the type's largest times exponentials up to 2^-26, added up over 2^25 keys, stay
  // in the range of f32, and keys count that lie 2^94 below the maximum.
  static constexpr float kOutgrown = 6.0f, kBelow = kBf16 ? -32.0f : 9.0f;
  static __device__ __forceinline__ float moved(float reference, float top) { return fmaxf(reference, top - kBelow); }
  static __device__ __forceinline__ bool outgrown(float reference, float top) { return __any(top - kBelow > reference + kOutgrown); }
  static __device__ __forceinline__ void score(const char* row, const Rows& r, Scores& s) {   // row: the lane's first operand
    constexpr int kProducts = 2 * QS, kBatches = (kProducts + kBatch - 1) / kBatch;   // numbered block by block of 32 keys
    half8_t k[2][kBatch];
    auto read = [&](int batch) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int at = batch * kBatch + j;
        if (at < kProducts) k[batch & 1][j] = *reinterpret_cast<const half8_t*>(row + at / QS * 32 * KP + at % QS * 32);
      }
    };
    __builtin_amdgcn_s_setprio(1);
    read(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
    for (int batch = 0; batch < kBatches; ++batch) {
      if (batch + 1 < kBatches) read(batch + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int at = batch * kBatch + j;
        if (at < kProducts) s[at / QS] = mfma_32x32x16<kBf16>(k[batch & 1][j], r.q[at % QS], s[at / QS]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // `check`: some row does not see all of these keys
  static __device__ __forceinline__ void soft_max(int key0, const Rows& r, State& st, float scale_log2, bool check, Scores& s, Probabilities& p) {
    if (check) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key0 + b * 32 + 8 * (i / 4) + 4 * (lane_id() >> 5) + i % 4;
          s[b][i] = key >= r.lo && key <= r.hi ? s[b][i] : -__builtin_inff();
        }
    }
    __builtin_amdgcn_s_setprio(0);
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    top = half_waves_max(top) * scale_log2;
    if (outgrown(st.m, top)) {
      const float m = moved(st.m, top);
      const float a = __builtin_amdgcn_exp2f(st.m - m);
      st.l *= a;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[t][i] *= a;
      st.m = m;
    }
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[b][i] * scale_log2 - st.m);
        sum += e;
        half_t lead, rest;
        split(e, lead, rest);
        p.lead[b * 2 + i / 8][i % 8] = lead;
        p.rest[b * 2 + i / 8][i % 8] = rest;
      }
    st.l += sum;
  }
  static __device__ __forceinline__ void weigh(const char* row, const Probabilities& p, State& st) {   // row: likewise
    constexpr int kProducts = DT * 4, kBatches = DT;   // numbered tile by tile of 32 output elements
    struct Pair { mononn_short4 lo, hi; };
    Pair v[2][kBatch];
    auto read = [&](int t) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[t & 1][k].lo = MONONN_LDS_READ_TR16(row + k * 16 * VP + t * 64);
        v[t & 1][k].hi = MONONN_LDS_READ_TR16(row + (k * 16 + 8) * VP + t * 64);
      }
    };
    __builtin_amdgcn_s_setprio(1);
    read(0);
#pragma unroll
    for (int t = 0; t < kBatches; ++t) {
      if (t + 1 < kBatches) read(t + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const half8_t values = __builtin_bit_cast(half8_t, v[t & 1][k]);
        st.o[t] = mfma_32x32x16<kBf16>(values, p.rest[k], st.o[t]);
        st.o[t] = mfma_32x32x16<kBf16>(values, p.lead[k], st.o[t]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    static_assert(kProducts == kBatches * kBatch, "a batch per tile");
  }

  // ---- results ---------------------------------------------------------------------------------------------------
  // Group g of four output elements of the lane's row: d = 32 * (g / 4) + 8 * (g % 4) + 4 * (lane / 32).
  // Groups g and g + 1: halves of the wave exchange four elements, so that a lane stores eight, of group g or g + 1
  static __device__ __forceinline__ void store_groups(T* out, const Rows& r, int g, const float16_t& o, float scale) {
    T four[2][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) four[i / 4][i % 4] = (T)(o[g % 4 * 4 + i] * scale);
    struct Two { unsigned d[2]; };
    const Two a = __builtin_bit_cast(Two, four[0]), b = __builtin_bit_cast(Two, four[1]);
    struct { unsigned d[4]; } eight;
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // lower lanes: their elements 0 .. 3 and the upper lane's 4 .. 7 of g; upper lanes likewise of g + 1
      const auto x = __builtin_amdgcn_permlane32_swap(a.d[i], b.d[i], false, false);
      eight.d[i] = x[0], eight.d[2 + i] = x[1];
    }
    const int at = (g / 4) * 32 + (g % 4 + (lane_id() >> 5)) * 8;
    struct Eight { T v[8]; };
    if (!r.valid || at >= D) return;
    store_run<COHERENT, T, 8>(out + r.out + at, __builtin_bit_cast(Eight, eight).v);
  }
  static __device__ __forceinline__ void store_part(float* to, int g, float a, float b, float c, float d) {
    const float v[4] = {a, b, c, d};
    stN<float, 4>(to + g * 256 + lane_id() * 4, v);
  }
  // maximum and sum of the 32 queries behind the tiles
  static __device__ __forceinline__ void store_part_sums(float* to, float m, float l) {
    const int lane = lane_id();
    st1(to + DT * 1024 + lane, lane < 32 ? m : l);
  }
  static __device__ __forceinline__ float inverse(float l) { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }   // a row without keys: zeros

  // ---- wide items ------------------------------------------------------------------------------------------------
  // Bound by the matrix units, and by how well two waves per SIMD hide the rest behind them: of the 5000 clocks of a step they
  // are busy for 3070 (two waves; a third of it the remainders of the probabilities), the vector units for 2700 (an
  // exponential per score takes a fifth of that), the LDS reads of K and V for 2000.  One barrier per step: it ends the stores of the
  // step's tile, while the next one is on its way in registers.  So that a SIMD's two waves are not at the same part at
  // the same time, the later one runs half a step behind: it begins with the products of the last step's values, which
  // therefore stay a step longer (three buffers).  Waves at their products go first where both could issue.
  // At 5 prompts of 6830 tokens in all on 32 / 8 heads of 128 elements in bf16: 612 us with the join, 720 TFLOP/s, 1080 with
  // the remainders' products, at a clock that falls to 1.9 GHz.
  // With probabilities in one value (476 us): without the shift 3 % more, without the priority 2 %, with a barrier per half step
  // that forces the waves to take turns 6 %, with the next item's first tile and queries requested before the last one's
  // results are stored 5 %.
  static constexpr int kRuns = (kWideKeys * CPR + MONONN_BLOCK_SIZE - 1) / MONONN_BLOCK_SIZE;   // pieces of K (and of V) a thread moves per step
  static __device__ __forceinline__ int wide_piece(const Lane& l, int run) { return (run * NW + l.wave) * kWaveSize; }
  static __device__ __forceinline__ void wide_store(const Lane& l, char* buf, int pitch, int mine, const half8_t (&x)[kRuns]) {
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      if (kWideKeys * CPR % MONONN_BLOCK_SIZE != 0 && l.row_of(wide_piece(l, i)) >= kWideKeys) break;
      *reinterpret_cast<half8_t*>(buf + l.lds(wide_piece(l, i), pitch, mine)) = x[i];
    }
  }
  // Values of keys outside [lo, hi), which no row of the tile sees, become zeros: whatever those cells hold, NaN included,
  // must not reach 0 * v.  (Their scores are replaced, not multiplied: keys may stay as they are.)
  static __device__ __forceinline__ void clear_unseen(const Lane& l, int key0, int lo, int hi, half8_t (&x)[kRuns]) {
    if (key0 + kWideKeys > hi || (WINDOW > 0 && key0 < lo)) {
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        const int key = key0 + l.row_of(wide_piece(l, i));
        if (key >= hi || (WINDOW > 0 && key < lo)) x[i] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
      }
    }
  }
  static __device__ __forceinline__ void wide(const T* q, const T* kc, const T* vc, const int* table, T* out, float* part, const Item& it, int from, int count, bool whole,
                                              float scale_log2, char* smem) {
    const Lane l;
    const int k_mine = l.row * KP + l.piece * 16, v_mine = l.row * VP + l.piece * 16;
    const int k_read = (l.lane & 31) * KP + (l.lane >> 5) * 16, v_read = (4 * (l.lane >> 5) + (l.lane & 15) / 4) * VP + ((l.lane >> 4) & 1) * 32 + (l.lane & 3) * 8;
    const int wave = l.wave;
    const int rows = it.s.len * G, row0 = it.tile * 32 * NW + wave * 32;
    const bool live = row0 < rows, later = kSkew && (wave / 4) % 2 == 1;   // wave w runs on SIMD w % 4
    char* const kbuf = smem;                                   // [2][64][KP]
    char* const vbuf = smem + 2 * kWideKeys * KP;              // [kValueBuffers][64][VP]
    const int begin = (it.first + from) * kWideKeys;
    half8_t k[kRuns], v[kRuns];   // the next tile, on its way
    int pages_next = lane_page(l, table, it.b, begin);
    // Behind the last step the same again, stored where nothing reads it any more: without branches around them the
    // compiler knows how many loads are on their way, and waits for no more than it needs.  The pages of the next tile
    // are asked for before this one's rows: loads return in order.
    auto load_tile = [&](int j) {
      const int pages = in_pool(pages_next);
      pages_next = lane_page(l, table, it.b, begin + (j + 1) * kWideKeys);
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        const Cell cell = cell_of(l, pages, begin + j * kWideKeys, wide_piece(l, i), it.h);
        k[i] = load_cell(kc, cell);
        v[i] = load_cell(vc, cell);
      }
    };
    int v_at = 0;   // the buffer of this step's values, in bytes
    auto next_buffer = [](int at) { return at == (kValueBuffers - 1) * kWideKeys * VP ? 0 : at + kWideKeys * VP; };
    load_tile(0);
    Rows r;
    load_rows(q, it, row0, r);
    // keys that the wave's first and last row see
    const int t_first = row0 / G, t_last = (row0 + 31 < rows ? row0 + 31 : rows - 1) / G;
    const int p_first = it.s.ctx - it.s.len + t_first, p_last = it.s.ctx - it.s.len + t_last;
    int seen_lo, seen_hi;
    tile_keys(it.s, it.tile, seen_lo, seen_hi);
    State st;
    st.clear();
    wide_store(l, kbuf, KP, k_mine, k);
    clear_unseen(l, begin, seen_lo, seen_hi, v);
    wide_store(l, vbuf, VP, v_mine, v);
    load_tile(1);
    Scores s;
    Probabilities p;
    bool weighing = false;   // the last step left probabilities to a later wave
    int v_last = 0;
    for (int i = 0; i < count; ++i) {
      const int key0 = begin + i * kWideKeys;
      const bool some = live && key0 <= p_last && !(WINDOW > 0 && key0 + kWideKeys - 1 < p_first - WINDOW + 1);
      const int v_next = next_buffer(v_at);
      __syncthreads();
      if (later && weighing) weigh(vbuf + v_last + v_read, p, st);
      if (some) {
        score(kbuf + (i & 1) * kWideKeys * KP + k_read, r, s);
        soft_max(key0, r, st, scale_log2, key0 + kWideKeys - 1 > p_first || (WINDOW > 0 && key0 < p_last - WINDOW + 1), s, p);
      }
      // the next tile, where the LDS has least to do
      wide_store(l, kbuf + ((i + 1) & 1) * kWideKeys * KP, KP, k_mine, k);
      clear_unseen(l, key0 + kWideKeys, seen_lo, seen_hi, v);
      wide_store(l, vbuf + v_next, VP, v_mine, v);
      load_tile(i + 2);
      if (!later && some) weigh(vbuf + v_at + v_read, p, st);
      weighing = some;
      v_last = v_at;
      v_at = v_next;
    }
    if (later && weighing) weigh(vbuf + v_last + v_read, p, st);   // stored behind it: the next buffer
    __syncthreads();
    st.finish();
    if (!live) return;
    if (whole) {
      const float inv = inverse(st.l);
#pragma unroll
      for (int g = 0; g < DT * 4; g += 2) store_groups(out, r, g, st.o[g / 4], inv);
    } else {
      float* to = part + wave * kPartWave;
#pragma unroll
      for (int g = 0; g < DT * 4; ++g) store_part(to, g, st.o[g / 4][g % 4 * 4], st.o[g / 4][g % 4 * 4 + 1], st.o[g / 4][g % 4 * 4 + 2], st.o[g / 4][g % 4 * 4 + 3]);
      store_part_sums(to, st.m, st.l);
    }
  }

  // ---- narrow items ----------------------------------------------------------------------------------------------
  // Bound by the reads of keys and values: 32 sequences of 200 .. 8191 keys on 32 / 8 heads of 128 in bf16 take 121 us, 108
  // of them at 5.0 TB/s in this stage (a large copy reaches 5.2); one of 131071 keys 106 us, 5.1 TB/s; 4 sequences of up to
  // 512 keys on 12 heads of 64, where the chain of lengths, pages, rows counts, 8.7 us.  Every wave streams its own 32 keys of a step: requested a step ahead into
  // registers, through the wave's own LDS rows (no workgroup barrier) into the products.  The next step may belong to
  // the next item: its keys, and that item's queries, are on their way while the waves' shares of the last one are added up.
  static constexpr int kMine = CPR / 2;   // pieces of K (and of V) a lane moves per step: 32 rows over 64 lanes
  struct Cursor {
    Item it;
    int step;   // inside the item
    __device__ __forceinline__ int key0(const Lane& l) const { return (it.first + step) * kNarrowKeys + l.wave * 32; }
  };
  struct NarrowRows {
    half8_t q[QN];
    int lo, hi;
    bool valid;
    long out;
  };
  static __device__ __forceinline__ void narrow_rows(const T* q, const Item& it, NarrowRows& r) {
    const int lane = lane_id(), count = it.s.len * G, g = lane >> 4;
    int row = lane & 15;
    r.valid = row < count;
    if (!r.valid) row = count > 0 ? count - 1 : 0;
    r.out = row_element(it, row);
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const half8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
      r.q[i] = D % 32 != 0 && i == QN - 1 && g >= 2 ? zero : load_piece(q + r.out + i * 32 + g * 8);
    }
    r.hi = it.s.ctx - it.s.len + row / G;
    r.lo = WINDOW > 0 ? r.hi - WINDOW + 1 : 0;
  }
  static __device__ __forceinline__ void narrow_load(const Lane& l, const T* kc, const T* vc, int pages, const Cursor& c, half8_t (&k)[kMine], half8_t (&v)[kMine]) {
    const int key0 = c.key0(l);
    if (key0 >= c.it.s.ctx) return;   // the wave has no key in this step
    pages = in_pool(pages);
    Cell cell[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      cell[i] = cell_of(l, pages, key0, i * kWaveSize, c.it.h);
      k[i] = load_cell(kc, cell[i]);
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) v[i] = load_cell(vc, cell[i]);
  }
  struct NarrowState {
    float4_t o[kTiles];
    float m, l;   // of the lane's query; l of the lane's keys until finish()
    __device__ __forceinline__ void clear() {
      m = kNothing;
      l = 0.0f;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) o[t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void finish() { l = quarter_waves_sum(half_waves_sum(l)); }
  };
  // 32 keys on 16 query rows
  static __device__ __forceinline__ void narrow_step(const Lane& l, const char* krow, const char* vrow, int key0, const NarrowRows& r, NarrowState& st, float scale_log2, bool check) {
    const int g = l.lane >> 4;
    float4_t s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const char* row = krow + b * 16 * KP;
#pragma unroll
      for (int i = 0; i < QN; ++i) {
        // half a step at the end of the head: the queries are zero there, any elements of the row will do
        const int back = D % 32 != 0 && i == QN - 1 && g >= 2 ? 32 : 0;
        s[b] = mfma_16x16x32<kBf16>(*reinterpret_cast<const half8_t*>(row + i * 64 - back), r.q[i], s[b]);
      }
    }
    if (check) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = key0 + b * 16 + 4 * g + i;
          s[b][i] = key >= r.lo && key <= r.hi ? s[b][i] : -__builtin_inff();
        }
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = quarter_waves_max(half_waves_max(top)) * scale_log2;
    if (outgrown(st.m, top)) {   // as in soft_max()
      const float m = moved(st.m, top);
      const float a = __builtin_amdgcn_exp2f(st.m - m);
      st.l *= a;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) st.o[t] *= a;
      st.m = m;
    }
    half8_t lead, rest;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(s[b][i] * scale_log2 - st.m);
        st.l += e;
        half_t l16, r16;
        split(e, l16, r16);
        lead[b * 4 + i] = l16;
        rest[b * 4 + i] = r16;
      }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      struct { mononn_short4 lo, hi; } v;
      v.lo = MONONN_LDS_READ_TR16(vrow + t * 32);
      v.hi = MONONN_LDS_READ_TR16(vrow + 16 * VPN + t * 32);
      const half8_t values = __builtin_bit_cast(half8_t, v);
      st.o[t] = mfma_16x16x32<kBf16>(values, rest, st.o[t]);
      st.o[t] = mfma_16x16x32<kBf16>(values, lead, st.o[t]);
    }
  }
  static __device__ __forceinline__ void narrow_out(T* out, long row, bool valid, int tile, float4_t o, float inv) {
    if (!valid) return;
    const T v[4] = {(T)(o[0] * inv), (T)(o[1] * inv), (T)(o[2] * inv), (T)(o[3] * inv)};
    store_run<COHERENT, T, 4>(out + row + tile * 16 + (lane_id() >> 4) * 4, v);
  }
  // Works from step `inside` of `it` to the end of the range or of the run of narrow items; `it` and `inside` become
  // where it stopped.  Returns the steps done.
  static __device__ __forceinline__ int narrow(const T* q, const T* kc, const T* vc, const int* table, const int* qs, const int* cl, T* out, float* part, int range, Item& it, int& inside,
                                               int left, float scale_log2, char* smem) {
    const Lane l;
    const int wave = l.wave, lane = l.lane, query = lane & 15;
    const bool live = wave < NN;
    char* const kbuf = smem + (live ? wave : 0) * kWaveBuffer;
    char* const vbuf = kbuf + 32 * KP;
    const int k_mine = l.row * KP + l.piece * 16, v_mine = l.row * VPN + l.piece * 16;
    const int k_read = (lane & 15) * KP + (lane >> 4) * 16, v_read = (4 * (lane >> 4) + (lane & 15) / 4) * VPN + (lane & 3) * 8;
    Cursor cur = {it, inside};
    // the step behind `c`; false when the range ends before it or it is a wide item's (`c` is that item then)
    auto advance = [&](Cursor& c, int remaining) {
      if (remaining <= 0) return false;
      if (++c.step < c.it.steps) return true;
      next_item(qs, cl, c.it);
      c.step = 0;
      return c.it.narrow != 0;
    };
    half8_t k[kMine], v[kMine];
    int done = 0, begun = inside;   // step of the item at which this part begins
    NarrowRows r, rn;
    narrow_rows(q, cur.it, r);
    if (live) narrow_load(l, kc, vc, lane_page(l, table, cur.it.b, cur.key0(l)), cur, k, v);
    Cursor nxt = cur;
    bool more = advance(nxt, left - 1);
    int pages = more ? lane_page(l, table, nxt.it.b, nxt.key0(l)) : 0;
    NarrowState st;
    st.clear();
    __syncthreads();   // the buffers may still be read by a wide item's last step
    for (;;) {
      const int key0 = cur.key0(l);
      const bool some = live && key0 < cur.it.s.ctx;
      if (some) {
        const int lo = WINDOW > 0 ? cur.it.s.ctx - cur.it.s.len - WINDOW + 1 : 0;   // first key that some row sees
        if (key0 + 32 > cur.it.s.ctx || (WINDOW > 0 && key0 < lo)) {   // values that no row sees: as in clear_unseen()
#pragma unroll
          for (int j = 0; j < kMine; ++j) {
            const int key = key0 + l.row_of(j * kWaveSize);
            if (key >= cur.it.s.ctx || (WINDOW > 0 && key < lo)) v[j] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
          }
        }
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          *reinterpret_cast<half8_t*>(kbuf + l.lds(j * kWaveSize, KP, k_mine)) = k[j];
          *reinterpret_cast<half8_t*>(vbuf + l.lds(j * kWaveSize, VPN, v_mine)) = v[j];
        }
      }
      Cursor behind = nxt;
      bool more_behind = false;
      if (more) {
        if (live) narrow_load(l, kc, vc, pages, nxt, k, v);
        more_behind = advance(behind, left - done - 2);
        if (more_behind) pages = lane_page(l, table, behind.it.b, behind.key0(l));
      }
      if (some) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();   // the wave's own rows: written above, read below
        const int p_first = cur.it.s.ctx - cur.it.s.len, p_last = cur.it.s.ctx - 1;
        if (!(WINDOW > 0 && key0 + 31 < p_first - WINDOW + 1)) {
          const bool check = key0 + 31 > p_first || (WINDOW > 0 && key0 < p_last - WINDOW + 1);
          narrow_step(l, kbuf + k_read, vbuf + v_read, key0, r, st, scale_log2, check);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      ++done;
      if (cur.step + 1 == cur.it.steps || done == left) {
        // the end of the item, or of the range: the waves' shares of the keys meet in LDS, every wave adds up some tiles
        const bool whole = begun == 0 && cur.step + 1 == cur.it.steps;
        if (more) narrow_rows(q, nxt.it, rn);
        st.finish();
        __syncthreads();
        float* sums = reinterpret_cast<float*>(smem);             // [NN][32]: maxima, sums
        float* tiles = sums + NN * 32;                            // [NN][kTiles][64][4]
        if (live) {
          if (lane < 32) sums[wave * 32 + lane] = lane < 16 ? st.m : st.l;
#pragma unroll
          for (int t = 0; t < kTiles; ++t) *reinterpret_cast<float4_t*>(tiles + (wave * kTiles + t) * 256 + lane * 4) = st.o[t];
        }
        __syncthreads();
        float m = kNothing, l = 0.0f, w[NN];
#pragma unroll
        for (int i = 0; i < NN; ++i) m = fmaxf(m, sums[i * 32 + query]);
#pragma unroll
        for (int i = 0; i < NN; ++i) {
          w[i] = __builtin_amdgcn_exp2f(sums[i * 32 + query] - m);
          l += w[i] * sums[i * 32 + 16 + query];
        }
        float* to = part + (long)(2 * range + (begun == 0 ? 1 : 0)) * kPart;
        const float inv = inverse(l);
        for (int t = wave; t < kTiles; t += NW) {
          float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < NN; ++i) o += w[i] * *reinterpret_cast<const float4_t*>(tiles + (i * kTiles + t) * 256 + lane * 4);
          if (whole) narrow_out(out, r.out, r.valid, t, o, inv);
          else store_part(to, t, o[0], o[1], o[2], o[3]);
        }
        if (!whole && wave == 0 && lane < 32) st1(to + kTiles * 256 + lane, lane < 16 ? m : l);
        __syncthreads();
        begun = 0;
        st.clear();
        r = rn;
      }
      if (!more) break;
      cur = nxt, nxt = behind, more = more_behind;
    }
    it = nxt.it, inside = nxt.step;
    return done;
  }

  // ---- stages ----------------------------------------------------------------------------------------------------
  // part: [2 * GRID][kPart]; slot 2 r: a part that an earlier range began, slot 2 r + 1: one that range r begins
  static __device__ __forceinline__ void partial(int unit, const T* q, const T* kc, const T* vc, const int* table, const int* qs, const int* cl, T* out, float* part, float scale,
                                                 char* smem) {
    const int first_token = qs[0], end_token = qs[SEQS];   // on their way with the lengths
    const Plan p = plan(qs, cl);
    const int inside0 = clamp_int(first_token, 0, TOKENS), inside1 = clamp_int(end_token, 0, TOKENS);
    // tokens of no sequence: zeros
    if (inside0 > 0 || inside1 < TOKENS) {
      const T zero[8] = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
      for (int t = unit; t < TOKENS; t += GRID)
        if (t < inside0 || t >= inside1)
          for (int c = thread_id(); c < H * CPR; c += MONONN_BLOCK_SIZE) store_run<COHERENT, T, 8>(out + (long)t * H * D + c * 8, zero);
    }
    const int range = range_of(unit);
    int at = range_begin(p.total, range), end = range_begin(p.total, range + 1);
    const float scale_log2 = scale * 1.44269504088896f;
    if (at >= end) return;
    int inside;
    Item it = locate(p, qs, cl, at, inside);
    if (p.whole) end = at + it.steps;
    __syncthreads();
    while (at < end) {
      if (it.narrow) {
        at += narrow(q, kc, vc, table, qs, cl, out, part, range, it, inside, end - at, scale_log2, smem);
        continue;
      }
      if constexpr (!kAllNarrow) {
        const int count = it.steps - inside < end - at ? it.steps - inside : end - at;
        const bool whole = inside == 0 && count == it.steps;
        wide(q, kc, vc, table, out, part + (long)(2 * range + (inside == 0 ? 1 : 0)) * kPart, it, inside, count, whole, scale_log2, smem);
        at += count;
        inside = 0;
        next_item(qs, cl, it);
      }
    }
    __syncthreads();
  }

  template <int N>
  struct Count { static constexpr int value = N; };
  // Adds up the parts of the items that were split: a few loads behind each other, 3 us for single
  // tokens; 29 us behind 580 of products for 6830 prompt tokens, whose 512 parts are 68 MB, written and read (left to the
  // range in which an item begins, one workgroup for each, one sequence of 131071 keys takes 157 us instead of 104).  The workgroups whose ranges hold a part of an item share its
  // output groups among them: `rank` of `count` is this workgroup's.  With many parts the waves of a workgroup take the
  // parts of a group between them, with few every wave its own groups.
  static __device__ __forceinline__ void join_item(const float* part, const Plan& p, const Item& it, int item0, int rank, int count, T* out, char* smem) {
    if (kAllNarrow || it.narrow) join_tiles<true>(part, p, it, item0, rank, count, out, smem);
    else if constexpr (!kAllNarrow) join_tiles<false>(part, p, it, item0, rank, count, out, smem);
  }
  // A unit of work is a tile of a block of queries: 16 output elements of 16 queries in a narrow item, 32 of 32 in a wide one.
  template <bool NARROW>
  static __device__ __forceinline__ void join_tiles(const float* part, const Plan& p, const Item& it, int item0, int rank, int count, T* out, char* smem) {
    constexpr int QUERIES = NARROW ? 16 : 32, GROUPS = NARROW ? 1 : 4, TILES = NARROW ? kTiles : DT;   // groups: four elements per lane
    constexpr int SUMS = TILES * GROUPS * 256;   // maxima and sums lie behind a block's tiles
    const int wave = __builtin_amdgcn_readfirstlane(wave_id()), lane = lane_id(), query = lane & (QUERIES - 1);
    const int rows = it.s.len * G, row0 = NARROW ? 0 : it.tile * 32 * NW;
    const int blocks = NARROW ? 1 : clamp_int((rows - row0 + 31) / 32, 1, NW);
    const int first = range_with_step(p.total, item0);
    // part i: ranges follow each other, unless there are fewer steps than ranges; then every step is a part
    auto slot = [&](int i) { return (long)(i == 0 ? 2 * first + 1 : 2 * (p.total >= GRID ? first + i : range_with_step(p.total, item0 + i))) * kPart; };
    const bool shared = count >= NW;
    float* share = reinterpret_cast<float*>(smem);   // [NW][GROUPS][64][4] outputs, [NW][64] maxima, [NW][64] sums
    const int step = shared ? NW : 1;
    struct Sum {
      float4_t o[GROUPS];
      float m, l;
      __device__ __forceinline__ void add(float pm, float pl, const float4_t (&po)[GROUPS]) {
        const float top = fmaxf(m, pm), a = __builtin_amdgcn_exp2f(m - top), b = __builtin_amdgcn_exp2f(pm - top);
        m = top;
        l = l * a + pl * b;
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) o[j] = o[j] * a + po[j] * b;
      }
    };
    for (int unit = shared ? rank : rank * NW + wave; unit < blocks * TILES; unit += shared ? count : count * NW) {
      const int block = unit / TILES, tile = unit % TILES;
      const float* from = part + block * kPartWave;
      Sum sum;
      sum.m = kNothing, sum.l = 0.0f;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) sum.o[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      // PARTS parts from i on: all loads on their way before the first is used
      auto add_parts = [&](auto parts_at_once, int i) {
        constexpr int PARTS = parts_at_once.value;
        float pm[PARTS], pl[PARTS];
        float4_t po[PARTS][GROUPS];
#pragma unroll
        for (int k = 0; k < PARTS; ++k) {
          const float* t = from + slot(i + k * step);
          pm[k] = t[SUMS + query], pl[k] = t[SUMS + QUERIES + query];
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) po[k][j] = *reinterpret_cast<const float4_t*>(t + (tile * GROUPS + j) * 256 + lane * 4);
        }
#pragma unroll
        for (int k = 0; k < PARTS; ++k) sum.add(pm[k], pl[k], po[k]);
      };
      int i = shared ? wave : 0;
      for (; i + 3 * step < count; i += 4 * step) add_parts(Count<4>(), i);
      for (; i + step < count; i += 2 * step) add_parts(Count<2>(), i);
      for (; i < count; i += step) add_parts(Count<1>(), i);
      if (shared) {   // the waves' sums, one after the other through the first one's hands
        float4_t* const outputs = reinterpret_cast<float4_t*>(share);
        float* const maxima = share + NW * GROUPS * 256;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < GROUPS; ++j) outputs[(wave * GROUPS + j) * 64 + lane] = sum.o[j];
        maxima[wave * 64 + lane] = sum.m;
        maxima[(NW + wave) * 64 + lane] = sum.l;
        __syncthreads();
        if (wave != 0) continue;
        for (int w = 1; w < NW; ++w) {
          float4_t po[GROUPS];
#pragma unroll
          for (int j = 0; j < GROUPS; ++j) po[j] = outputs[(w * GROUPS + j) * 64 + lane];
          sum.add(maxima[w * 64 + lane], maxima[(NW + w) * 64 + lane], po);
        }
      }
      Rows r;
      const int row = row0 + block * 32 + query;
      r.valid = row < rows;
      r.out = row_element(it, r.valid ? row : 0);
      const float inv = inverse(sum.l);
      if constexpr (NARROW) narrow_out(out, r.out, r.valid, tile, sum.o[0], inv);
      else {
        float16_t o;
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = sum.o[e / 4][e % 4];
        store_groups(out, r, tile * 4, o, inv);
        store_groups(out, r, tile * 4 + 2, o, inv);
      }
    }
  }
  static constexpr int join_lds_bytes() { return NW * ((kAllNarrow ? 1 : 4) * 256 + 128) * 4; }
  static __device__ __forceinline__ void join(int unit, const float* part, const int* qs, const int* cl, T* out, char* smem) {
    const Plan p = plan(qs, cl);
    const int range = range_of(unit), begin = range_begin(p.total, range), end = range_begin(p.total, range + 1);
    if (p.whole || begin >= end) return;
    // the item that an earlier range began, if there is one, and the one that this range leaves unfinished
    for (int k = 0; k < 2; ++k) {
      int inside;
      const Item it = locate(p, qs, cl, k == 0 ? begin : end - 1, inside);
      const int item0 = (k == 0 ? begin : end - 1) - inside, item1 = item0 + it.steps;
      if (k == 0 ? inside == 0 : (item0 < begin || item1 <= end)) continue;
      const int first = range_with_step(p.total, item0), last = range_with_step(p.total, item1 - 1);
      const bool dense = p.total >= GRID;
      join_item(part, p, it, item0, dense ? range - first : begin - item0, dense ? last - first + 1 : it.steps, out, smem);
    }
  }
};

// ---------------------------------------------------------------------------------------------
// 4-bit weights
// ---------------------------------------------------------------------------------------------
// y[m, n] = sum over groups of scale[n, group] * sum over k of (w[n, k] - zero[n, group]) * x[m, k], weights two to a
// byte along k (the low half is the lower k), zero = 8 without a tensor of zero points.
//
// Bound by the reads of the weights as long as a byte of them costs few instructions: one row on 4096 x 4096 weights 3.7
// us (a launch is 2.5), 3 rows on 14337 x 4096 in groups of 32 with zero points 10.2 us (35 MB), 16 rows on 4096 x 14336 in
// groups of 64 12.9 us (33 MB: x has to arrive before the first product, the rest streams, then a barrier and the join).  A wave takes 16 weight rows; lane
// (r, g) = (lane % 16, lane / 16) reads row r, of every 128 P columns the 32 P that belong to its lane group g, in P
// pieces of 16 bytes.  The products run on v_mfma_f32_16x16x32 with x as the left operand and the weights, small
// integers and so exact, as the right one: a lane's result column is one weight row, scales are applied to f32 results.
// A contraction step takes 8 columns from each lane group, so the groups' scales must not meet in it:
//   kSpread  M <= 4: the 16 rows of the left operand hold x once per lane group, with zeros for the other groups'
//            columns.  Result row 4 g + m then is lane group g's share of row m, in the lanes that hold its scales.
//   kWhole   groups of 128 columns or more, P = 1: all four lane groups share a scale.
//   kSwap    otherwise: a 4 x 4 transposition of dwords between the lane groups gives every step 32 consecutive columns.
template <class T>
struct Nibbles;
template <>
struct Nibbles<half_t> {
  static constexpr bool kExact = true;   // operands are value - zero
  // (w >> s) & 15 in f16 by setting exponent bits: 1024 + v where the four bits are the last of the mantissa, 64 + v where
  // they stand four places higher; elements 0, 4, 1, 5, 2, 6, 3, 7 of the dword.  Less 1024 or 64 and the zero point (any
  // byte): all are whole numbers that f16 holds.
  static __device__ __forceinline__ half8_t operands(unsigned w, unsigned zero) {
    half8_t r;
    unsigned low = 0x64006400u, high = 0x54005400u;   // in vector registers: one instruction then masks and sets (two constants would need two)
    MONONN_KEEP_IN_VGPR(low);
    MONONN_KEEP_IN_VGPR(high);
    const half2_t l8 = __builtin_bit_cast(half2_t, zero * 0x00010001u + 0x64006400u), h8 = l8 - half2_t{(half_t)960.0f, (half_t)960.0f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned x = i ? w >> 8 : w;
      const half2_t lo = __builtin_bit_cast(half2_t, (x & 0x000f000fu) | low) - l8, hi = __builtin_bit_cast(half2_t, (x & 0x00f000f0u) | high) - h8;
      r[4 * i] = lo[0], r[4 * i + 1] = lo[1], r[4 * i + 2] = hi[0], r[4 * i + 3] = hi[1];
    }
    return r;
  }
};
template <>
struct Nibbles<__bf16> {
  // 128 + v: there is no packed bf16 subtraction, a sum of x takes 128 and the zero point out again.  That leaves the result
  // off by what 128 + zero times the sum of |x| loses in f32, and x that is not finite without a result (infinity less infinity).
  static constexpr bool kExact = false;
  static constexpr int kBias = 128;
  static __device__ __forceinline__ half8_t operands(unsigned w, unsigned) {
    struct { unsigned d[4]; } r;
    unsigned bits = 0x43004300u;
    MONONN_KEEP_IN_VGPR(bits);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.d[i] = ((w >> (4 * i)) & 0x000f000fu) | bits;
    return __builtin_bit_cast(half8_t, r);
  }
};

// 8 consecutive elements in the order of Nibbles::operands
__device__ __forceinline__ half8_t nibble_order(half8_t x) {
  return __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7);
}

// exchanges dword i of lane group j with dword j of lane group i (groups of 16 lanes)
__device__ __forceinline__ void transpose_lane_groups(unsigned (&d)[4]) {
  auto swap32 = [](unsigned& a, unsigned& b) {   // upper half of a <-> lower half of b
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  auto swap16 = [](unsigned& a, unsigned& b) {   // odd groups of a <-> even groups of b
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  swap32(d[0], d[2]);
  swap32(d[1], d[3]);
  swap16(d[0], d[1]);
  swap16(d[2], d[3]);
}

// WK waves of a workgroup share a tile of 16 weight rows by splitting the columns; SK workgroups do where x does not fit
// one's LDS (`parts`, added up by `join`)
template <class T, int M, int N, int K, int GROUP, bool ZEROS, int WK, int SK, int P, bool COHERENT>
struct MatvecW4 {
  static constexpr int NW = MONONN_BLOCK_SIZE / kWaveSize;
  static constexpr int TILES = NW / WK;                       // tiles of 16 weight rows a workgroup takes at once
  static constexpr int MT = (M + 15) / 16 < 4 ? (M + 15) / 16 : 4;   // blocks of 16 rows of x per pass over the weights
  static constexpr int XROWS = M < 16 * MT ? M : 16 * MT;     // rows of x in a pass
  static constexpr bool kSpread = M <= 4, kWhole = !kSpread && GROUP >= 128, kSwap = !kSpread && !kWhole;
  static_assert(!kWhole || P == 1, "the lane groups of a step share a scale");
  static constexpr int BLOCK = 128 * P;                       // columns a wave reads at a time
  static constexpr int BLOCKS = (K + BLOCK - 1) / BLOCK;
  static constexpr int PER_GROUP = (BLOCKS + SK - 1) / SK;    // blocks of a workgroup
  static constexpr int MINE = (PER_GROUP + WK - 1) / WK;      // blocks of a wave (consecutive)
  static constexpr int GROUPS = K / GROUP;
  static constexpr int SCALES = kSwap ? BLOCK / GROUP : (kSpread && 32 * P > GROUP ? 32 * P / GROUP : 1);   // scales of a block that a lane needs
  static constexpr int AHEAD = 8 / P;
  static constexpr int DEPTH = MINE < AHEAD ? MINE : AHEAD;   // blocks in flight
  static constexpr bool kBf16 = IsBf16<T>::value;
  static constexpr bool kSums = !Nibbles<T>::kExact;
  static constexpr int ROWS = M < 4 ? M : 4;                  // result rows a lane looks at
  static constexpr int kShareBytes = WK > 1 ? NW * MT * 1024 : 0;
  static constexpr int kPieces = PER_GROUP * BLOCK / 8;       // x in LDS: [piece of 8 columns][row][8], elements in the operands' order
  static constexpr int ROW_UNITS = ((N + 15) / 16 + TILES - 1) / TILES;
  static constexpr int num_units() { return ROW_UNITS * SK * ((M + 16 * MT - 1) / (16 * MT)); }
  static constexpr int XPITCH = XROWS % 2 == 0 ? XROWS + 1 : XROWS;   // an odd number of 16-byte cells per piece: columns of cells fall on different banks
  static constexpr int lds_bytes() { return kShareBytes + kPieces * XPITCH * 16; }

  struct Scales { T v[SCALES]; };
  struct Zeros { unsigned char v[SCALES]; };
  struct Weights {
    int4_t w[P];
    Scales scale;
    Zeros zero;
  };
  // of a lane's scales, which belongs to piece j and set q of its products
  static __device__ __forceinline__ constexpr int group_of(int q, int j) { return kSwap ? (q * 32 * P + 32 * j) / GROUP : (kSpread ? 32 * j / GROUP : 0); }
  static __device__ __forceinline__ unsigned zero_of(const Weights& c, int q, int j) {
    if constexpr (ZEROS) return c.zero.v[group_of(q, j)];
    else return 8;
  }
  // what a lane needs of `E`[N, GROUPS] for a block
  template <class V, class E>
  static __device__ __forceinline__ V load_groups(const E* p, long row, int block) {
    const int first = kSpread ? (block * BLOCK + (lane_id() >> 4) * 32 * P) / GROUP : block * BLOCK / GROUP;
    V r;
    if constexpr (K % BLOCK == 0) {
      struct alignas(sizeof(V)) Run { V v; };
      r = reinterpret_cast<const Run*>(p + row * GROUPS + first)->v;
    } else {
#pragma unroll
      for (int i = 0; i < SCALES; ++i) r.v[i] = p[row * GROUPS + (first + i < GROUPS ? first + i : GROUPS - 1)];
    }
    return r;
  }
  static __device__ __forceinline__ void load(const unsigned char* weight, const T* scale, const unsigned char* zero, long row, int block, Weights& c) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      int at = block * (BLOCK / 2) + (lane_id() >> 4) * 16 * P + i * 16;
      if (K % BLOCK != 0 && at > K / 2 - 16) at = K / 2 - 16;     // behind the last column: any weights, x is zero there
      c.w[i] = *reinterpret_cast<const int4_t*>(weight + row * (K / 2) + at);
    }
    c.scale = load_groups<Scales>(scale, row, block);
    if constexpr (ZEROS) c.zero = load_groups<Zeros>(zero, row, block);
  }
  // x goes to the LDS through registers, kRun pieces of a thread at a time.  The last of these rounds is split in two, so
  // that the first weights can be asked for between its loads and its stores: loads return in order.
  static constexpr int kCells = kPieces * XROWS, kRounds = (kCells + MONONN_BLOCK_SIZE - 1) / MONONN_BLOCK_SIZE, kRun = kRounds < 8 ? kRounds : 8;
  static __device__ __forceinline__ void request_x(const T* x, int m0, int piece0, int round, half8_t (&v)[kRun]) {
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const int i = (round + j) * MONONN_BLOCK_SIZE + thread_id();
      const int piece = i % kPieces, m = i / kPieces;   // neighbouring threads read along a row
      v[j] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
      if (m < XROWS && m0 + m < M && (piece0 + piece) * 8 < K) v[j] = *reinterpret_cast<const half8_t*>(x + (long)(m0 + m) * K + (piece0 + piece) * 8);
    }
  }
  static __device__ __forceinline__ void keep_x(int round, const half8_t (&v)[kRun], half8_t* xs) {
#pragma unroll
    for (int j = 0; j < kRun; ++j) {
      const int i = (round + j) * MONONN_BLOCK_SIZE + thread_id();
      if (i < kCells) xs[i % kPieces * XPITCH + i / kPieces] = nibble_order(v[j]);
    }
  }
  // left operands of piece i of a block, for its four steps; `a` keeps its zeros in the lanes that hold no x
  static __device__ __forceinline__ void x_operands(const half8_t* xs, int block, int i, half8_t (&a)[MT][4]) {
    const int g = lane_id() >> 4, r16 = lane_id() & 15;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // first column of the lane's 8: of its own lane group's, or of the 32 that step k holds after the transposition
        const int piece = block * (BLOCK / 8) + (kSwap ? k * 4 * P + i * 4 + g : g * 4 * P + i * 4 + k);
        if constexpr (kSpread) {
          if (r16 >> 2 == g && (r16 & 3) < M) a[t][k] = xs[piece * XPITCH + (r16 & 3)];
        } else {
          const int m = t * 16 + r16 < XROWS ? t * 16 + r16 : XROWS - 1;   // rows behind the last: some row, the results are not stored
          a[t][k] = xs[piece * XPITCH + m];
        }
      }
  }

  // result: y, or with SK > 1 the f32 partial sums [SK][M][N]
  // fresh: x is not in the LDS yet
  static __device__ __forceinline__ void unit(int unit, bool fresh, const T* x, const unsigned char* weight, const T* scale, const unsigned char* zero, T* y, float* parts, char* smem) {
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), g = lane >> 4, r16 = lane & 15;
    const int pass = unit / (ROW_UNITS * SK), slice = unit / ROW_UNITS % SK, tile = unit % ROW_UNITS * TILES + wave / WK, part = wave % WK;
    const int n = tile * 16 + r16, m0 = pass * 16 * MT;
    const long row = n < N ? n : N - 1;
    const int first = slice * PER_GROUP, b0 = first + part * MINE;
    const int behind = first + PER_GROUP < BLOCKS ? first + PER_GROUP : BLOCKS, count = clamp_int(behind - b0, 0, MINE);
    half8_t* xs = reinterpret_cast<half8_t*>(smem + kShareBytes);
    __syncthreads();   // the rows of the unit before
    Weights ring[DEPTH];
    auto block_at = [&](int i) { return clamp_int(b0 + (i < count ? i : count - 1), 0, BLOCKS - 1); };   // the last one again behind the end
    auto request_weights = [&] {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) load(weight, scale, zero, row, block_at(i), ring[i]);
    };
    if (fresh) {
      half8_t staged[kRun];
      int round = 0;
      for (; round + kRun < kRounds; round += kRun) {
        request_x(x, m0, first * (BLOCK / 8), round, staged);
        keep_x(round, staged, xs);
      }
      request_x(x, m0, first * (BLOCK / 8), round, staged);
      request_weights();
      keep_x(round, staged, xs);
    } else {
      request_weights();
    }
    float4_t acc[MT];
    half8_t a[2][MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      acc[t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < 4; ++k) a[0][t][k] = a[1][t][k] = half8_t{0, 0, 0, 0, 0, 0, 0, 0};
    }
    __syncthreads();
    if (count > 0) x_operands(xs, block_at(0) - first, 0, a[0]);   // a wave behind the slice's last block has none
    for (int base = 0; base < count; base += DEPTH) {
#pragma unroll
      for (int i = 0; i < DEPTH; ++i) {
        if (base + i >= count) break;
        const Weights c = ring[i];
        load(weight, scale, zero, row, block_at(base + i + DEPTH), ring[i]);
        constexpr int SETS = kSwap ? 4 : 1;   // results with scales of their own
        float4_t dot[MT][SETS], sum[MT][SETS];
#pragma unroll
        for (int j = 0; j < P; ++j) {
          constexpr bool kAlternate = (DEPTH * P) % 2 == 0;   // operands one piece ahead, in the other set of registers
          half8_t(&now)[MT][4] = a[kAlternate ? (i * P + j) % 2 : 0];
          half8_t(&ahead)[MT][4] = a[kAlternate ? (i * P + j + 1) % 2 : 1];
          x_operands(xs, (j + 1 < P ? block_at(base + i) : block_at(base + i + 1)) - first, (j + 1) % P, ahead);
          unsigned w[4] = {(unsigned)c.w[j][0], (unsigned)c.w[j][1], (unsigned)c.w[j][2], (unsigned)c.w[j][3]};
          if constexpr (kSwap) transpose_lane_groups(w);
          // the first product of a set starts from zero; a set ends where its columns end a group, or with the block
          const bool fresh = j == 0 || (32 * j) % GROUP == 0, done = (32 * (j + 1)) % GROUP == 0 || j + 1 == P;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const half8_t b = Nibbles<T>::operands(w[k], zero_of(c, kSwap ? k : 0, j));
            constexpr float4_t kZero = {0.0f, 0.0f, 0.0f, 0.0f};
            const int set = kSwap ? k : 0;
            const bool start = fresh && (kSwap || k == 0);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              dot[t][set] = mfma_16x16x32<kBf16>(now[t][k], b, start ? kZero : dot[t][set]);
              if constexpr (kSums) {
                const half_t o = __builtin_bit_cast(half_t, (T)1.0f);
                sum[t][set] = mfma_16x16x32<kBf16>(now[t][k], half8_t{o, o, o, o, o, o, o, o}, start ? kZero : sum[t][set]);
              }
            }
          }
          if (done) {
#pragma unroll
            for (int q = 0; q < SETS; ++q) {
              const float s = (float)c.scale.v[group_of(q, j)];
#pragma unroll
              for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < ROWS; ++e) {
                  if constexpr (kSums) acc[t][e] += s * (dot[t][q][e] - (float)(zero_of(c, q, j) + Nibbles<T>::kBias) * sum[t][q][e]);
                  else acc[t][e] += s * dot[t][q][e];
                }
            }
          }
          if constexpr (!kAlternate) {
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int k = 0; k < 4; ++k) a[0][t][k] = a[1][t][k];
          }
        }
      }
    }
    if constexpr (kSpread) {   // the lane groups' shares
#pragma unroll
      for (int e = 0; e < ROWS; ++e) acc[0][e] = quarter_waves_sum(half_waves_sum(acc[0][e]));
    }
    if constexpr (WK > 1) {
      float* shares = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int t = 0; t < MT; ++t) *reinterpret_cast<float4_t*>(shares + ((wave * MT + t) * 64 + lane) * 4) = acc[t];
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int o = 1; o < WK; ++o) acc[t] += *reinterpret_cast<const float4_t*>(shares + (((wave + o) * MT + t) * 64 + lane) * 4);
      }
    }
    if (part == 0 && n < N) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < ROWS; ++e) {
          const int m = kSpread ? e : m0 + t * 16 + 4 * g + e;
          if (m >= M || (kSpread && g != 0)) continue;
          if constexpr (SK > 1) {
            st1(parts + ((long)slice * M + m) * N + n, acc[t][e]);
          } else {
            const T v[1] = {(T)acc[t][e]};
            store_run<COHERENT, T, 1>(y + (long)m * N + n, v);
          }
        }
    }
  }

  // A workgroup's units, UNITS apart.  Where all of them read the same x it is brought once, which lets a plan cut the
  // columns finer and deal more evenly: 8 rows on 11008 x 4096 weights in groups of 32 16.4 -> 12.6 us, one row 7.6 -> 7.3.
  template <int UNITS>
  static __device__ __forceinline__ void units(int first, const T* x, const unsigned char* weight, const T* scale, const unsigned char* zero, T* y, float* parts, char* smem) {
    constexpr bool kOneX = SK * ((M + 16 * MT - 1) / (16 * MT)) == 1;
    if constexpr (num_units() <= UNITS) unit(first, true, x, weight, scale, zero, y, parts, smem);
    else
      for (int u = first; u < num_units(); u += UNITS) unit(u, !kOneX || u == first, x, weight, scale, zero, y, parts, smem);
  }

  static constexpr int join_units() { return (M * N + MONONN_BLOCK_SIZE - 1) / MONONN_BLOCK_SIZE; }
  static __device__ __forceinline__ void join(int unit, const float* parts, T* y) {
    const long i = (long)unit * MONONN_BLOCK_SIZE + thread_id();
    if (i >= (long)M * N) return;
    float v = parts[i];
#pragma unroll 64
    for (int s = 1; s < SK; ++s) v += parts[(long)s * M * N + i];
    const T r[1] = {(T)v};
    store_run<COHERENT, T, 1>(y + i, r);
  }
};

}  // namespace mononn_dev
