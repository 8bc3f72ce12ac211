// Attention over the paged cache for a ragged batch, each sequence's queries
// before the keys it owns (causal, the last query at the last key) and, where
// the batch shares a prefix, all of the prefix's keys.
//
// For a query row q: o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m) over the
// keys it sees, s_j = scale q.k_j, in one pass over the keys with a running
// reference r in place of m: weights 2^(s_j scale log2(e) - r), and sums and
// outputs scaled by 2^(r - r') when r moves to r'. r only has to stay within
// 2^8 of the largest weight, so it moves when a score exceeds it by 8, not at
// every new maximum; until then a step needs no exchange between lanes and no
// rescaling. Each row's reference moves by its own scores alone, so a row's bits
// do not depend on the rows beside it. Scores, weights' sums and outputs are
// fp32; the product with V takes 16-bit weights. In tiles of few rows, where HBM
// leaves MFMA idle, what the rounding leaves of a weight goes through a second
// product (so weights are kept to 2^-16 or 2^-22; 29.1 and 28.8 us with and
// without for the ragged 64 below, 133.5 both for the long ones). In tiles of
// many rows, where MFMA is half the time, weights are rounded (a relative 2^-8
// or 2^-11 at most for bf16 and fp16, of mixed signs) and their sum is that of
// the rounded ones, by one instruction a pair: a second product there takes 740
// us instead of 532 for a prompt of 8192 tokens, 104 instead of 83 for questions
// after a prefix, 32.3 instead of 30.6 for 64 tokens over a prefix of 8192, where
// the output's own rounding is 1.7e-3 of the 2.3e-3 that bf16 outputs are off by.
// fp16 weights are 2^7 larger, up to 2^15, so that those that many keys share
// stay normal numbers.
//
// Both products run on MFMA with the keys on the A side: S^T = K Q^T leaves
// each lane the scores of one query row, and the score tile's registers are,
// with no move between lanes, the B operand of O^T = V^T P^T, if V^T's k slots
// take the keys in the same order; ds_read_b64_tr_b16 reads V that way from
// row-major tiles. So a row's reference, sum and rescaling are one lane's.
//
// K and V tiles go from global memory to LDS directly (16 bytes a lane), with
// their 16-byte chunks XOR-swizzled so that both kinds of reads meet 256
// bytes of distinct banks.
#include <type_traits>

#include "attention.h"

namespace jv {

constexpr float kRescaleAt = 8.0f;

// Exponents are one FMA, s scale - r, of a reference r that was rounded as s
// scale was: from 2^20 on what the rounding took from r would show in the
// weights (2^24 and more of it passes what fp16 holds, 2^31 fp32). Scores of
// such rows have r taken off their rounded product first, at every tile: their
// wave's limit lets every tile in where references are moved. `sub`: what the
// FMA takes off; s: N registers V of scores. Returns the wave's new limit.
constexpr float kRoundAt = 1048576.0f;
template <class H, int N, class V>
__device__ __forceinline__ float moved_to(float ref, float scale, float* sub, V* s) {
  *sub = ref == -__builtin_inff() ? 0.0f : ref - H::kShift;
  const bool large = fabsf(ref) >= kRoundAt && ref != -__builtin_inff();
  if (!__any(large)) return ref + kRescaleAt;
  const float inv = 1.0f / scale;
#pragma unroll
  for (int b = 0; b < N; ++b)
#pragma unroll
    for (int e = 0; e < (int)(sizeof(V) / 4); ++e) s[b][e] = large ? (s[b][e] * scale - *sub) * inv : s[b][e];
  if (large) *sub = 0.0f;
  return -__builtin_inff();
}

__device__ __forceinline__ void load_lds16(const uint8_t* src, uint8_t* dst_wave_base) {
  typedef __attribute__((address_space(3))) void lds_void;
  typedef __attribute__((address_space(1))) void global_void;
  __builtin_amdgcn_global_load_lds((global_void*)(src), (lds_void*)(dst_wave_base), 16, 0, 0);
}

// s_waitcnt with only the vector-memory counter constrained (vmcnt in bits 3:0
// and 15:14; expcnt and lgkmcnt left at their maxima).
template <int N>
__device__ __forceinline__ void wait_vmem_below() {
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

__device__ __forceinline__ i32x4 lds_read16(const uint8_t* p) { return *reinterpret_cast<const i32x4*>(p); }

// Lane constants that feed many addresses go through this once a key tile, so
// that the compiler computes the addresses there (an XOR each) and does not
// keep all of them in registers over the loop.
__device__ __forceinline__ uint32_t fresh(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

__device__ __forceinline__ i32x4 lds_read16(uint32_t at, uint32_t offset) {
  typedef __attribute__((address_space(3))) const i32x4 lds_i32x4;
  typedef __attribute__((address_space(3))) const uint8_t lds_u8;
  return *(lds_i32x4*)((lds_u8*)(uintptr_t)at + offset);
}

// Transposing reads: of the 4 x 16 block of 16-bit values that 16 consecutive
// lanes address (8 bytes a lane, four lanes a row), lane i gets column i. Four
// addresses plus OFF bytes, as one block with its wait: before the builtin the
// compiler waits for every copy to LDS in flight, the next tile's too; the
// block waits for the LDS reads alone.
template <int OFF>
__device__ __forceinline__ void lds_read_tr4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, s16x4* out) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  i32x2 x0, x1, x2, x3;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%c8\n"
      "ds_read_b64_tr_b16 %1, %5 offset:%c8\n"
      "ds_read_b64_tr_b16 %2, %6 offset:%c8\n"
      "ds_read_b64_tr_b16 %3, %7 offset:%c8\n"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(x0), "=&v"(x1), "=&v"(x2), "=&v"(x3)
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(OFF)
      : "memory");
  out[0] = __builtin_bit_cast(s16x4, x0), out[1] = __builtin_bit_cast(s16x4, x1);
  out[2] = __builtin_bit_cast(s16x4, x2), out[3] = __builtin_bit_cast(s16x4, x3);
}
// 8-value operands from N addresses (2 or 4), each of the reads at A0 and A1.
template <int N, int A0, int A1>
__device__ __forceinline__ void lds_read_tr8(const uint32_t* at, i32x4* out) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  i32x2 x[2 * N];
  if constexpr (N == 4) {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8 offset:%c12\n"
        "ds_read_b64_tr_b16 %1, %8 offset:%c13\n"
        "ds_read_b64_tr_b16 %2, %9 offset:%c12\n"
        "ds_read_b64_tr_b16 %3, %9 offset:%c13\n"
        "ds_read_b64_tr_b16 %4, %10 offset:%c12\n"
        "ds_read_b64_tr_b16 %5, %10 offset:%c13\n"
        "ds_read_b64_tr_b16 %6, %11 offset:%c12\n"
        "ds_read_b64_tr_b16 %7, %11 offset:%c13\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(A0), "n"(A1)
        : "memory");
  } else {
    asm volatile(
        "ds_read_b64_tr_b16 %0, %4 offset:%c6\n"
        "ds_read_b64_tr_b16 %1, %4 offset:%c7\n"
        "ds_read_b64_tr_b16 %2, %5 offset:%c6\n"
        "ds_read_b64_tr_b16 %3, %5 offset:%c7\n"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
        : "v"(at[0]), "v"(at[1]), "n"(A0), "n"(A1)
        : "memory");
  }
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = i32x4{x[2 * i].x, x[2 * i].y, x[2 * i + 1].x, x[2 * i + 1].y};
}

// Waits out a 16x16 MFMA's result registers, which other instructions may not
// read for up to 11 issue slots. Where a wave-uniform branch follows the MFMA
// the compiler has left the wait out on the taken path (rows of scores then
// differed from run to run), so it stands here, ahead of the branch.
__device__ __forceinline__ void settle(f32x4* r) { asm volatile("s_nop 7\n\ts_nop 2" : "+v"(*r)); }

// LDS byte address of a pointer into a __shared__ array.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  typedef __attribute__((address_space(3))) const uint8_t lds_u8;
  return (uint32_t)(uintptr_t)(lds_u8*)p;
}

// Both are linear over XOR: swizzle(r | s) = swizzle(r) ^ swizzle(s) for rows
// without common bits, and so are the addresses made from them.
// A tile's rows are D / 8 chunks of 16 bytes; what XORs a row's chunk index.
// LDS serves 256 bytes (64 banks) at a time. K is read 16 rows at one chunk:
// the row within the rows that start at bank 0 separates them. V is read by
// 32 lanes, 4 rows x 4 chunks or 8 rows x 2: bits 2 and 1 from the row.
template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
  return D == 64 ? (row >> 1) & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  if constexpr (D == 64) return ((row >> 1) & 1) * 4 + ((row >> 2) & 1) * 2;
  else return (row & 3) * 4 + ((row >> 2) & 1) * 2;
}

// ---------------------------------------------------------------------------
// Which rows and keys a workgroup has.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int clamped(int v, int lo, int hi) { return max(lo, min(v, hi)); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A value of an array that no kernel of the call writes, by a scalar load
// where the index is the same in all lanes.
__device__ __forceinline__ int32_t read_only(const int32_t* p, int64_t i) {
  typedef __attribute__((address_space(4))) const int32_t constant_i32;
  return ((constant_i32*)p)[i];
}

__device__ __forceinline__ int start_of(const AttnArgs& a, int b) {
  return a.starts ? clamped(read_only(a.starts, b), 0, a.tokens) : b;
}

// First tile slot of a sequence whose queries start at token `start`.
__device__ __forceinline__ int first_tile(const AttnArgs& a, int b, int start, int rows) {
  if (!a.starts && a.group <= rows) return b;
  return (int)(((uint32_t)start * (uint32_t)a.group) / (uint32_t)rows) + b;
}

// A sequence of the batch: its first token, its tokens and its own keys.
struct Sequence {
  int start, n, len;
};
__device__ __forceinline__ Sequence sequence(const AttnArgs& a, int b) {
  Sequence s{b, 1, clamped(read_only(a.lengths, b), 0, a.table_cols << a.page_shift)};
  if (a.starts) {
    s.start = clamped(read_only(a.starts, b), 0, a.tokens);
    s.n = max(0, clamped(read_only(a.starts, b + 1), 0, a.tokens) - s.start);
  }
  return s;
}

// The sequence that a tile slot belongs to: the last whose first slot is not
// past it, 64 sequences a step (every lane active, the same slot in each).
__device__ __forceinline__ int sequence_of_slot(const AttnArgs& a, int slot, int rows) {
  if (!a.starts && a.group <= rows) return min(slot, a.batch - 1);
  const int lane = threadIdx.x & 63;
  int count = 0;
  for (int base = 0; base < a.batch; base += 64) {
    const int b = base + lane;
    const int c = __popcll(__ballot(b < a.batch && first_tile(a, b, start_of(a, min(b, a.batch - 1)), rows) <= slot));
    count += c;
    if (c < 64) break;
  }
  return max(count - 1, 0);
}

// Sums over the lanes up to each one (DPP row shifts, then row 0's total into
// row 1 and row 2's into row 3, then the lower half's into the upper).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// Where keys are split over workgroups: the (sequence, row tile, key chunk) of
// a unit, computed by each wave for itself, 64 sequences a step, from the
// lengths on the device. `shared`: keys before the own ones that count too.
//
// Keys are counted in steps of 16, or of the keys by which a row tile sees more
// than the one before it. A tile that sees at most x + 1 steps is cut into
// 1 + x / m chunks of equal shares. m, of CHUNK keys at least, is chosen so that
// the chunks of all tiles, the units, fit `own_units`: with W the sum of the x, W / (own_units - tiles) + 1
// does, as each tile begins one chunk more than its share.
//
// Tiles of few rows are cut alike within a sequence (what its last tile sees is
// taken for all), from kWorthSplit steps on, and into half a device of chunks
// more than there are tiles where these fill it. Cutting what is near the
// average, for up to twice the tiles, took 24.3 instead of 16.7 us for 64
// sequences of 300 keys (32 heads of 128), 45 instead of 30 for 128, 48 instead
// of 42 for 64 of 1000; cutting 500 keys 18.5 instead of 15.0 for 32 sequences,
// but 10.0 instead of 10.9 for 4.
//
// Of many rows, tile t of a sequence has x = a + t, so that a prompt's early
// tiles, which see little, are cut less, and up to 64 sequences take the least
// of eight m from W / own_units on that fits. (A prompt of 2048 tokens of 16
// heads of 256: 70 us, 90 with chunks alike; of 1500 tokens of 32 heads of 128
// 42 us, 49 with up to twice as many units as the device holds.)
constexpr uint32_t kWorthSplit = 32;
struct Unit {
  int b, tile, chunk, chunks;  // sequence, row tile and chunk of the unit, chunks of the tile
  Sequence seq;
};
// Sum of i / m over the i below x, modulo 2^32.
__device__ __forceinline__ uint32_t sum_below(uint32_t x, uint32_t m) {
  const uint32_t q = x / m;
  return m * (q * (q - 1) / 2) + q * (x - q * m);
}
// False if there is no such unit.
template <int ROWS, int CHUNK>
__device__ __forceinline__ bool find_unit(const AttnArgs& a, int unit, int shared, Unit* u) {
  constexpr bool MANY = ROWS == kManyRows;
  const int lane = threadIdx.x & 63, batches = (a.batch + 63) >> 6;
  const uint32_t step = MANY ? max(16u, (uint32_t)(ROWS + a.group - 1) / (uint32_t)a.group) : 16;
  uint32_t weight = 0, m = 1;
  int all_tiles = 0, before = 0;
  Sequence s;
  // `batches` times to add the keys up, as often again to find the unit; up to
  // 64 sequences are read once
  for (int i = 0; i < 2 * batches; ++i) {
    const int base = (i < batches ? i : i - batches) * 64;
    if (i == 0 || batches > 1) {
      s = sequence(a, min(base + lane, a.batch - 1));
      if (base + lane >= a.batch) s.n = 0;
    }
    const uint32_t tiles = (uint32_t)(s.n * a.group + ROWS - 1) / (uint32_t)ROWS;
    // x of the first tile, or of all
    const uint32_t x = (MANY ? (uint32_t)(shared + max(0, s.len - s.n)) + step - 1 : (uint32_t)max(shared + s.len - 1, 0)) / step;
    const auto units = [&](uint32_t m) {
      if (MANY) return (int)(tiles + sum_below(x + tiles, m) - sum_below(x, m));
      return (int)(a.p.split && x >= kWorthSplit ? tiles * (1 + x / m) : tiles);
    };
    if (i < batches) {
      weight += (uint32_t)lane_value(wave_scan((int)(tiles * x + (MANY ? tiles * (tiles - 1) / 2 : 0))), 63);
      all_tiles = min(all_tiles + lane_value(wave_scan((int)tiles), 63), (1 << 30) - 1);
      if (i + 1 < batches) continue;
      if (all_tiles > a.p.tiles) return false;  // starts that decrease
      const int most = MANY ? a.p.own_units : min(a.p.own_units, max(a.p.at_once, all_tiles + a.p.at_once / 2));
      const uint32_t least = (CHUNK + step - 1) / step;
      m = max(least, weight / (uint32_t)max(1, most - all_tiles) + 1);
      if (MANY && batches == 1) {
        const uint32_t low = max(least, weight / (uint32_t)most + 1), each = (m - low + 6) / 7;
        for (uint32_t t = low; t < m; t += each) {
          if (lane_value(wave_scan(units(t)), 63) <= most) m = t;
        }
      }
      m = (uint32_t)uniform((int)m);
      continue;
    }
    const int n = units(m);
    const int upto = wave_scan(n);
    const uint64_t past = __ballot(before + upto > unit);
    if (past) {
      const int l = uniform(__ffsll((unsigned long long)past) - 1);
      const int of = unit - (before + lane_value(upto, l) - lane_value(n, l));  // the sequence's
      const int its_tiles = lane_value((int)tiles, l);
      const uint32_t its_x = (uint32_t)lane_value((int)x, l);
      u->b = base + l;
      u->seq = Sequence{lane_value(s.start, l), lane_value(s.n, l), lane_value(s.len, l)};
      if (!MANY) {
        u->chunks = a.p.split && its_x >= kWorthSplit ? uniform((int)(1 + its_x / m)) : 1;
        u->tile = uniform((int)((uint32_t)of / (uint32_t)u->chunks));
        u->chunk = of - u->tile * u->chunks;
        return true;
      }
      // the last tile whose units begin at or before this one, 64 tiles a step
      u->tile = 0, u->chunk = of;
      const uint32_t sum0 = sum_below(its_x, m);
      for (int t0 = 0; t0 < its_tiles; t0 += 64) {
        const int t = t0 + lane, begins = t + (int)(sum_below(its_x + (uint32_t)t, m) - sum0);
        const int count = __popcll(__ballot(t < its_tiles && begins <= of));
        if (count == 0) break;
        u->tile = t0 + count - 1, u->chunk = of - lane_value(begins, count - 1);
        if (count < 64) break;
      }
      u->chunks = uniform((int)(1 + (its_x + (uint32_t)u->tile) / m));
      return true;
    }
    before += lane_value(upto, 63);
  }
  return false;
}

// Own keys that the last of `rows` rows from row0 on sees.
__device__ __forceinline__ int visible_keys(const Sequence& s, int row0, int rows, int group) {
  return max(0, s.len - s.n + (int)((uint32_t)(row0 + rows - 1) / (uint32_t)group) + 1);
}

// A run of keys that a workgroup goes through: page ids, the first and the
// last key (inclusive).
struct Keys {
  const int32_t* ids;
  int first, last;
};

// What a workgroup does: up to two runs of keys (the prefix's, then the
// sequence's own) for `rows` query rows. Every field is the same in all lanes.
struct Job {
  Keys prefix, own;
  int tiles0, tiles;       // key tiles of the prefix, of both
  int token0, row0, rows;  // query row r: token token0 + (row0 + r) / group
  int own_base;            // own key index that row r sees last: own_base + (row0 + r) / group
  int sequence, first, chunk, chunks;  // whose rows; their units, and which of them this one is
};

// kWhole: all keys of a row tile, the prefix's and its own. kSplit: a chunk of
// them. kOwn: a chunk of its own keys; the prefix's come as partial results
// from kPrefix: a share of the prefix for a tile of all the tokens' rows.
enum Mode { kWhole, kSplit, kOwn, kPrefix };

// Fills a job from the block index; false if the block has nothing to do.
template <Mode MODE, int ROWS, int KT, int GRAIN, int CHUNK>
__device__ __forceinline__ bool find_job(const AttnArgs& a, int unit, Job* j) {
  j->prefix = j->own = Keys{a.prefix_pages, 0, -1};
  j->sequence = 0, j->first = unit, j->chunk = 0, j->chunks = 1;
  if constexpr (MODE == kPrefix) {
    const int splits = a.p.prefix_splits, tile = (int)((uint32_t)unit / (uint32_t)splits), s = unit - tile * splits;
    const int each = (int)(((uint32_t)(a.prefix_len + splits - 1) / (uint32_t)splits + GRAIN - 1) / GRAIN) * GRAIN;
    j->prefix.first = min(s * each, a.prefix_len);
    j->prefix.last = min(j->prefix.first + each, a.prefix_len) - 1;
    j->token0 = 0;
    j->row0 = tile * ROWS;
    j->rows = min(ROWS, a.tokens * a.group - j->row0);
    j->own_base = -1;
    j->tiles0 = j->tiles = (j->prefix.last - j->prefix.first + KT) / KT;
    return true;
  }
  const int shared = MODE == kOwn ? 0 : a.prefix_len;
  Sequence s;
  int b;
  if constexpr (MODE == kWhole) {
    b = uniform(sequence_of_slot(a, unit, ROWS));
    s = sequence(a, b);
    s = Sequence{uniform(s.start), uniform(s.n), uniform(s.len)};
    j->row0 = uniform((unit - first_tile(a, b, s.start, ROWS)) * ROWS);
    // a slot before those of a first sequence that starts late
    if (j->row0 < 0) return false;
  } else {
    Unit u;
    if (!find_unit<ROWS, CHUNK>(a, unit, shared, &u)) return false;
    s = Sequence{uniform(u.seq.start), uniform(u.seq.n), uniform(u.seq.len)};
    b = uniform(u.b), j->chunk = uniform(u.chunk), j->chunks = uniform(u.chunks);
    j->row0 = uniform(u.tile) * ROWS;
    j->first = unit - j->chunk;
  }
  j->sequence = b;
  j->rows = min(ROWS, s.n * a.group - j->row0);
  if (j->rows <= 0) return false;
  const int visible = shared + uniform(visible_keys(s, j->row0, j->rows, a.group));
  j->token0 = s.start;
  j->own_base = s.len - s.n;
  j->own.ids = a.table + b * a.table_stride;
  // this chunk's keys [k0, k1) of those that the rows see, the prefix's before the own
  int k0 = 0, k1 = visible;
  if constexpr (MODE != kWhole) {
    const int each = uniform((int)(((uint32_t)(visible + j->chunks - 1) / (uint32_t)j->chunks + GRAIN - 1) / GRAIN) * GRAIN);
    k0 = min(j->chunk * each, visible);
    k1 = min(k0 + each, visible);
  }
  j->prefix.first = min(k0, shared), j->prefix.last = min(k1, shared) - 1;
  // own keys are aligned to their pages: a chunk's bounds go down to whole groups of 16 of them
  const int o0 = max(0, k0 - shared), o1 = max(0, k1 - shared);
  j->own.first = o0 & ~15;
  j->own.last = (k0 == k1 ? j->own.first : k1 == visible ? o1 : o1 & ~15) - 1;
  j->tiles0 = (j->prefix.last - j->prefix.first + KT) / KT;
  j->tiles = j->tiles0 + (j->own.last - j->own.first + KT) / KT;
  return true;
}

// A job's fields again as values that the compiler knows to be the same in all
// lanes (page ids then come by scalar loads).
__device__ __forceinline__ Keys uniform(const Keys& k) {
  const uint64_t p = (uint64_t)k.ids;
  const uint64_t ids = (uint32_t)uniform((int)(uint32_t)p) | (uint64_t)(uint32_t)uniform((int)(p >> 32)) << 32;
  return Keys{(const int32_t*)ids, uniform(k.first), uniform(k.last)};
}
__device__ __forceinline__ Job uniform(const Job& j) {
  return Job{uniform(j.prefix), uniform(j.own),      uniform(j.tiles0), uniform(j.tiles), uniform(j.token0), uniform(j.row0),
             uniform(j.rows),   uniform(j.own_base), uniform(j.sequence), uniform(j.first), uniform(j.chunk), uniform(j.chunks)};
}

// ---------------------------------------------------------------------------
// Joining the chunks of a row tile: each workgroup writes its partial result
// with device-scope stores, which gfx950 performs past the XCD's L2, waits for
// them, and counts in on the tile's counter; the one that counts last joins
// the partials, in chunk order whichever it is, and leaves the counter at 0.
// No cache-wide fence, one launch.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void store_device(float* p, float x, float y) {
  const uint64_t v = (uint64_t)__float_as_uint(x) | (uint64_t)__float_as_uint(y) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_device(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return float2{__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32))};
}
// Whether this workgroup is the tile's last; `flag`: a word of LDS.
__device__ __forceinline__ bool counts_last(int32_t* counter, int chunks, volatile int* flag) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == chunks - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = last;
  }
  __syncthreads();
  return *flag != 0;
}

template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (N > 0) {
    static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// The factors that bring a result with reference `top` and one with reference
// `ref` to their common one, which becomes `top`. A part without keys has the
// reference -inf and counts for nothing. One with a NaN score has the reference
// NaN, which no later part takes away: fmaxf would drop it.
__device__ __forceinline__ float2 join_factors(float* top, float ref) {
  const float next = __builtin_isunordered(*top, ref) ? __builtin_nanf("") : fmaxf(*top, ref);
  const float2 f{*top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(*top - next),
                 ref == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref - next)};
  *top = next;
  return f;
}
// a f.x + b f.y. The sums of a part without keys are 0; a NaN under a factor
// that is 0 in 32 bits stays NaN, as it does under such a weight.
__device__ __forceinline__ float joined(float2 f, float a, float b) { return a * f.x + b * f.y; }

// Where the copies of a key tile come from. A wave copies rows of one aligned
// group of 16 keys, which lies in one page: the page's id comes by a scalar
// load a tile ahead of its use. Keys past a run's last come from its last
// group or are the last key again, so nothing outside a sequence's keys is
// read; the scores mask them.
struct Group {
  int first, left;  // key index of the group's first key, and how many the run has after it
  int id;           // its page
};
__device__ __forceinline__ Group group_at(const AttnArgs& a, const Keys& run, int key) {
  const int first = min(key & ~15, run.last & ~15);
  return Group{first, run.last - first, read_only(run.ids, first >> a.page_shift)};
}
// Offset of the group in K and in V, for one head, in bytes.
__device__ __forceinline__ int64_t group_offset(const AttnArgs& a, const Group& g, int head, int row_bytes) {
  const uint32_t id = min((uint32_t)max(g.id, 0), (uint32_t)(a.pages - 1));
  return ((((int64_t)id * a.kv_heads + head) << a.page_shift) + (g.first & ((1 << a.page_shift) - 1))) * row_bytes;
}

// Output rows: o of channels d .. d + 3 of a row, as the 16-bit type.
template <class H>
__device__ __forceinline__ void store4(uint16_t* p, f32x4 o) {
  *reinterpret_cast<uint2*>(p) = uint2{H::pack(o.x, o.y), H::pack(o.z, o.w)};
}

// Non-finite values of V where some row does not see them. 0 * V is not 0
// there, so a key tile that is masked for any row is looked through before its
// product; if it holds such values (rare), they are set to 0 in LDS and each
// channel's first key of each kind is noted. A row sees a channel's values
// if it sees the first, so at the end the output takes what the noted ones
// bring: NaN, or an infinity of the one sign that it sees.
constexpr int kNever = 0x7FFFFFFF, kAlways = -kNever;
template <int D>
struct NonFinite {
  int first[3 * D];  // NaN, +inf, -inf of each channel: the key's index, kNever if there is none
  int tile;          // a tile that holds some, plus 1
};

template <int D>
__device__ __forceinline__ void init_non_finite(NonFinite<D>* n, int threads) {
  for (int i = threadIdx.x; i < 3 * D; i += threads) n->first[i] = kNever;
  if (threadIdx.x == 0) n->tile = 0;
}

// Whether any of the wave's 16-byte chunks of a tile (64 lanes x STEPS, from
// v = tile + lane * 16 on) has all exponent bits set in some 16-bit value.
template <class H, int STEPS>
__device__ __forceinline__ bool holds_non_finite(const uint8_t* v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const i32x4 x = lds_read16(v + i * 1024);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      bad |= ((uint32_t)x[e] & H::kInf) == H::kInf || (((uint32_t)x[e] >> 16) & H::kInf) == H::kInf;
  }
  return __any(bad);
}

// Sets the non-finite values of the same chunks to 0 and notes them. key0: key
// index of the tile's row 0, or kAlways where every row sees the tile's keys;
// rows past the run's last key (copies of it) are not noted.
template <class H, int D, int STEPS>
__device__ __forceinline__ void take_non_finite(uint8_t* tile, int chunk0, int key0, int rows, NonFinite<D>* n) {
#pragma unroll 1
  for (int i = 0; i < STEPS * 8; ++i) {
    const int chunk = chunk0 + (i >> 3) * 64, row = chunk / (D / 8);
    uint16_t* at = reinterpret_cast<uint16_t*>(tile + chunk * 16) + (i & 7);
    const uint32_t x = *at, m = x & 0x7FFFu;
    if (m < H::kInf) continue;
    *at = 0;
    if (row >= rows) continue;
    const int d = ((chunk % (D / 8)) ^ v_swizzle<D>(row)) * 8 + (i & 7);
    atomicMin(&n->first[(m > H::kInf ? 0 : x == H::kInf ? D : 2 * D) + d], key0 == kAlways ? kAlways : key0 + row);
  }
}

// The output of channel d for a row that sees the own keys up to `sees`.
template <int D>
__device__ __forceinline__ float with_non_finite(float o, const NonFinite<D>& n, int d, int sees) {
  const bool up = n.first[D + d] <= sees, down = n.first[2 * D + d] <= sees;
  if (n.first[d] <= sees || (up && down)) return __builtin_nanf("");
  return up ? o + __builtin_inff() : down ? o - __builtin_inff() : o;
}

// ---------------------------------------------------------------------------
// Few rows (up to 16): a decode step. HBM-bound: each wave streams 16-key
// tiles of its own through its own ring of two stages, with no barrier, and
// the waves' results meet in LDS at the end. 16x16 MFMA; a lane holds row
// lane % 16 and keys 4 (lane / 16) + 0..3 of a tile.
//
// 4 sequences of 32000 to 59000 keys (4 heads of 256, 719 MB) take 128 us, 5.6
// TB/s; a ragged batch of 64 (8 heads of 128, 124 MB) 31, 4.0 TB/s: a workgroup
// has about 5 us of finding its unit, the first copies and the join beside its
// keys. One sequence of 517 keys takes 8.6 us, a launch and that chain. (Thirty
// calls of a graph, their inputs in turn.)
// ---------------------------------------------------------------------------
// Partial results that a thread has in flight when it joins them.
constexpr int kJoinAhead = 8;

// Tokens that belong to no sequence come out as 0: those before the first start
// and past the last. A workgroup clears its share of a head's, a wave a token
// at a time. (One workgroup a head took 900 us for a prompt of 100 tokens padded
// to 8192, 32 heads of 128 channels; the prompt alone takes 12, filling the
// output 12, both now 21.) The starts come by one vector load ahead of those
// that find the workgroup's job: 0.2 us at most for calls without such tokens,
// 0.4 if they come by scalar loads.
__device__ __forceinline__ int edge_starts(const AttnArgs& a, int lane) { return a.starts ? a.starts[lane & 1 ? a.batch : 0] : 0; }
template <int D>
__device__ __forceinline__ void zero_loose_tokens(const AttnArgs& a, int edges, int unit, int head, int wave, int lane) {
  if (!a.starts) return;
  const int first = clamped(lane_value(edges, 0), 0, a.tokens), end = clamped(lane_value(edges, 1), first, a.tokens);
  const int n = first + a.tokens - end;
  for (int i = unit * 4 + wave; i < n; i += a.p.own_units * 4) {
    const int64_t token = i < first ? i : end + (i - first);
    uint4* to = reinterpret_cast<uint4*>(a.out + (token * a.q_heads + (int64_t)head * a.group) * D);
    for (int c = lane; c < a.group * (D / 8); c += 64) to[c] = uint4{0, 0, 0, 0};
  }
}

// Four channels of a row put together from parts.
struct Joined {
  float top = -__builtin_inff(), total = 0.0f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(float ref, float sum, f32x4 x) {
    const float2 f = join_factors(&top, ref);
    total = joined(f, total, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = joined(f, o[e], x[e]);
  }
};

template <int D>
struct Few {
  static constexpr int kWaves = 4, kTile = 16, kStage = 2 * kTile * 2 * D, kGrain = kTile * kWaves, kChunk = 2 * kGrain;
  static constexpr int kRings = kWaves * 2 * kStage, kMerge = kWaves * kFewRows * (D + 2) * 4 + 64 * kWaves * 24;
  static constexpr int kLds = kRings > kMerge ? kRings : kMerge;  // NonFinite comes after
};

template <class H, int D, Mode MODE>
__device__ __forceinline__ void attend_few(const AttnArgs& a, int block, uint8_t* lds) {
  constexpr int W = Few<D>::kWaves, KT = Few<D>::kTile, STAGE = Few<D>::kStage, ROWB = 2 * D;
  constexpr int COPIES = KT * ROWB / 1024, CHUNKS = D / 8, RPC = 64 / CHUNKS;  // copies of a tile, rows of a copy
  NonFinite<D>& bad = *reinterpret_cast<NonFinite<D>*>(lds + Few<D>::kLds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  init_non_finite(&bad, 64 * W);
  const int unit = (int)((uint32_t)block / (uint32_t)a.kv_heads), head = block - unit * a.kv_heads;
  const bool joined_later = a.prefix_len > 0;  // by join_kernel, with the prefix's shares
  const int edges = MODE == kOwn ? edge_starts(a, lane) : 0;
  Job found;
  const bool any = find_job<MODE, kFewRows, KT, Few<D>::kGrain, Few<D>::kChunk>(a, unit, &found);
  if (MODE == kOwn && !joined_later) zero_loose_tokens<D>(a, edges, unit, head, wave, lane);
  if (!any) return;
  const Job j = uniform(found);
  constexpr bool PREFIX = MODE == kPrefix;
  const Keys run = PREFIX ? j.prefix : j.own;
  const int group = a.group, li = lane & 15, quarter = lane >> 4;

  // Q as the B operand: row li, channels 32 ks + 8 quarter ..
  const int row = min(li, j.rows - 1);
  const uint32_t qrow = (uint32_t)(j.row0 + row), qtoken = qrow / (uint32_t)group, qg = qrow % (uint32_t)group;
  const uint16_t* qp = a.q + (j.token0 + (int64_t)qtoken) * a.q_ts + (int64_t)(head * group + (int)qg) * a.q_hs + quarter * 8;
  i32x4 q[D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) q[ks] = *reinterpret_cast<const i32x4*>(qp + ks * 32);
  const int sees = PREFIX ? run.last : min(j.own_base + (int)qtoken, run.last);
  // below this key every row of the tile sees all
  const int all_see = PREFIX ? run.last : min(j.own_base + (int)((uint32_t)j.row0 / (uint32_t)group), run.last);

  uint8_t* ring = lds + wave * 2 * STAGE;
  const int copy_row = lane / CHUNKS;
  const uint32_t k_chunk = (uint32_t)((lane & (CHUNKS - 1)) ^ k_swizzle<D>(copy_row));
  const uint32_t v_chunk = (uint32_t)((lane & (CHUNKS - 1)) ^ v_swizzle<D>(copy_row));
  const int n_tiles = (j.tiles - wave + W - 1) / W;  // this wave's: wave, wave + W, ..
  const auto group_of = [&](int t) { return group_at(a, run, run.first + (t * W + wave) * KT); };
  const auto issue = [&](int t, const Group& g) {
    uint8_t* dst = ring + (t & 1) * STAGE;
    const int64_t off = group_offset(a, g, head, ROWB);
    const uint8_t *ks = reinterpret_cast<const uint8_t*>(a.k_pages) + off, *vs = reinterpret_cast<const uint8_t*>(a.v_pages) + off;
#pragma unroll
    for (int i = 0; i < COPIES; ++i)
      load_lds16(ks + ((uint32_t)min(i * RPC + copy_row, g.left) * ROWB + (k_chunk ^ k_swizzle<D>(i * RPC)) * 16), dst + i * 1024);
#pragma unroll
    for (int i = 0; i < COPIES; ++i)
      load_lds16(vs + ((uint32_t)min(i * RPC + copy_row, g.left) * ROWB + (v_chunk ^ v_swizzle<D>(i * RPC)) * 16),
                 dst + KT * ROWB + i * 1024);
  };

  f32x4 o[D / 16];
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float ref = -__builtin_inff(), sum = 0.0f;
  float limit = ref, sub = 0.0f;  // what moves the reference, what is taken off an exponent
  lds_barrier();  // `bad` is set up
  Group next{};
  if (n_tiles > 0) {
    issue(0, group_of(0));
    next = group_of(min(1, n_tiles - 1));
  }
  for (int t = 0; t < n_tiles; ++t) {
    const int key0 = run.first + (t * W + wave) * KT;
    const uint8_t* kt = ring + (t & 1) * STAGE;
    uint8_t* vt = ring + (t & 1) * STAGE + KT * ROWB;
    if (t + 1 < n_tiles) {
      issue(t + 1, next);
      next = group_of(min(t + 2, n_tiles - 1));
      wait_vmem_below<3 * COPIES>();
    } else {
      wait_vmem_below<COPIES>();
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x4 s{0.f, 0.f, 0.f, 0.f};
    i32x4 kf[D / 32];
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) kf[ks] = lds_read16(kt + li * ROWB + (((ks * 4 + quarter) ^ k_swizzle<D>(li)) * 16));
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks) s = H::mfma16(kf[ks], q[ks], s);
    settle(&s);
    const bool masked = key0 + KT - 1 > all_see;
    if (masked) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (key0 + quarter * 4 + e > sees) s[e] = -__builtin_inff();
    }
    float top = fmaxf(fmaxf(s.x, s.y), fmaxf(s.z, s.w));
    if (__any(top * a.scale_log2 > limit)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float next = top * a.scale_log2 > ref + kRescaleAt ? top * a.scale_log2 : ref;
      const float f = ref == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref - next);
      sum *= f;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) o[dt] *= f;
      ref = next;
      limit = moved_to<H, 1>(ref, a.scale_log2, &sub, &s);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.scale_log2, -sub));
      sum += s[e];
    }
    asm volatile("" : "+v"(sum));  // added up here, not after the weights' last use
    // what the 16-bit weights leave goes through the product as well
    const uint2 pw{H::pack(s.x, s.y), H::pack(s.z, s.w)};
    const uint2 rest{H::pack(s.x - H::lo(pw.x), s.y - H::hi(pw.x)), H::pack(s.z - H::lo(pw.y), s.w - H::hi(pw.y))};
    const s16x4 pb = __builtin_bit_cast(s16x4, pw), pr = __builtin_bit_cast(s16x4, rest);
    if (t + 1 < n_tiles) wait_vmem_below<2 * COPIES>();
    else wait_vmem_below<0>();
    __builtin_amdgcn_sched_barrier(0);
    if (masked && holds_non_finite<H, COPIES>(vt + lane * 16)) {
      take_non_finite<H, D, COPIES>(vt, lane, PREFIX ? kAlways : key0, run.last - key0 + 1, &bad);
      if (lane == 0) bad.tile = 1;
    }
    // V^T: channels 16 dt + li, keys 4 quarter + 0..3; a chunk's swizzle changes
    // its lower four bits only, so dt + 8 lies 256 bytes on
    constexpr int AHEAD = D == 64 ? 4 : 8;
    uint32_t at[AHEAD];
    {
      const int r = quarter * 4 + (li >> 2);
      const uint32_t base = lds_address(vt) + r * ROWB + (li & 1) * 8;
#pragma unroll
      for (int dt = 0; dt < AHEAD; ++dt) at[dt] = base + (((dt * 2 + ((li >> 1) & 1)) ^ v_swizzle<D>(r)) * 16);
    }
    s16x4 v[D / 16];
#pragma unroll
    for (int dt = 0; dt < AHEAD; dt += 4) lds_read_tr4<0>(at[dt], at[dt + 1], at[dt + 2], at[dt + 3], v + dt);
    if constexpr (D == 256) {
#pragma unroll
      for (int dt = 0; dt < AHEAD; dt += 4) lds_read_tr4<256>(at[dt], at[dt + 1], at[dt + 2], at[dt + 3], v + 8 + dt);
    }
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[dt] = H::mfma16k16(v[dt], pr, o[dt]);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[dt] = H::mfma16k16(v[dt], pb, o[dt]);
  }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (sum != sum) ref = sum;  // a NaN that no score set the reference for

  // The waves' results, in wave order: [wave][row][D + 2] floats over the rings.
  __syncthreads();
  float* m = reinterpret_cast<float*>(lds);
  {
    float* mine = m + (wave * kFewRows + li) * (D + 2);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[dt * 16 + quarter * 4 + e] = o[dt][e];
    if (quarter == 0) mine[D] = ref, mine[D + 1] = sum;
  }
  __syncthreads();
  const int items = j.rows * (D / 4);  // four channels of a row each
  const int64_t part = (int64_t)unit * a.kv_heads + head;
  float* part_o = (PREFIX ? a.prefix_o : a.part_o) + part * kFewRows * D;
  float2* part_ml = (PREFIX ? a.prefix_ml : a.part_ml) + part * kFewRows;
  const auto write = [&](int i, const Joined& x) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    const uint32_t rr = (uint32_t)(j.row0 + r), tk = rr / (uint32_t)group, g = rr % (uint32_t)group;
    store4<H>(a.out + ((j.token0 + (int64_t)tk) * a.q_heads + head * group + (int)g) * D + d,
              x.o * (x.total == 0.0f ? 0.0f : 1.0f / x.total));
  };
  for (int i = threadIdx.x; i < items; i += 64 * W) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    Joined x;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float* from = m + (w * kFewRows + r) * (D + 2);
      x.add(from[D], from[D + 1], f32x4{from[d], from[d + 1], from[d + 2], from[d + 3]});
    }
    if (bad.tile) {
      const int sees_own = j.own_base + (int)((uint32_t)(j.row0 + r) / (uint32_t)group);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.o[e] = with_non_finite(x.o[e], bad, d + e, PREFIX ? 0 : sees_own);
    }
    if (PREFIX || joined_later) {
      *reinterpret_cast<f32x4*>(part_o + r * D + d) = x.o;
      if (d == 0) part_ml[r] = float2{x.top, x.total};
    } else if (j.chunks == 1) {
      write(i, x);
    } else {
      store_device(part_o + r * D + d, x.o.x, x.o.y);
      store_device(part_o + r * D + d + 2, x.o.z, x.o.w);
      if (d == 0) store_device(reinterpret_cast<float*>(part_ml + r), x.top, x.total);
    }
  }
  if (PREFIX) return;
  if (joined_later) {
    if (head == 0 && j.chunk == 0 && j.row0 == 0 && threadIdx.x == 0) a.info[j.sequence] = int2{j.first, j.chunks};
    return;
  }
  if (j.chunks == 1) return;
  if (!counts_last(a.counters + (int64_t)j.first * a.kv_heads + head, j.chunks, &bad.tile)) return;
  // The chunks' results: `each` threads take turns on an item's parts, several
  // in flight a thread, and meet in LDS.
  const int each = items >= 64 * W ? 1 : 64 * W / items;
  for (int base = 0; base < items; base += 64 * W) {
    const int turn = each == 1 ? 0 : (int)((uint32_t)threadIdx.x / (uint32_t)items);
    const int i = base + (int)threadIdx.x - turn * items;
    const bool active = i < items && turn < each;
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    Joined x;
    if (active) {
      const int64_t first = ((int64_t)j.first * a.kv_heads + head) * kFewRows + r;
      for (int c = turn; c < j.chunks; c += each * kJoinAhead) {
        float2 ml[kJoinAhead], v[kJoinAhead][2];
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
          const int64_t at = first + (int64_t)min(c + u * each, j.chunks - 1) * a.kv_heads * kFewRows;
          ml[u] = load_device(reinterpret_cast<const float*>(a.part_ml + at));
          v[u][0] = load_device(a.part_o + at * D + d);
          v[u][1] = load_device(a.part_o + at * D + d + 2);
        }
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u)
          if (c + u * each < j.chunks) x.add(ml[u].x, ml[u].y, f32x4{v[u][0].x, v[u][0].y, v[u][1].x, v[u][1].y});
      }
    }
    if (each > 1) {
      float* red = m + W * kFewRows * (D + 2);
      if (active && turn > 0) {
        float* to = red + threadIdx.x * 6;
        to[0] = x.top, to[1] = x.total;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[2 + e] = x.o[e];
      }
      __syncthreads();
      if (turn == 0) {
        for (int k = 1; k < each; ++k) {
          const float* from = red + (threadIdx.x + k * items) * 6;
          x.add(from[0], from[1], f32x4{from[2], from[3], from[4], from[5]});
        }
      }
    }
    if (active && turn == 0) write(i, x);
  }
}

// ---------------------------------------------------------------------------
// Many rows: tiles of 128, four waves of 32 rows that share the key tiles.
// 32x32x16 MFMA; a lane holds row lane % 32 and keys 8 i + 4 (lane / 32) + 0..3.
// Two stages: while a tile is multiplied the next one's copies are in flight;
// one barrier a tile. The next 16 keys' weights are worked out between the
// products of the ones before, which hides the exponentials (8% of the time
// without that).
//
// Prompts of 8192 tokens take 558 us with 32 heads of 128 (985 TFLOP/s; a large
// bf16 library product reaches 1200 beside it), 535 with 16 of 256 (1025) and 326
// with 32 of 64 (840), in thirty calls of a graph. Nothing alone bounds it: with
// 32 heads of 128 MFMA is busy 48% of the time and LDS 24%, without conflicts, and
// VALU instructions, the exponentials among them, take 30% at four cycles each; a
// wave does one after the other but for what is laid between the products. Eight
// waves a workgroup (108 instead of 85 us for 16 sequences over a prefix of 2000)
// and 32-key tiles at three waves a SIMD (even) were no better. Short prompts wait
// for HBM beside it: 16 of 512 tokens move 167 MB in 73 us.
// ---------------------------------------------------------------------------
template <int D>
struct Many {
  // A chunk's partial results, 4 D bytes a row, have to be worth its keys. With
  // 256, 384, 640 and 896 keys at least: 64 queries of 32 heads over 4000 keys
  // 33, 29, 29 and 31 us; 4 sequences of 200 queries of 16 heads of 256 over 1000
  // keys 55, 52, 44 and 44; prompts of 1024 tokens of those heads 46, 37, 39 and
  // 46, of 1500 tokens of 32 heads of 128 51, 51, 48 and 46.
  static constexpr int kTile = D == 256 ? 32 : 64, kGrain = 64, kChunk = 640;
  static constexpr int kLds = 2 * 2 * kTile * 2 * D;  // two stages; NonFinite comes after
};

// The tile of the nth workgroups of whole tiles. The last tiles, which see the
// most keys, come first; of the workgroups that come to a CU second, though,
// those of the fewest keys, so that a long and a short tile share a CU.
__device__ __forceinline__ int whole_unit(const AttnPlan& p, int nth) {
  const int both = min(p.own_units, 2 * p.cu_units);
  if (nth >= p.cu_units && nth < both) nth = p.cu_units + both - 1 - nth;
  return p.own_units - 1 - nth;
}

template <class H, int D, Mode MODE>
__device__ __forceinline__ void attend_many(const AttnArgs& a, int block, uint8_t* lds) {
  constexpr int KT = Many<D>::kTile, SUB = KT / 32, ROWB = 2 * D, STAGE = 2 * KT * ROWB;
  constexpr int CHUNKS = D / 8, RPC = 64 / CHUNKS, COPIES = KT * ROWB / 1024 / 4;  // copies of a wave, of K and of V
  NonFinite<D>& bad = *reinterpret_cast<NonFinite<D>*>(lds + Many<D>::kLds);
  init_non_finite(&bad, 256);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nth = (int)((uint32_t)block / (uint32_t)a.kv_heads), head = block - nth * a.kv_heads;
  const int unit = MODE == kWhole ? whole_unit(a.p, nth) : nth;
  const int group = a.group, li = lane & 31, half = lane >> 5;
  const int edges = MODE == kPrefix ? 0 : edge_starts(a, lane);
  Job found;
  const bool any = find_job<MODE, kManyRows, KT, Many<D>::kGrain, Many<D>::kChunk>(a, unit, &found);
  if (MODE != kPrefix) zero_loose_tokens<D>(a, edges, unit, head, wave, lane);
  if (!any) return;
  const Job j = uniform(found);

  const int row = min(wave * 32 + li, j.rows - 1);
  const uint32_t qrow = (uint32_t)(j.row0 + row), qtoken = qrow / (uint32_t)group, qg = qrow % (uint32_t)group;
  const uint16_t* qp = a.q + (j.token0 + (int64_t)qtoken) * a.q_ts + (int64_t)(head * group + (int)qg) * a.q_hs + half * 8;
  i32x4 q[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) q[ks] = *reinterpret_cast<const i32x4*>(qp + ks * 16);
  const int sees = j.own_base + (int)qtoken;
  // own keys that every row of the wave sees, and every row of the workgroup
  const int all_see = j.own_base + (int)((uint32_t)(j.row0 + min(wave * 32, j.rows - 1)) / (uint32_t)group);
  const int wg_sees = j.own_base + (int)((uint32_t)j.row0 / (uint32_t)group);

  const int copy_row = lane / CHUNKS;
  // the 16-byte chunk that a lane copies of a row, for the copy's rows from 0 on
  const uint32_t k_chunk = (uint32_t)((lane & (CHUNKS - 1)) ^ k_swizzle<D>(copy_row));
  const uint32_t v_chunk = (uint32_t)((lane & (CHUNKS - 1)) ^ v_swizzle<D>(copy_row));
  constexpr int ROWS_OF_WAVE = COPIES * RPC;
  static_assert(16 % ROWS_OF_WAVE == 0, "a wave's rows lie in one group of 16 keys");
  const auto group_of = [&](int t) {
    const bool first = MODE == kPrefix || t < j.tiles0;
    const Keys run{first ? j.prefix.ids : j.own.ids, first ? j.prefix.first : j.own.first, first ? j.prefix.last : j.own.last};
    return group_at(a, run, run.first + (first ? t : t - j.tiles0) * KT + wave * ROWS_OF_WAVE);
  };
  const auto issue = [&](int t, const Group& g) {
    uint8_t* dst = lds + (t & 1) * STAGE + wave * ROWS_OF_WAVE * ROWB;
    const int64_t off = group_offset(a, g, head, ROWB);
    const uint8_t *ks = reinterpret_cast<const uint8_t*>(a.k_pages) + off, *vs = reinterpret_cast<const uint8_t*>(a.v_pages) + off;
    const uint32_t kc = fresh(k_chunk), vc = fresh(v_chunk);
#pragma unroll
    for (int i = 0; i < COPIES; ++i) {
      const int r = wave * ROWS_OF_WAVE + i * RPC;  // row of the tile; of the group, r % 16
      const uint32_t row = (uint32_t)min((r & 15) + copy_row, g.left) * ROWB;
      load_lds16(ks + (row + (kc ^ k_swizzle<D>(r)) * 16), dst + i * 1024);
      load_lds16(vs + (row + (vc ^ v_swizzle<D>(r)) * 16), dst + KT * ROWB + i * 1024);
    }
  };
  // LDS addresses in stage 0: K row li, channels 8 half ..; V rows 4 half + ..,
  // channels (li / 16) 16 .. for the transposing read
  const int v_row = half * 4 + ((li & 15) >> 2);
  const uint32_t k_at = lds_address(lds) + li * ROWB + ((half ^ k_swizzle<D>(li)) * 16);
  const uint32_t v_at = lds_address(lds) + (KT + v_row) * ROWB +
                        ((((li >> 4) * 2 + ((li >> 1) & 1)) ^ v_swizzle<D>(v_row)) * 16) + (li & 1) * 8;

  f32x16 o[D / 32];
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
  float ref = -__builtin_inff(), sum = 0.0f;
  float limit = ref, sub = 0.0f;  // what moves the reference, what is taken off an exponent
  Group next{};
  if (j.tiles > 0) {
    issue(0, group_of(0));
    next = group_of(min(1, j.tiles - 1));
  }
  for (int t = 0; t < j.tiles; ++t) {
    // this wave's copies of tile t have landed, then all waves': and all have
    // read the stage that the next copies overwrite
    wait_vmem_below<0>();
    lds_barrier();
    if (t + 1 < j.tiles) {
      issue(t + 1, next);
      next = group_of(min(t + 2, j.tiles - 1));
    }
    const bool first = MODE == kPrefix || t < j.tiles0;
    const int key0 = first ? j.prefix.first + t * KT : j.own.first + (t - j.tiles0) * KT;
    const int last = first ? j.prefix.last : j.own.last;
    const int row_last = first ? last : min(sees, last);
    const uint32_t stage = (uint32_t)(t & 1) * STAGE;
    // masked for some wave's rows: each wave looks through the quarter of V that it copied
    if (key0 + KT - 1 > (first ? last : min(wg_sees, last))) {
      uint8_t* vt = lds + stage + KT * ROWB;
      if (holds_non_finite<H, COPIES>(vt + wave * COPIES * 1024 + lane * 16) && lane == 0) bad.tile = t + 1;
      lds_barrier();
      if (bad.tile == t + 1) {
        take_non_finite<H, D, COPIES>(vt, wave * COPIES * 64 + lane, first ? kAlways : key0, last - key0 + 1, &bad);
        lds_barrier();
      }
    }
    if (wave * 32 >= j.rows) continue;  // a wave without rows has its copies and its looking through alone
    const uint32_t kt = fresh(k_at) + stage;
    f32x16 s[SUB];
#pragma unroll
    for (int b = 0; b < SUB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[b][e] = 0.0f;
    // channels 16 ks + 8 half ..: the chunk's index takes 2 ks by XOR. AHEAD
    // reads are under way while as many before them are multiplied.
    constexpr int AHEAD = D == 256 ? 2 : 4, STEPS = AHEAD / SUB, BATCHES = D / 16 / STEPS;
    i32x4 kf[2][AHEAD];
    const auto read_k = [&](int i) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) kf[i & 1][u] = lds_read16(kt ^ ((i * STEPS + u / SUB) * 32), (u % SUB) * 32 * ROWB);
    };
    read_k(0);
#pragma unroll
    for (int i = 0; i < BATCHES; ++i) {
      if (i + 1 < BATCHES) read_k(i + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) s[u % SUB] = H::mfma32(kf[i & 1][u], q[i * STEPS + u / SUB], s[u % SUB]);
    }
    const bool masked = key0 + KT - 1 > (first ? last : min(all_see, last));
    if (masked) {
#pragma unroll
      for (int b = 0; b < SUB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (key0 + b * 32 + (e >> 2) * 8 + half * 4 + (e & 3) > row_last) s[b][e] = -__builtin_inff();
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < SUB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[b][e]);
    if (__any(top * a.scale_log2 > limit)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float next = top * a.scale_log2 > ref + kRescaleAt ? top * a.scale_log2 : ref;
      const float f = ref == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref - next);
      sum *= f;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt) o[dt] *= f;
      ref = next;
      limit = moved_to<H, SUB>(ref, a.scale_log2, &sub, s);
    }
    // The weights of 16 keys, as the B operand of their step.
    const auto weights = [&](int ks) {
      i32x4 p;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks >> 1][(ks & 1) * 8 + e], a.scale_log2, -sub));
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[ks >> 1][(ks & 1) * 8 + e + 1], a.scale_log2, -sub));
        const uint32_t w = H::pack(x, y);
        sum = H::add2(w, sum);
        p[e >> 1] = (int)w;
      }
      asm volatile("" : "+v"(sum));  // added up here, not after the weights' last use
      return p;
    };
    // V^T: channels 32 dt + li (the chunk takes 4 dt by XOR), keys 16 ks + 4 half
    // + 0..3 and 8 more. The next 16 keys' weights are worked out while a step's
    // products run.
    constexpr int NB = D == 64 ? 2 : 4;  // channel blocks of a read
    const uint32_t vt = fresh(v_at) + stage;
    i32x4 p = weights(0);
    static_for<2 * SUB>([&](auto kc) {
      constexpr int ks = decltype(kc)::value;
      i32x4 next_p = p;
      static_for<D / 32 / NB>([&](auto gc) {
        constexpr int g = decltype(gc)::value;
        uint32_t at[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) at[i] = vt ^ (uint32_t)((g * NB + i) * 64);
        i32x4 v[NB];
        lds_read_tr8<NB, ks * 16 * ROWB, (ks * 16 + 8) * ROWB>(at, v);
#pragma unroll
        for (int i = 0; i < NB; ++i) o[g * NB + i] = H::mfma32(v[i], p, o[g * NB + i]);
        if constexpr (g == 0 && ks + 1 < 2 * SUB) next_p = weights(ks + 1);
      });
      p = next_p;
    });
  }
  sum += __shfl_xor(sum, 32);
  if (sum != sum) ref = sum;  // a NaN that no score set the reference for
  if (j.tiles > 0 && bad.tile) {
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        o[dt][e] = with_non_finite(o[dt][e], bad, dt * 32 + (e >> 2) * 8 + half * 4 + (e & 3), MODE == kPrefix ? 0 : sees);
  }
  const bool mine = wave * 32 + li < j.rows;
  const int64_t part = (int64_t)unit * a.kv_heads + head;
  if constexpr (MODE == kPrefix) {
    if (!mine) return;
    float* to = a.prefix_o + (part * kManyRows + row) * D + half * 4;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(to + dt * 32 + e * 2) = f32x4{o[dt][e], o[dt][e + 1], o[dt][e + 2], o[dt][e + 3]};
    if (half == 0) a.prefix_ml[part * kManyRows + row] = float2{ref, sum};
    return;
  }
  if (MODE == kSplit && j.chunks > 1) {
    // partials in register order: a wave's value pairs are 512 bytes apart
    const auto slot = [&](int c) { return (((int64_t)j.first + c) * a.kv_heads + head) * kManyRows; };
    const auto o_at = [&](int c, int dt, int e) {
      return a.part_o + slot(c) * D + wave * (32 * D) + ((dt * 8 + (e >> 1)) * 64 + lane) * 2;
    };
    const auto ml_at = [&](int c) { return reinterpret_cast<float*>(a.part_ml + slot(c) + wave * 32 + li); };
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 16; e += 2) store_device(o_at(j.chunk, dt, e), o[dt][e], o[dt][e + 1]);
    if (half == 0) store_device(ml_at(j.chunk), ref, sum);
    if (!counts_last(a.counters + (int64_t)j.first * a.kv_heads + head, j.chunks, &bad.tile)) return;
    // in chunk order, this one's from memory as well
    float top = -__builtin_inff(), total = 0.0f;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[dt][e] = 0.0f;
    constexpr int AHEAD = D < 128 ? D / 32 : 4;  // 32-channel blocks whose loads are in flight: 64 registers at most
    for (int c = 0; c < j.chunks; ++c) {
      const float2 ml = load_device(ml_at(c));
      float2 f;
#pragma unroll
      for (int dt = 0; dt < D / 32; dt += AHEAD) {
        float2 x[AHEAD][8];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
          for (int e = 0; e < 16; e += 2) x[u][e >> 1] = load_device(o_at(c, dt + u, e));
        if (dt == 0) f = join_factors(&top, ml.x), total = joined(f, total, ml.y);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            o[dt + u][e] = joined(f, o[dt + u][e], x[u][e >> 1].x);
            o[dt + u][e + 1] = joined(f, o[dt + u][e + 1], x[u][e >> 1].y);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    sum = total;
  }
  if (!mine) return;
  uint16_t* to = a.out + ((j.token0 + (int64_t)qtoken) * a.q_heads + head * group + (int)qg) * D + half * 4;
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      store4<H>(to + dt * 32 + e * 2, f32x4{o[dt][e], o[dt][e + 1], o[dt][e + 2], o[dt][e + 3]} * inv);
}

// ---------------------------------------------------------------------------
// The kernels: workgroups of 256 threads; registers for two waves a SIMD. One
// LDS array each: with two, the compiler's wait for copies into the one before
// reads of the other would empty the ring at every tile.
// ---------------------------------------------------------------------------
template <class H, int D>
__global__ __launch_bounds__(256) void attend_few_kernel(AttnArgs a) {
  __shared__ __align__(1024) uint8_t lds[Few<D>::kLds + sizeof(NonFinite<D>)];
  attend_few<H, D, kOwn>(a, blockIdx.x, lds);
}

template <class H, int D, Mode MODE>
__global__ __launch_bounds__(256, 2) void attend_many_kernel(AttnArgs a) {
  __shared__ __align__(1024) uint8_t lds[Many<D>::kLds + sizeof(NonFinite<D>)];
  attend_many<H, D, MODE>(a, blockIdx.x, lds);
}

// A decode batch with a prefix: shares of the prefix for all rows (the first
// workgroups) and chunks of the sequences' own keys side by side. 64 sequences
// (32 heads of 128) over 8192 keys: 22 us, a share of 8 key tiles most of them, and
// 6 of the join, which reads the 18 MB of parts that this kernel writes beside
// the case's 48 MB; in two launches, the own keys' after the prefix's, 6 more.
template <class H, int D, bool FEW_PREFIX>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_shared_kernel(AttnArgs a) {
  constexpr int LDS = FEW_PREFIX || Few<D>::kLds > Many<D>::kLds ? Few<D>::kLds : Many<D>::kLds;
  __shared__ __align__(1024) uint8_t lds[LDS + sizeof(NonFinite<D>)];
  const int prefix_blocks = a.p.prefix_tiles * a.p.prefix_splits * a.kv_heads, block = (int)blockIdx.x;
  if (block >= prefix_blocks) attend_few<H, D, kOwn>(a, block - prefix_blocks, lds);
  else if (FEW_PREFIX) attend_few<H, D, kPrefix>(a, block, lds);
  else attend_many<H, D, kPrefix>(a, block, lds);
}

// Joins a row's parts after attend_shared_kernel, the prefix's shares, then its
// own chunks: one wave a (token, head), all of up to 16 parts in flight.
template <class H, int D>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a) {
  constexpr int PER = D / 64, AHEAD = 16;
  const int lane = threadIdx.x & 63, id = (int)blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  if (id >= a.tokens * a.q_heads) return;
  const int token = (int)((uint32_t)id / (uint32_t)a.q_heads), qh = id - token * a.q_heads;
  const int head = (int)((uint32_t)qh / (uint32_t)a.group), g = qh - head * a.group;
  // The last sequence that starts at or before the token: those after it hold no token.
  int b = token;
  if (a.starts) {
    int count = 0;
    for (int base = 0; base < a.batch; base += 64) {
      const int c = __popcll(__ballot(base + lane < a.batch && start_of(a, min(base + lane, a.batch - 1)) <= token));
      count += c;
      if (c < 64) break;
    }
    b = uniform(count - 1);
  }
  uint16_t* to = a.out + (int64_t)id * D + lane * PER;
  const Sequence s = sequence(a, max(b, 0));
  const int r = (token - s.start) * a.group + g;
  if (b < 0 || (uint32_t)r >= (uint32_t)(s.n * a.group)) {  // a token of no sequence
#pragma unroll
    for (int e = 0; e < PER; ++e) to[e] = 0;
    return;
  }
  const int2 own = a.info[b];  // first unit, chunks of a tile
  const int prows = a.p.few_prefix ? kFewRows : kManyRows, prow = token * a.group + g, n_pre = a.p.prefix_splits;
  const int64_t pre0 = ((int64_t)(prow / prows) * n_pre * a.kv_heads + head) * prows + prow % prows;
  // held in range: starts that decrease leave sequences without units
  const int own0 = own.x + r / kFewRows * own.y, n = n_pre + clamped(own.y, 1, a.p.own_units);
  const auto part = [&](int i) {
    if (i < n_pre) return pre0 + (int64_t)i * a.kv_heads * prows;
    const int unit = clamped(own0 + i - n_pre, 0, a.p.own_units - 1);
    return ((int64_t)unit * a.kv_heads + head) * kFewRows + r % kFewRows;
  };
  float o[PER], top = -__builtin_inff(), total = 0.0f;
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.0f;
  for (int i = 0; i < n; i += AHEAD) {
    float2 ml[AHEAD];
    float x[AHEAD][PER];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int k = min(i + u, n - 1);
      const int64_t at = part(k);
      const float* from = (k < n_pre ? a.prefix_o : a.part_o) + at * D + lane * PER;
      ml[u] = (k < n_pre ? a.prefix_ml : a.part_ml)[at];
#pragma unroll
      for (int e = 0; e < PER; ++e) x[u][e] = from[e];
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (i + u < n) {
        const float2 f = join_factors(&top, ml[u].x);
        total = joined(f, total, ml[u].y);
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = joined(f, o[e], x[u][e]);
      }
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if constexpr (PER == 1) {
    to[0] = (uint16_t)H::pack(o[0] * inv, 0.0f);
  } else {
#pragma unroll
    for (int e = 0; e < PER; e += 2) reinterpret_cast<uint32_t*>(to)[e / 2] = H::pack(o[e] * inv, o[e + 1] * inv);
  }
}

// ---------------------------------------------------------------------------
// The plan and the launches.
// ---------------------------------------------------------------------------
AttnPlan attention_plan(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t prefix_len,
                        bool ragged, int cus) {
  AttnPlan p{};
  const int64_t group = q_heads / kv_heads, all_rows = tokens * group;
  // 16 sequences over 1000 keys, 8 heads of 4 query heads each: of 4 queries 21.5
  // us in tiles of few rows and 22.5 of many, of 8 queries 21.6 and 22.9, of 16
  // 36 and 24; one query of 2000 keys 11 and 21.
  p.few_own = all_rows <= batch * kFewRows;
  const int64_t rows = p.few_own ? kFewRows : kManyRows;
  const int64_t tiles = !ragged && group <= rows ? batch : all_rows / rows + batch;
  // units that the device holds at a time: by LDS, two workgroups a CU of the
  // many-row kernel, 4, 2 or 1 of the few-row kernel
  const int64_t at_once = cus * (p.few_own ? 256 / dim : 2) / kv_heads;
  // Many-row tiles that fill the device stay whole: cutting them too, a prompt
  // of 2048 tokens (32 heads of 128) takes 73 us instead of 56, 16 sequences of
  // 128 queries over 1000 keys 77 instead of 51.
  p.split = p.few_own || tiles < at_once;
  p.at_once = (int)std::max<int64_t>(1, at_once);
  p.cu_units = (int)(cus / kv_heads);
  p.tiles = (int)tiles;
  p.own_units = (int)(!p.split ? tiles : p.few_own ? std::max<int64_t>(at_once, tiles + at_once / 2) : at_once);
  // chunks that are not joined in a launch of their own are counted in
  const bool counted = p.split && !(p.few_own && prefix_len > 0);
  if (counted && p.own_units * kv_heads > kAttnCounters) p.split = false, p.own_units = (int)tiles;
  if (p.few_own && prefix_len > 0) {
    // in tiles of few rows and of many: 16 rows over 1000 keys 10.8 and 12.7 us, 32
    // rows 10.9 and 12.9, 32 over 8192 16.6 and 18.4; 64 rows 19.8 and 20.1
    p.few_prefix = all_rows <= 2 * kFewRows;
    const int64_t prows = p.few_prefix ? kFewRows : kManyRows;
    p.prefix_tiles = (int)((all_rows + prows - 1) / prows);
    // one workgroup a CU, of 256 keys at least: each writes its rows' results in
    // 32 bits (two a CU: 37 us instead of 31 for 64 sequences over 8192 keys; 128
    // keys: 24.7 instead of 19.2 for 32 over 4096, 14.0 instead of 15.9 over 1024)
    const int64_t share = std::max<int64_t>(1, cus / (kv_heads * p.prefix_tiles));
    p.prefix_splits = (int)std::min(share, (prefix_len + 255) / 256);
  }
  return p;
}

static int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// Bytes of a call's workspace; with `a`, its parts from `base` on.
static int64_t carve(const AttnPlan& p, int64_t batch, int64_t kv_heads, int64_t dim, uint8_t* base, AttnArgs* a) {
  const bool parts = p.split || p.prefix_tiles;
  const int64_t own = parts ? (int64_t)p.own_units * kv_heads * (p.few_own ? kFewRows : kManyRows) : 0;
  const int64_t pre = (int64_t)p.prefix_tiles * p.prefix_splits * kv_heads * (p.few_prefix ? kFewRows : kManyRows);
  const int64_t sizes[] = {own * dim * 4, own * 8, pre * dim * 4, pre * 8, pre ? batch * 8 : 0};
  int64_t at[6] = {0};
  for (int i = 0; i < 5; ++i) at[i + 1] = at[i] + up256(sizes[i]);
  if (a) {
    a->part_o = (float*)(base + at[0]), a->part_ml = (float2*)(base + at[1]);
    a->prefix_o = (float*)(base + at[2]), a->prefix_ml = (float2*)(base + at[3]);
    a->info = (int2*)(base + at[4]);
  }
  return at[5];
}

int64_t attention_workspace(const AttnPlan& p, int64_t batch, int64_t kv_heads, int64_t dim) {
  return carve(p, batch, kv_heads, dim, nullptr, nullptr);
}

template <class H, int D>
static void launch_attention(const AttnArgs& a, hipStream_t stream) {
  const AttnPlan& p = a.p;
  const unsigned own = (unsigned)(p.own_units * a.kv_heads), pre = (unsigned)(p.prefix_tiles * p.prefix_splits * a.kv_heads);
  if (pre) {
    if (p.few_prefix) attend_shared_kernel<H, D, true><<<pre + own, 256, 0, stream>>>(a);
    else attend_shared_kernel<H, D, false><<<pre + own, 256, 0, stream>>>(a);
    join_kernel<H, D><<<(unsigned)((a.tokens * a.q_heads + 3) / 4), 256, 0, stream>>>(a);
  } else if (p.few_own) {  // also where not split: a chunk a tile
    attend_few_kernel<H, D><<<own, 256, 0, stream>>>(a);
  } else if (p.split) {
    attend_many_kernel<H, D, kSplit><<<own, 256, 0, stream>>>(a);
  } else {
    attend_many_kernel<H, D, kWhole><<<own, 256, 0, stream>>>(a);
  }
}

hipError_t paged_attention(AttnArgs a, int dim, bool fp16, void* workspace, hipStream_t stream) {
  carve(a.p, a.batch, a.kv_heads, dim, (uint8_t*)workspace, &a);
  if (dim == 64) fp16 ? launch_attention<Fp16, 64>(a, stream) : launch_attention<Bf16, 64>(a, stream);
  else if (dim == 128) fp16 ? launch_attention<Fp16, 128>(a, stream) : launch_attention<Bf16, 128>(a, stream);
  else if (dim == 256) fp16 ? launch_attention<Fp16, 256>(a, stream) : launch_attention<Bf16, 256>(a, stream);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace jv
