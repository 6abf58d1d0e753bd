// Attention of new tokens over a paged key/value cache held in 8 bits, for gfx950.
//
//   out[i] = sum_j softmax_j(q_i . k_j * scale) v_j,  k_j = ks[block(j), head] * e4m3 codes, v alike;
//   token i of the n new ones of a sequence of L tokens stands at place L - n + i and sees the keys
//   j <= place (causal), j >= place - window.
//
// The query heads that share a key/value head are rows of one product, so every cache byte is
// read once for all of them.  Codes are widened to bf16 (keys) and half (values) without loss and
// go through the 16-bit matrix instructions; scales never touch the codes:
//   p~_j = exp2(s_j * (ks * scale * log2 e) + log2(vs_j) - m)      one exponential for each score
//   O   += p~_j * codes_j,   l += p~_j / vs_j,   out = O / l
// with m a running reference near the row's maximum of the exponent.  So a value block's scale
// costs one addend in the exponent.  p~ is rounded to half for the second product, the only rounding
// below 32 bits before the output's own: 2^-11 of each weight, where the output's bf16 takes 2^-8.  The
// row sum l takes p~ as it is, in fp32.
//
// Work is cut into items: a tile of rows of one sequence and key/value head against a chunk of
// its keys.  Lengths are known on the device only, so each workgroup adds up the work of all
// sequences, from that takes the length of a chunk with which the items fill one round of
// workgroups, and finds its own item.  Chunks of one row tile are joined by a second kernel; keys
// that are not worth it stay in one piece.
#include <algorithm>
#include <atomic>

#include "common.h"
#include "overlap.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __fp16 hw_f16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef int i32x2 __attribute__((ext_vector_type(2)));

constexpr int KT = 64;               // keys of a tile
// Reference of a row without weight, among those that have some: the lowest number, since a row whose
// scores all lie below -10^30, say, has its weight all the same.
constexpr float M_EMPTY = -3.402823466e38f;
// A row's largest weight lies in [2^ROOM, 2^LAZY] of its reference: half holds up to 2^16, and what it
// cannot hold as a normal number lies 2^22 or more below that weight, off by 2^-33 of it at most.  (With
// the largest weight at 1, a key of 2^25 times the others took all of theirs: 500 of them, behind a first
// key of no value, came out as 0.)  The seven steps between keep the reference from moving often.
constexpr float ROOM = 8.f, LAZY = 15.f;

struct PagedParams {
  const unsigned short* q;
  unsigned short* o;
  float* lse;
  const unsigned char *kc, *vc;
  const float *ks, *vs;
  const int32_t *cu, *lens, *table;
  int64_t q_sb, q_ss, q_sh, o_sb, o_ss, o_sh, lse_sb, lse_sh;
  int64_t kc_sb, kc_sh, vc_sb, vc_sh;
  int kc_st, vc_st;
  int64_t table_stride;
  int B, Hk, G, Sq;  // Sq: rows of q (packed) or of each sequence (cu == nullptr)
  int cap;           // tokens that a row of the table has room for
  int num_blocks, lb, causal, window;
  float scale_log2;
  // items
  int items, chunk_min, split, hw, turns;  // hw: heads of a workgroup, turns: waves of each
  float join_cost;   // of an item, in tiles
  int by_length;     // items longest first
  float slots;       // workgroups of one round, for each group of heads
  float* part;       // [Hk * items][M][D + 2]
  int32_t* info;     // [B][2]: first item of the sequence, chunks of each of its row tiles
};

struct Seq {
  int first, n, len;  // first row of q, new tokens, tokens in all
};
__device__ __forceinline__ Seq seq_of(const PagedParams& p, int b) {
  Seq s;
  s.len = min(max(p.lens[b], 0), p.cap);
  if (p.cu) {
    s.first = min(max(p.cu[b], 0), p.Sq);
    s.n = max(min(p.cu[b + 1], p.Sq) - s.first, 0);
  } else {
    s.first = 0;
    s.n = p.Sq;
  }
  return s;
}
// tiles of keys that any row of the sequence sees: [lo, hi)
__device__ __forceinline__ void seq_tiles(const PagedParams& p, const Seq& s, int& lo, int& hi) {
  const int64_t first = p.window >= 0 ? (int64_t)s.len - s.n - p.window : 0;
  lo = first > 0 ? (int)(first / KT) : 0;
  hi = (s.len + KT - 1) / KT;
  if (hi < lo) hi = lo;
}

// the value of a wave's last lane: of a scan the sum
__device__ __forceinline__ int wave_last(int v) { return __builtin_amdgcn_readlane(v, 63); }

struct Item {
  Seq s;
  int b, tile, chunk, chunks;  // sequence (-1: none), row tile, chunk of keys and how many there are
  int length;                  // tiles of a chunk
};

// Items of whole rows (no chunks) of a few sequences with causal rows, longest first: what is left
// for the last round of workgroups is short then, whatever the sequences' order (prompts of 4096,
// 1115 and 1341 tokens, 32 heads over 8, the first calls after a pause: 215 us, one sequence after the
// other 224).  Row tiles are put in order by the place of their last row, in levels of `unit` tiles of
// keys.  Lanes count the tiles at and above 64 levels at a time: two rounds find the level of the item, a
// walk over the sequences its tile.
constexpr int SORTED_SEQS = 16;
template <int M>
__device__ __forceinline__ void find_longest(const PagedParams& p, int item, Item* found) {
  const int lane = threadIdx.x;
  if (lane == 0) found->b = -1;
  const Seq s = seq_of(p, min(lane, p.B - 1));
  const int base = s.len - s.n, tiles = (s.n * p.G + M - 1) / M;
  // levels there are, at most, in tiles of keys; step <= 33
  const int most = __builtin_amdgcn_readfirstlane((int)group_max<64>((float)(s.len >> 6))) + 2;
  const int unit = (most >> 11) + 1, step = (most / unit + 64) >> 6;
  // tiles of sequence b whose last row is at level x or above: the last tile if x begins before the
  // end, and those from row (x's place - base) G on
  auto upper = [&](int b, int x) {
    const int rb = __builtin_amdgcn_readlane(base, b), rt = __builtin_amdgcn_readlane(tiles, b);
    const unsigned at = (unsigned)x * unit * KT;
    if (x == 0) return rt;
    if (at >= (unsigned)__builtin_amdgcn_readlane(s.len, b)) return 0;
    const int first = (int)at > rb ? ((int)at - rb) * p.G / M : 0;
    return rt - min(max(rt - 1, 0), first);
  };
  auto above = [&](int x) {
    int n = 0;
    for (int b = 0; b < p.B; ++b) n += upper(b, x);
    return n;
  };
  int level = 0;
#pragma unroll 1
  for (int s2 = step; s2; s2 = s2 > 1 ? 1 : 0) {
    const int n = __popcll(__builtin_amdgcn_ballot_w64(above(level + lane * s2) > item));
    if (n == 0) return;  // behind the last item
    level += (n - 1) * s2;
  }
  int k = item - above(level + 1);
  for (int b = 0; b < p.B; ++b) {
    const int from = upper(b, level), n = from - upper(b, level + 1);
    if (k < n) {
      const int rt = __builtin_amdgcn_readlane(tiles, b);
      if (lane == b) *found = Item{s, b, rt - from + k, 0, 1, 1 << 30};
      return;
    }
    k -= n;
  }
}

// The item'th item of a key/value head, for the whole workgroup; false behind the last one.  One
// wave adds up the sequences, `per` that follow each other to a lane, and hands the item on.
template <int M>
__device__ bool find_item(const PagedParams& p, int item, int group, Item* out) {
  __shared__ Item found;
  if (p.by_length) {
    if (threadIdx.x < 64) find_longest<M>(p, item, &found);
  } else if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const int per = (p.B + 63) >> 6;
    const int b0 = lane * per, b1 = min(p.B, b0 + per);
    int length = 1 << 30;  // tiles of the longest chunk
    Seq s{0, 0, 0};
    if (b0 < b1) s = seq_of(p, b0);
    auto tiles_of = [&](const Seq& q) { return (q.n * p.G + M - 1) / M; };
    auto keys_of = [&](const Seq& q) {
      int lo, hi;
      seq_tiles(p, q, lo, hi);
      return hi - lo;
    };
    // (every workgroup adds the same numbers in the same order)
    auto whole = [&](float tiles) {  // chunks are at least chunk_min long, and whole turns of a head's waves
      const int t = (int)fminf(1e9f, fmaxf((float)p.chunk_min, ceilf(tiles)));
      return (t + p.turns - 1) & -p.turns;
    };
    if (p.split && per == 1) {
      const int tiles = b0 < b1 ? tiles_of(s) : 0, keys = b0 < b1 ? keys_of(s) : 0;
      const int64_t mine = (int64_t)tiles * keys;  // below 2^49: summed in halves, lane to lane
      const float work = 0x1p24f * (float)wave_last(wave_scan((int)(mine >> 24))) +
                         (float)wave_last(wave_scan((int)(mine & 0xffffff)));
      const float rows = (float)wave_last(wave_scan(tiles));
      // one round of workgroups, or two where tiles of rows alone take more than 0.6 of one
      const float slots = rows > 0.6f * p.slots ? 2.f * p.slots : p.slots;
      auto items = [&](unsigned l) { return (float)wave_last(wave_scan(tiles * max(1u, (keys + l - 1u) / l))); };
      // between as many chunks as there are slots and as many as fit whatever the last ones' lengths
      float less = work / slots, most = work / fmaxf(slots - rows, 0.125f * slots);
      length = whole(less);
      if (items(length) > slots) {
        for (int i = 0; i < 4; ++i) {
          const float mid = 0.5f * (less + most);
          if (items(whole(mid)) > slots) less = mid;
          else most = mid;
        }
        length = whole(most);
      }
      // What the parts cost is weighed: where the longest keys take no more in one piece than a chunk
      // and the writing and joining of all of them, they stay in one (one prompt of 1000 tokens, 32
      // heads over 8: 38 us, in two pieces 54)
      const float split = slots / p.slots * (float)length + p.join_cost * items(length);
      if (__builtin_amdgcn_ballot_w64((float)keys * fmaxf(1.f, rows / p.slots) > split) == 0) length = 1 << 30;
    } else if (p.split) {
      // (more sequences than lanes: half the tiles of rows are taken off instead, about what the
      // last chunks are short of)
      float work = 0.f, rows = 0.f;
      for (int b = b0; b < b1; ++b) {
        s = seq_of(p, b);
        rows += (float)tiles_of(s);
        work += (float)tiles_of(s) * (float)keys_of(s);
      }
      rows = group_sum<64>(rows);
      length = whole(group_sum<64>(work) / (p.slots - 0.5f * fminf(rows, p.slots)));
    }
    // chunks of a sequence, of one length
    auto chunks_of = [&](const Seq& q, int& l) {
      const unsigned keys = keys_of(q), n = max(1u, (keys + length - 1) / (unsigned)length);
      l = length;
      if (n == 1) return 1;
      l = ((keys + n - 1) / n + p.turns - 1) & -p.turns;
      return (int)((keys + l - 1) / (unsigned)l);
    };
    int mine = 0, chunks = 1, own = length;
    if (per == 1) {
      if (b0 < b1) {
        chunks = chunks_of(s, own);
        mine = tiles_of(s) * chunks;
      }
    } else {
      for (int b = b0; b < b1; ++b) {
        s = seq_of(p, b);
        mine += tiles_of(s) * chunks_of(s, own);
      }
    }
    const int upto = wave_scan(mine);
    if (lane == 0) found.b = -1;
    int at = upto - mine;
    if (item >= at && item < upto) {
      for (int b = b0; b < b1; ++b) {
        if (per > 1) {
          s = seq_of(p, b);
          chunks = chunks_of(s, own);
        }
        const int tiles = tiles_of(s), k = item - at;
        if (k >= 0 && k < (int64_t)tiles * chunks) {
          // causal rows further down see more: they begin first
          found = Item{s, b, tiles - 1 - k / chunks, k % chunks, chunks, own};
          if (p.split && k == 0 && group == 0) {  // for the join
            p.info[2 * b] = item;
            p.info[2 * b + 1] = chunks;
          }
          break;
        }
        at += tiles * chunks;
      }
    }
  }
  __syncthreads();
  *out = found;
  return found.b >= 0;
}

// What a workgroup reads of its item: rows, the tiles of keys and the places its rows stand at.
struct Job {
  Seq s;
  int b, hk, rows, row0;       // rows of the sequence for this head, first one of the tile
  int place_lo, place_hi;      // of the tile's first and last row
  int t0, t1;                  // tiles of keys
};
template <int M>
__device__ __forceinline__ Job job_of(const PagedParams& p, const Item& it, int hk) {
  Job j;
  j.s = it.s;
  j.b = it.b;
  j.hk = hk;
  j.rows = j.s.n * p.G;
  j.row0 = it.tile * M;
  const int base = j.s.len - j.s.n;
  j.place_lo = base + j.row0 / p.G;
  j.place_hi = base + min(j.row0 + M - 1, j.rows - 1) / p.G;
  int lo, hi;
  seq_tiles(p, j.s, lo, hi);
  j.t0 = lo + it.chunk * it.length;
  j.t1 = (int)min((int64_t)hi, (int64_t)j.t0 + it.length);
  if (p.causal) j.t1 = min(j.t1, j.place_hi < 0 ? 0 : j.place_hi / KT + 1);
  if (p.window >= 0 && j.place_lo - p.window > 0) j.t0 = max(j.t0, (j.place_lo - p.window) / KT);
  return j;
}

// A tile is four pieces of 16 keys, each inside one block (blocks hold 16 tokens or more).  Table
// entries are fetched two tiles ahead of the products and scales one, so that neither the entry a
// block's address hangs on nor the scale its scores need is waited for.
// What a wave keeps of the tiles ahead of it, piece l & 3 in lane l: a block (0 where there is
// none), and which of the four pieces there are.  Kept in vector registers and loaded by vector
// loads: scalar loads return out of order, and waiting for one drains the LDS queue with it.
struct Ahead {
  int block;
  unsigned ok;  // bit c: piece c is there
};
__device__ __forceinline__ int load_entry(const PagedParams& p, const Job& j, int t) {
  const int key = min(t * KT + 16 * (int)(threadIdx.x & 3), j.s.len - 1);
  return p.table[j.b * p.table_stride + (key >> p.lb)];
}
__device__ __forceinline__ Ahead resolve(const PagedParams& p, const Job& j, int t, int entry) {
  const bool ok = (int)(t * KT + 16 * (int)(threadIdx.x & 3) < j.s.len) & (int)(entry >= 0) &
                  (int)(entry < p.num_blocks);
  return Ahead{ok ? entry : 0, (unsigned)__builtin_amdgcn_ballot_w64(ok) & 15u};
}
// Where the pieces begin, in bytes behind the head's first: lane c holds piece c's, formed for all
// four at once, and piece_at hands one to the scalar unit.
__device__ __forceinline__ int64_t piece_offsets(const PagedParams& p, const Ahead& a, int t, int64_t sb, int st) {
  const int key = t * KT + 16 * (int)(threadIdx.x & 3);
  const bool ok = (a.ok >> (threadIdx.x & 3)) & 1;
  return a.block * sb + (int64_t)(ok ? key & ((1 << p.lb) - 1) : 0) * st;
}
__device__ __forceinline__ const unsigned char* piece_at(const unsigned char* head, int64_t offsets, int c) {
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)offsets, c);
  const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(offsets >> 32), c);
  return head + (int64_t)(((uint64_t)hi << 32) | lo);
}
// scales of a tile's pieces: factor of the score, addend of the exponent, weight in the row sum
struct Scales {
  float k[4], v_log[4], v_inv[4];
};
__device__ __forceinline__ float lane_value(float x, int c) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), c));
}
__device__ __forceinline__ Scales scales_of(const PagedParams& p, float ks, float vs) {
  vs = fminf(fmaxf(vs, 0x1p-64f), 0x1p120f);
  const float k = ks * p.scale_log2, lg = __builtin_amdgcn_logf(vs), inv = __builtin_amdgcn_rcpf(vs);
  Scales s;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    s.k[c] = lane_value(k, c);
    s.v_log[c] = lane_value(lg, c);
    s.v_inv[c] = lane_value(inv, c);
  }
  return s;
}

// Where a row's reference goes, by the largest exponent of a tile (relative to the reference) and the
// weight that the row has so far: up to ROOM below that exponent, and for a row without weight yet
// (which starts from 0) also down to it.  Rows that see nothing stay.
struct Move {
  float by, shrink;
};
__device__ __forceinline__ Move move_reference(float top, float mass) {
  if (mass == 0.f) return Move{top == -INFINITY ? 0.f : top - ROOM, 0.f};
  const float by = fmaxf(top - ROOM, 0.f);
  return Move{by, __builtin_amdgcn_exp2f(-by)};
}

// Without branches on purpose: a conditional write into one element of a matrix instruction's
// result, with control flow around it, has come out of the compiler with the write missing.
__device__ __forceinline__ bool sees(bool ok, int key, int lo, int hi) {
  return (int)ok & (int)(key >= lo) & (int)(key <= hi);
}

__device__ __forceinline__ bf16x8 widen_bf16(unsigned a, unsigned b) {
  const bf16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, false);
  const bf16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.f, true);
  const bf16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, false);
  const bf16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.f, true);
  return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}
__device__ __forceinline__ f16x8 widen_f16(unsigned a, unsigned b) {
  const f16x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false);
  const f16x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true);
  const f16x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false);
  const f16x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true);
  return f16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}
// A row must not get a NaN from a value that it does not see, and 0 * NaN is NaN: in tiles that
// some row sees in part, NaN codes (0x7f, 0xff) go into the product as zeros, and the rows that do
// see them get theirs afterwards (poison, below), from the cache, where it costs the loop nothing.
__device__ __forceinline__ unsigned nan_codes(unsigned w) {  // 0x80 in each byte that is one
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ unsigned clear_nan(u32x4& v) {
  unsigned any = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const unsigned n = nan_codes(v[j]);
    any |= n;
    v[j] &= ~((n >> 7) * 0xffu);
  }
  return any;
}

// ----------------------------------------------------------------------- few rows: up to sixteen --
// What a decoding step has: it is bound by reading the cache, and built to read it in whole lines,
// early, once.  A wave owns a head and takes tiles of its chunk; the four waves of a workgroup have
// as many neighbouring heads as there are (what they read lies side by side: 4 x 1 token over 128k
// keys in 135 us, 6.1 TB/s of the 6.3 that a plain read of that memory reaches; with the waves side
// by side in the keys of one head 158 us) and take turns at the tiles where heads are fewer; their
// parts are joined through LDS.  Keys and values of the next tile are loaded into registers, past
// the caches, as soon as the current ones are in the wave's images in LDS: keys are read from there
// in rows, values by ds_read_b64_tr_b8, eight keys of one channel to a lane.
//   S^T[key][row] = K . Q^T: a lane holds row l & 15, keys 4 (l >> 4) + i of each piece;
//   O^T[channel][row] += V^T . P^T: the same registers are the second operand, if the k index
//   8 g + j counts keys 4 g + j of the first piece, then of the second one.
template <int D>
__global__ __launch_bounds__(256, D == 64 ? 4 : 2) void paged_few_rows_kernel(PagedParams p) {
  constexpr int M = 16, NH = D / 64, CPR = D / 16, DB = D / 16;
  __shared__ __attribute__((aligned(16))) unsigned char images[4][2 * KT * D];
  __shared__ float wave_m[4][M], wave_l[4][M];
  // eight items side by side, so that all heads of an item are on one of the eight XCDs
  const int groups = p.Hk / p.hw, item = (blockIdx.x / (8 * groups)) * 8 + blockIdx.x % 8;
  const int group = (blockIdx.x / 8) % groups;
  // (the grid is whole eights of items; running sums that are none could find work for the rest)
  if (item >= p.items) return;
  Item it;
  if (!find_item<M>(p, item, group, &it)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // `hw` heads, and `turns` waves for each that take the tiles in turn
  const int hw = p.hw, turns = 4 / hw, in_group = wave % hw, turn = wave / hw;
  const int hk = group * hw + in_group;
  const Job job = job_of<M>(p, it, hk);
  const int r = lane & 15, g = lane >> 4;

  bf16x8 qf[NH][2];
  int see_lo, see_hi;
  const int row = min(job.row0 + r, job.rows - 1), tok = row / p.G, h = row - tok * p.G;
  const unsigned short* qp = p.q + job.b * p.q_sb + (int64_t)(job.s.first + tok) * p.q_ss +
                             (int64_t)(hk * p.G + h) * p.q_sh + 16 * g;
#pragma unroll
  for (int h2 = 0; h2 < NH; ++h2)
#pragma unroll
    for (int u = 0; u < 2; ++u) qf[h2][u] = *reinterpret_cast<const bf16x8*>(qp + 64 * h2 + 8 * u);
  const int place = job.s.len - job.s.n + tok;
  see_hi = min(p.causal ? place : job.s.len - 1, job.s.len - 1);
  see_lo = p.window >= 0 ? place - p.window : 0;

  f32x4 o[DB];
  float m = 0.f, l = 0.f;
#pragma unroll
  for (int d = 0; d < DB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  u32x4 kr[CPR], vr[CPR];
  const unsigned char *k_head = p.kc + hk * p.kc_sh, *v_head = p.vc + hk * p.vc_sh;
  const unsigned k_lane = (unsigned)((lane / CPR) * p.kc_st + (lane % CPR) * 16);
  const unsigned v_lane = (unsigned)((lane / CPR) * p.vc_st + (lane % CPR) * 16);
  // past the caches where a head's row is a whole line; two heads of 64 share one, and the second wave
  // finds it in the cache (8 sequences of 16000, 16 heads of 64: 63 us, past the cache 73)
  auto once = [](const unsigned char* at) {
    if constexpr (D == 64) return *reinterpret_cast<const u32x4*>(at);
    else return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
  };
  auto load_k = [&](const Ahead& a, int t) {
    const int64_t offsets = piece_offsets(p, a, t, p.kc_sb, p.kc_st);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const unsigned char* at = piece_at(k_head, offsets, c);
#pragma unroll
      for (int i = 0; i < CPR / 4; ++i)
        kr[c * CPR / 4 + i] = once(at + (k_lane + (unsigned)(i * (64 / CPR) * p.kc_st)));
    }
  };
  auto load_v = [&](const Ahead& a, int t) {
    const int64_t offsets = piece_offsets(p, a, t, p.vc_sb, p.vc_st);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const unsigned char* at = piece_at(v_head, offsets, c);
#pragma unroll
      for (int i = 0; i < CPR / 4; ++i)  // 64 / CPR rows at a time
        vr[c * CPR / 4 + i] = once(at + (v_lane + (unsigned)(i * (64 / CPR) * p.vc_st)));
    }
  };
  auto swz = [](int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
  unsigned char *img = images[wave], *k_img = img + KT * D;
  const int tr_row = (r >> 1) < 4 ? 4 * g + (r >> 1) : 12 + 4 * g + (r >> 1);
  const int tr_swz = swz(tr_row);
  const unsigned char* tr_at = img + tr_row * D + (r & 1) * 8;
  // does some row of the tile not see some key of it?
  auto in_part = [&](int t, unsigned ok) {
    return t * KT + KT > job.s.len || ok != 15u || (p.causal && t * KT + KT - 1 > job.place_lo) ||
           (p.window >= 0 && t * KT < job.place_hi - p.window);
  };

  bool nan_values = false;
  int t = job.t0 + turn;
  Ahead now{0, 0}, next{0, 0};
  Scales sc{};
  if (t < job.t1) {
    now = resolve(p, job, t, load_entry(p, job, t));
    load_k(now, t);
    load_v(now, t);
    next = resolve(p, job, t + turns, load_entry(p, job, t + turns));
    const int64_t at = (int64_t)now.block * p.Hk + hk;
    sc = scales_of(p, p.ks[at], p.vs[at]);
  }
  // the queries are here before the loop begins: waited for inside it, they would hold up the loads
  // of the next tile with them at every turn
#pragma unroll
  for (int h2 = 0; h2 < NH; ++h2)
#pragma unroll
    for (int u = 0; u < 2; ++u) asm volatile("" : "+v"(qf[h2][u]));
  for (; t < job.t1; t += turns) {
    const bool more = t + turns < job.t1;
    const int key0 = t * KT;
    const bool masked = in_part(t, now.ok);
    // keys and values into the images; what is no key of the sequence as zeros (0 * NaN is NaN)
    if (masked) {
      unsigned any = 0;
#pragma unroll
      for (int i = 0; i < CPR; ++i) {
        const int row = (i * 64 + lane) / CPR;
        if (!((now.ok >> (row >> 4)) & 1) || key0 + row >= job.s.len) vr[i] = u32x4{0, 0, 0, 0};
        any |= clear_nan(vr[i]);
      }
      nan_values |= __builtin_amdgcn_ballot_w64(any != 0) != 0;
    }
#pragma unroll
    for (int i = 0; i < CPR; ++i) {
      const int row = (i * 64 + lane) / CPR;
      *reinterpret_cast<u32x4*>(img + row * D + (((lane % CPR) ^ swz(row)) << 4)) = vr[i];
      *reinterpret_cast<u32x4*>(k_img + row * D + (((lane % CPR) ^ swz(row)) << 4)) = kr[i];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (more) load_k(next, t + turns);
    // entries of the tile after the next, values and scales of the next
    const int entry = load_entry(p, job, t + 2 * turns);
    const int64_t scale_at = (int64_t)next.block * p.Hk + hk;
    const float ks = p.ks[scale_at], vs = p.vs[scale_at];
    if (more) load_v(next, t + turns);

    f32x4 s[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      s[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const u32x4 kk = *reinterpret_cast<const u32x4*>(k_img + (16 * c + r) * D + (((4 * h + g) ^ swz(16 * c + r)) << 4));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bf16x8 kf = widen_bf16(kk[2 * u], kk[2 * u + 1]);
          s[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[h][u], s[c], 0, 0, 0);
        }
      }
    }

    f16x8 pf[2];
    // exponents against the reference as it stands; it moves (move_reference), and O and l with
    // it, only where one of them is too large for a half, or a row has had no weight yet
    float x[4][4], sum[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float add = sc.v_log[c] - m;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[c][i] = fmaf(s[c][i], sc.k[c], add);
    }
    if (masked) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[c][i] = sees((now.ok >> c) & 1, key0 + 16 * c + 4 * g + i, see_lo, see_hi) ? x[c][i] : -INFINITY;
    }
    float top = x[0][0];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, x[c][i]);
    if (__builtin_amdgcn_ballot_w64(top > LAZY || l == 0.f) != 0) {
      float mass = l;
#pragma unroll
      for (int w = 16; w < 64; w <<= 1) {
        top = fmaxf(top, __shfl_xor(top, w, 64));
        mass += __shfl_xor(mass, w, 64);
      }
      const Move mv = move_reference(top, mass);
      m += mv.by;
      l *= mv.shrink;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[d] *= mv.shrink;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c][i] -= mv.by;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[c][i] = __builtin_amdgcn_exp2f(x[c][i]);
      sum[c] = (x[c][0] + x[c][1]) + (x[c][2] + x[c][3]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) l = fmaf(sum[c], sc.v_inv[c], l);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) pf[c >> 1][4 * (c & 1) + i] = (_Float16)x[c][i];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(tr_at + st * 32 * D + ((d ^ tr_swz) << 4)));
        const f16x8 vf = widen_f16((unsigned)w[0], (unsigned)w[1]);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[st], o[d], 0, 0, 0);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (!more) break;  // (so that whatever was loaded has been used before the next turn)
    now = next;
    next = resolve(p, job, t + 2 * turns, entry);
    sc = scales_of(p, ks, vs);
  }
  if (nan_values) {  // poison: the NaN among the values of tiles seen in part, for the rows that see them
    for (t = job.t0 + turn; t < job.t1; t += turns) {
      now = resolve(p, job, t, load_entry(p, job, t));
      if (!in_part(t, now.ok)) continue;
      const int64_t offsets = piece_offsets(p, now, t, p.vc_sb, p.vc_st);
      for (int k = 0; k < KT; ++k) {
        const int key = t * KT + k;
        if (!((now.ok >> (k >> 4)) & 1) || key >= job.s.len) continue;
        const unsigned char* at = piece_at(v_head, offsets, k >> 4) + (k & 15) * p.vc_st;
        const unsigned seen = (unsigned)sees(true, key, see_lo, see_hi);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const unsigned n = nan_codes(*reinterpret_cast<const unsigned*>(at + 16 * d + 4 * g));
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] = ((n >> (8 * i + 7)) & seen) ? __builtin_nanf("") : o[d][i];
        }
      }
    }
  }

  // ---- the parts of each row that the waves of a head hold, joined ----
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (l == 0.f) m = M_EMPTY;
  if (g == 0) {
    wave_m[wave][r] = m;
    wave_l[wave][r] = l;
  }
  float* part = nullptr;
  if (it.chunks > 1) part = p.part + ((int64_t)hk * p.items + item) * (M * (D + 2));
  __syncthreads();
  float top = M_EMPTY;
  for (int w = in_group; w < 4; w += hw) top = fmaxf(top, wave_m[w][r]);
  const float weight = __builtin_amdgcn_exp2f(m - top);
  // [16 rows][D] fp32 in the wave's image (64 D bytes), 16-byte pieces turned by the row
  float* mine = reinterpret_cast<float*>(images[wave]);
#pragma unroll
  for (int d = 0; d < DB; ++d)
    *reinterpret_cast<f32x4*>(mine + r * D + (((4 * d + g) ^ (r & 7)) << 2)) = o[d] * weight;
  __syncthreads();
  // four channels of a row for each thread of the head
  for (int i = turn * 64 + lane; i < 16 * D / 4; i += turns * 64) {
    const int row = i / (D / 4), c4 = i % (D / 4), at = row * D + ((c4 ^ (row & 7)) << 2);
    const int q_row = job.row0 + row;
    if (q_row >= job.rows) continue;
    float rm = M_EMPTY, rl = 0.f;
    for (int w = in_group; w < 4; w += hw) rm = fmaxf(rm, wave_m[w][row]);
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = in_group; w < 4; w += hw) {
      sum = sum + *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(images[w]) + at);
      rl = fmaf(wave_l[w][row], __builtin_amdgcn_exp2f(wave_m[w][row] - rm), rl);
    }
    if (part) {
      *reinterpret_cast<f32x4*>(part + row * D + 4 * c4) = sum;
      if (c4 == 0) {
        part[M * D + 2 * row] = rm;
        part[M * D + 2 * row + 1] = rl;
      }
      continue;
    }
    const int tok = q_row / p.G, head = hk * p.G + q_row - tok * p.G;
    const float inv = rl == 0.f ? 0.f : 1.f / rl;
    *reinterpret_cast<u32x2*>(p.o + job.b * p.o_sb + (int64_t)(job.s.first + tok) * p.o_ss + head * p.o_sh +
                              4 * c4) = u32x2{pack_bf2(sum[0] * inv, sum[1] * inv), pack_bf2(sum[2] * inv, sum[3] * inv)};
    if (p.lse && c4 == 0)
      p.lse[job.b * p.lse_sb + head * p.lse_sh + job.s.first + tok] =
          rl == 0.f ? -INFINITY : (rm + __builtin_amdgcn_logf(rl)) * 0.6931471805599453f;
  }
}

// --------------------------------------------------------------------------------- many rows --
// 32 rows for each of four waves, which share the tiles of keys in LDS, widened to 16 bits once
// for all of them while they are stored there: half the waves load keys, half values, to registers a
// tile ahead, and convert; two stages, one barrier for each tile.  Products and layouts are those of
// the dense kernel (attention.hip): S^T = K . Q^T with 32x32x16 instructions, the row on the lane;
// P^T is the second operand of O^T += V^T . P^T as it stands; values through the transposing LDS
// read.
// Up to 64 rows (HALVES = 2) two waves share 32 rows, each with half of a tile's keys, since a wave's
// chain of products, exponentials and products is what a tile then takes: 32 rows over 60 thousand
// keys 104 us, with two waves idle 116; 64 rows 120 and 143.
// Prompts of 4096, 1115 and 1341 tokens, 32 heads over 8: 188 us = 0.86 PF/s at the clock that a few dozen
// calls in a row settle to (the first ones after a pause take 217-226, with a profiler or without), 201
// with other inputs for each call.  A large bf16 library product reaches 1.19 PF/s, this repository's dense
// kernel 1.17 at 4096 tokens, 0.83 at 1536.  By counters matrix instructions are busy 0.39 of the time
// (dense: 0.63) and the vector unit (32 exponentials a lane and tile, and the widening) 0.54 (0.48); the
// two hardly overlap, neither across waves nor when the second half's exponentials are put between the
// first half's products (223 us where this order took 211, after a pause).  256 rows with eight waves
// halve the widening and take as long.
template <int D, int NW, int HALVES>
__global__ __launch_bounds__(NW * 64, 8 / NW) void paged_many_rows_kernel(PagedParams p) {
  constexpr int RANKS = NW / HALVES, M = 32 * RANKS, KB = 2 / HALVES, ROWB = 2 * D, CPR = ROWB / 16, KSTEPS = D / 16, DVB = D / 32;
  constexpr int TILE = KT * ROWB, LOADS = KT * D / 16 / (NW * 32);
  static_assert(LOADS >= 1, "every thread loads");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ int nan_values;
  const int item = blockIdx.x / p.Hk, hk = blockIdx.x % p.Hk;
  Item it;
  if (!find_item<M>(p, item, hk, &it)) return;
  const Job job = job_of<M>(p, it, hk);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const int rank = wave % RANKS, half = wave / RANKS;  // rows, and keys of each tile, of the wave
  auto k_swz = [](int key) { return key & 15 & (CPR - 1); };
  auto v_swz = [](int key) { return (((key & 3) << 2) | ((key >> 2) & 3)) & (CPR - 1); };

  const int row = min(job.row0 + 32 * rank + r, job.rows - 1), tok = row / p.G, head = hk * p.G + row - tok * p.G;
  const int base = job.s.len - job.s.n, place = base + tok;
  const int see_hi = min(p.causal ? place : job.s.len - 1, job.s.len - 1);
  const int see_lo = p.window >= 0 ? place - p.window : 0;
  // places of the wave's first and last row
  const int wave_row = min(job.row0 + 32 * rank, job.rows - 1);
  const int w_lo = base + wave_row / p.G, w_hi = base + min(wave_row + 31, job.rows - 1) / p.G;
  bf16x8 qf[KSTEPS];
  {
    const unsigned short* qp = p.q + job.b * p.q_sb + (int64_t)(job.s.first + tok) * p.q_ss + (int64_t)head * p.q_sh;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s + 8 * hh);
  }

  // One half of the waves stages keys, the other values: 16 bytes of a key (or value) for each
  // thread and load, all of a wave in one piece.
  const bool loads_v = wave >= NW / 2;
  const unsigned char* head_at = loads_v ? p.vc + hk * p.vc_sh : p.kc + hk * p.kc_sh;
  const int64_t my_sb = loads_v ? p.vc_sb : p.kc_sb;
  const int my_st = loads_v ? p.vc_st : p.kc_st;
  const int my_c = tid % (D / 16), my_key = (tid % (NW * 32)) / (D / 16);
  constexpr int KEYS = NW * 32 * 16 / D;  // keys of one load of all these threads
  u32x4 raw[LOADS];
  auto load = [&](const Ahead& a, int t) {
    const int64_t offsets = piece_offsets(p, a, t, my_sb, my_st);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int key = i * KEYS + my_key, c = __builtin_amdgcn_readfirstlane(key >> 4);
      raw[i] = *reinterpret_cast<const u32x4*>(piece_at(head_at, offsets, c) + (unsigned)((key & 15) * my_st + 16 * my_c));
    }
  };
  // does some row of the workgroup not see some key of the tile?
  auto in_part = [&](int t, unsigned ok) {
    return t * KT + KT > job.s.len || ok != 15u || (p.causal && t * KT + KT - 1 > job.place_lo) ||
           (p.window >= 0 && t * KT < job.place_hi - p.window);
  };
  auto store = [&](const Ahead& a, int t, int buf) {
    if (!loads_v) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int key = i * KEYS + my_key;
        unsigned char* to = smem + buf * 2 * TILE + key * ROWB;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<bf16x8*>(to + (((2 * my_c + h) ^ k_swz(key)) << 4)) = widen_bf16(raw[i][2 * h], raw[i][2 * h + 1]);
      }
      return;
    }
    if (in_part(t, a.ok)) {
      unsigned any = 0;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int key = i * KEYS + my_key;
        if (!((a.ok >> (key >> 4)) & 1) || t * KT + key >= job.s.len) raw[i] = u32x4{0, 0, 0, 0};
        any |= clear_nan(raw[i]);
      }
      if (any) nan_values = 1;
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int key = i * KEYS + my_key;
      unsigned char* to = smem + buf * 2 * TILE + TILE + key * ROWB;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f16x8*>(to + (((2 * my_c + h) ^ v_swz(key)) << 4)) = widen_f16(raw[i][2 * h], raw[i][2 * h + 1]);
    }
  };

  int koff[KSTEPS];
#pragma unroll
  for (int s = 0; s < KSTEPS; ++s) koff[s] = r * ROWB + (((2 * s + hh) ^ k_swz(r)) << 4);
  const int li = lane & 15, qq = li >> 2, pp = li & 3, g2 = (lane >> 4) & 1;
  int vlane[DVB][2];
#pragma unroll
  for (int d = 0; d < DVB; ++d)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key = half * 8 + 4 * hh + qq, col = d * 32 + g2 * 16 + 4 * pp;
      vlane[d][half] = key * ROWB + (((col >> 3) ^ v_swz(key)) << 4) + ((col & 7) << 1);
    }

  f32x16 o[DVB];
#pragma unroll
  for (int d = 0; d < DVB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = 0.f, l = 0.f;

  if (tid == 0) nan_values = 0;
  __syncthreads();
  Ahead now{0, 0}, next{0, 0};
  Scales sc{};
  if (job.t0 < job.t1) {
    now = resolve(p, job, job.t0, load_entry(p, job, job.t0));
    load(now, job.t0);
    next = resolve(p, job, job.t0 + 1, load_entry(p, job, job.t0 + 1));
    const int64_t at = (int64_t)now.block * p.Hk + hk;
    sc = scales_of(p, p.ks[at], p.vs[at]);
    store(now, job.t0, 0);
  }
  const bool live_wave = job.row0 + 32 * rank < job.rows;
  // the queries are here before the loop begins: waited for inside it, they would hold up the loads
  // of the next tile with them at every turn
#pragma unroll
  for (int s = 0; s < KSTEPS; ++s) asm volatile("" : "+v"(qf[s]));
  for (int t = job.t0, buf = 0; t < job.t1; ++t, buf ^= 1) {
    const int key0 = t * KT;
    __syncthreads();
    const bool more = t + 1 < job.t1;
    // entries of the tile after the next, keys, values and scales of the next
    const int entry = load_entry(p, job, t + 2);
    const int64_t scale_at = (int64_t)next.block * p.Hk + hk;
    const float ks = p.ks[scale_at], vs = p.vs[scale_at];
    if (more) load(next, t + 1);
    if (live_wave && !(p.causal && key0 > w_hi) && !(p.window >= 0 && key0 + KT - 1 < w_lo - p.window)) {
      const unsigned char *kt = smem + buf * 2 * TILE + half * 32 * ROWB, *vt = kt + TILE;
      const int key1 = key0 + 32 * half;
      f32x16 s[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
      bf16x8 kf[2][KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) kf[0][kb] = *reinterpret_cast<const bf16x8*>(kt + kb * 32 * ROWB + koff[0]);
#pragma unroll
      for (int st = 0; st < KSTEPS; ++st) {
        if (st + 1 < KSTEPS) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
            kf[(st + 1) & 1][kb] = *reinterpret_cast<const bf16x8*>(kt + kb * 32 * ROWB + koff[st + 1]);
        }
        __builtin_amdgcn_sched_barrier(0);  // the reads of a step stay ahead of the products before it
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[st & 1][kb], qf[st], s[kb], 0, 0, 0);
      }
      const bool masked = key0 + KT > job.s.len || now.ok != 15u || (p.causal && key0 + KT - 1 > w_lo) ||
                          (p.window >= 0 && key0 < w_hi - p.window);
      // as in the kernel above: x[c][e] is element e of piece c
      float x[2 * KB][8], sum[2 * KB];
      auto mine = [&](const float (&v)[4], int c) { return HALVES == 2 && half ? v[2 + c % 2] : v[c]; };
#pragma unroll
      for (int c = 0; c < 2 * KB; ++c) {
        const float add = mine(sc.v_log, c) - m, scale = mine(sc.k, c);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[c][e] = fmaf(s[c >> 1][8 * (c & 1) + e], scale, add);
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            x[c][e] = sees((now.ok >> (2 * half + c)) & 1, key1 + 16 * c + (e & 3) + 8 * (e >> 2) + 4 * hh, see_lo, see_hi)
                          ? x[c][e] : -INFINITY;
      }
      float top = x[0][0];
#pragma unroll
      for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, x[c][e]);
      if (__builtin_amdgcn_ballot_w64(top > LAZY || l == 0.f) != 0) {
        const Move mv = move_reference(fmaxf(top, __shfl_xor(top, 32, 64)), l + __shfl_xor(l, 32, 64));
        m += mv.by;
        l *= mv.shrink;
#pragma unroll
        for (int d = 0; d < DVB; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] *= mv.shrink;
#pragma unroll
        for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[c][e] -= mv.by;
      }
#pragma unroll
      for (int c = 0; c < 2 * KB; ++c) {
        sum[c] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[c][e] = __builtin_amdgcn_exp2f(x[c][e]);
          sum[c] += x[c][e];
        }
      }
#pragma unroll
      for (int c = 0; c < 2 * KB; ++c) l = fmaf(sum[c], mine(sc.v_inv, c), l);
      f16x8 pf[KB][2];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int j = 0; j < 8; ++j) pf[kb][st][j] = (_Float16)x[2 * kb + st][j];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int d = 0; d < DVB; ++d) {
            const unsigned char* at = vt + (kb * 32 + st * 16) * ROWB;
            const f16x4 a = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                (__attribute__((address_space(3))) hw_f16x4*)(at + vlane[d][0])));
            const f16x4 b = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                (__attribute__((address_space(3))) hw_f16x4*)(at + vlane[d][1])));
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7),
                                                          pf[kb][st], o[d], 0, 0, 0);
          }
    }
    if (!more) break;  // (so that whatever was loaded has been used before the next turn)
    store(next, t + 1, buf ^ 1);
    now = next;
    next = resolve(p, job, t + 2, entry);
    sc = scales_of(p, ks, vs);
  }
  __syncthreads();
  if (nan_values) {  // poison, as above
    for (int t = job.t0; t < job.t1; ++t) {
      now = resolve(p, job, t, load_entry(p, job, t));
      if (!in_part(t, now.ok)) continue;
      const int64_t offsets = piece_offsets(p, now, t, p.vc_sb, p.vc_st);
      for (int k = 0; k < KT; ++k) {
        const int key = t * KT + k;
        if (!((now.ok >> (k >> 4)) & 1) || key >= job.s.len) continue;
        const unsigned char* at = piece_at(p.vc + hk * p.vc_sh, offsets, k >> 4) + (k & 15) * p.vc_st + 4 * hh;
        const unsigned seen = (unsigned)sees(true, key, see_lo, see_hi);
#pragma unroll
        for (int d = 0; d < DVB; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const unsigned n = nan_codes(*reinterpret_cast<const unsigned*>(at + 32 * d + 8 * g));
#pragma unroll
            for (int i = 0; i < 4; ++i) o[d][4 * g + i] = ((n >> (8 * i + 7)) & seen) ? __builtin_nanf("") : o[d][4 * g + i];
          }
      }
    }
  }

  l += __shfl_xor(l, 32, 64);
  if constexpr (HALVES == 2) {
    // the two waves of each row, through LDS as they lie in the lanes
    float* at = reinterpret_cast<float*>(smem) + rank * (DVB * 16 + 2) * 64 + lane;
    if (l == 0.f) m = M_EMPTY;
    __syncthreads();
    if (half) {
#pragma unroll
      for (int d = 0; d < DVB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) at[(16 * d + e) * 64] = o[d][e];
      at[16 * DVB * 64] = m;
      at[(16 * DVB + 1) * 64] = l;
    }
    __syncthreads();
    if (half) return;
    const float m1 = at[16 * DVB * 64], l1 = at[(16 * DVB + 1) * 64], top = fmaxf(m, m1);
    const float w0 = __builtin_amdgcn_exp2f(m - top), w1 = __builtin_amdgcn_exp2f(m1 - top);
#pragma unroll
    for (int d = 0; d < DVB; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[d][e] = fmaf(o[d][e], w0, at[(16 * d + e) * 64] * w1);
    l = fmaf(l, w0, l1 * w1);
    m = top;
  }
  const int in_tile = 32 * rank + r;
  if (it.chunks > 1) {
    float* part = p.part + ((int64_t)hk * p.items + item) * (M * (D + 2));
#pragma unroll
    for (int d = 0; d < DVB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(part + in_tile * D + d * 32 + 8 * g + 4 * hh) =
            f32x4{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (hh == 0) {
      part[M * D + 2 * in_tile] = l == 0.f ? M_EMPTY : m;
      part[M * D + 2 * in_tile + 1] = l;
    }
    return;
  }
  const bool live = job.row0 + in_tile < job.rows;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (p.lse && live && hh == 0)
    p.lse[job.b * p.lse_sb + head * p.lse_sh + job.s.first + tok] =
        l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
  unsigned short* op = p.o + job.b * p.o_sb + (int64_t)(job.s.first + tok) * p.o_ss + head * p.o_sh;
#pragma unroll
  for (int d = 0; d < DVB; ++d) {
    unsigned pk[4][2];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      pk[g][0] = pack_bf2(o[d][4 * g] * inv, o[d][4 * g + 1] * inv);
      pk[g][1] = pack_bf2(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv);
    }
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        auto sw = __builtin_amdgcn_permlane32_swap(pk[g][w], pk[g + 1][w], false, false);
        pk[g][w] = sw[0];
        pk[g + 1][w] = sw[1];
      }
      if (live)
        *reinterpret_cast<u32x4*>(op + d * 32 + 8 * (g + hh)) = u32x4{pk[g][0], pk[g][1], pk[g + 1][0], pk[g + 1][1]};
    }
  }
}

// ------------------------------------------------------------------------------------- joint --
// Parts are weighed by 2^(their reference - the row's largest), also where that is 0: a part's NaN is the
// row's, as it would be in one piece.  Parts that see nothing hold zeros.
// The sequence and token of row t of q, for a whole wave; false where there is nothing to join: a
// row behind the last sequence, or one whose keys were not split.
struct JoinRow {
  int b, tok, base, chunks, tiles;
};
__device__ __forceinline__ bool join_row(const PagedParams& p, int M, int64_t t, JoinRow* j) {
  const int lane = threadIdx.x & 63;
  if (p.cu) {  // the sequence whose rows t is among: those that end at or before t come before it
    j->b = 0;
    for (int i0 = 0; i0 < p.B; i0 += 64) {
      const int i = i0 + lane;
      const unsigned long long before = __builtin_amdgcn_ballot_w64(i < p.B && p.cu[min(i, p.B - 1) + 1] <= (int)t);
      j->b += __popcll(before);
      if (before != ~0ull) break;
    }
    if (j->b >= p.B) return false;  // a row behind the last sequence
    j->tok = (int)t - seq_of(p, j->b).first;
  } else {
    j->b = (int)(t / p.Sq);
    j->tok = (int)(t - (int64_t)j->b * p.Sq);
  }
  const int n = seq_of(p, j->b).n;
  j->base = p.info[2 * j->b];
  j->chunks = p.info[2 * j->b + 1];
  j->tiles = (n * p.G + M - 1) / M;
  // one chunk: written by the kernel itself.  (Running sums that are none would leave this unset.)
  return j->tok >= 0 && j->tok < n && j->chunks > 1 && j->base >= 0 &&
         j->base + (int64_t)j->tiles * j->chunks <= p.items;
}
__device__ __forceinline__ const float* parts_of(const PagedParams& p, int M, int64_t step, const JoinRow& j, int hk, int row) {
  return p.part + ((int64_t)hk * p.items + j.base + (int64_t)(j.tiles - 1 - row / M) * j.chunks) * step;
}

// Few rows of q: four waves for each.  Lane c weighs chunk c; the sums run over a few chunks at a
// time, so that their loads are in flight together.  Bound by three loads that hang on each other
// and by the launch: 4 us for 32 rows, 5 for 1024.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p, int M) {
  __shared__ f32x4 others[3][D / 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int H = p.Hk * p.G;
  const int64_t t = blockIdx.x / H;
  const int head = (int)(blockIdx.x - t * H);
  JoinRow j;
  if (!join_row(p, M, t, &j)) return;
  const int hk = head / p.G, row = j.tok * p.G + head - hk * p.G;
  const int chunks = j.chunks, in_tile = row % M;
  const int64_t step = (int64_t)M * (D + 2);
  const float* part = parts_of(p, M, step, j, hk, row);
  float top = M_EMPTY;
  for (int c = lane; c < chunks; c += 64) top = fmaxf(top, part[c * step + M * D + 2 * in_tile]);
  top = group_max<64>(top);
  // lanes hold four channels; 256 / D chunks side by side
  constexpr int SIDE = 256 / D, LANES = D / 4;
  const int mine = lane / LANES, ch = lane % LANES;
  f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    const int c = min(c0 + lane, chunks - 1);
    const float* ml = part + c * step + M * D + 2 * in_tile;
    const float w = c0 + lane < chunks ? __builtin_amdgcn_exp2f(ml[0] - top) : 0.f;
    l = c0 + lane < chunks ? fmaf(ml[1], w, l) : l;
    const int here = min(64, chunks - c0);
    for (int k = wave * 4 * SIDE; k < here; k += 16 * SIDE) {
      f32x4 v[4];
      float wv[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int at = k + u * SIDE + mine;
        wv[u] = __shfl(w, min(at, 63), 64);
        v[u] = *reinterpret_cast<const f32x4*>(part + min(c0 + at, chunks - 1) * step + in_tile * D + 4 * ch);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = k + u * SIDE + mine < here ? fmaf(v[u][i], wv[u], acc[i]) : acc[i];
    }
  }
  l = group_sum<64>(l);
#pragma unroll
  for (int w = LANES; w < 64; w <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], w, 64);
  if (wave && mine == 0) others[wave - 1][ch] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) acc = acc + others[w][ch];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t q_row = p.cu ? t : j.tok;
  if (mine == 0)
    *reinterpret_cast<u32x2*>(p.o + j.b * p.o_sb + q_row * p.o_ss + head * p.o_sh + 4 * ch) =
        u32x2{pack_bf2(acc[0] * inv, acc[1] * inv), pack_bf2(acc[2] * inv, acc[3] * inv)};
  if (p.lse && lane == 0)
    p.lse[j.b * p.lse_sb + head * p.lse_sh + q_row] =
        l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// Many rows: a wave for four heads of a token, sixteen lanes for each, all chunks in one pass with
// a running maximum, four of them in flight (19200 rows of 3 chunks, 30 MB: 8.8 us, with a wave for
// each row 16).
template <int D>
__global__ __launch_bounds__(256) void paged_join_rows_kernel(PagedParams p, int M, int64_t waves, int head_groups) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = (int64_t)blockIdx.x * 4 + wave;
  if (id >= waves) return;
  const int64_t t = id / head_groups;
  JoinRow j;
  if (!join_row(p, M, t, &j)) return;
  const int H = p.Hk * p.G, ch = lane & 15;
  const int mine = (int)(id - t * head_groups) * 4 + (lane >> 4), head = min(mine, H - 1);
  const int hk = head / p.G, row = j.tok * p.G + head - hk * p.G;
  const int chunks = j.chunks, in_tile = row % M;
  const int64_t step = (int64_t)M * (D + 2);
  const float* part = parts_of(p, M, step, j, hk, row);
  constexpr int NV = D / 64;  // lanes hold channels 4 (ch + 16 n) and on
  f32x4 acc[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float top = M_EMPTY, l = 0.f;
  for (int c0 = 0; c0 < chunks; c0 += 4) {
    float m[4], lc[4];
    f32x4 v[4][NV];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* at = part + min(c0 + u, chunks - 1) * step;
      m[u] = at[M * D + 2 * in_tile];
      lc[u] = at[M * D + 2 * in_tile + 1];
#pragma unroll
      for (int n = 0; n < NV; ++n) v[u][n] = *reinterpret_cast<const f32x4*>(at + in_tile * D + 4 * (ch + 16 * n));
    }
    const float was = top;
#pragma unroll
    for (int u = 0; u < 4; ++u) top = fmaxf(top, m[u]);
    const float shrink = __builtin_amdgcn_exp2f(was - top);
    l *= shrink;
#pragma unroll
    for (int n = 0; n < NV; ++n) acc[n] *= shrink;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool there = c0 + u < chunks;
      const float w = __builtin_amdgcn_exp2f(m[u] - top);
      l = there ? fmaf(lc[u], w, l) : l;
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = there ? fmaf(v[u][n][i], w, acc[n][i]) : acc[n][i];
    }
  }
  if (mine >= H) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t q_row = p.cu ? t : j.tok;
  unsigned short* out = p.o + j.b * p.o_sb + q_row * p.o_ss + head * p.o_sh;
#pragma unroll
  for (int n = 0; n < NV; ++n)
    *reinterpret_cast<u32x2*>(out + 4 * (ch + 16 * n)) =
        u32x2{pack_bf2(acc[n][0] * inv, acc[n][1] * inv), pack_bf2(acc[n][2] * inv, acc[n][3] * inv)};
  if (p.lse && ch == 0)
    p.lse[j.b * p.lse_sb + head * p.lse_sh + q_row] =
        l == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// -------------------------------------------------------------------------------------- host --
int cu_count() {
  static std::atomic<int> cus{0};
  int n = cus.load(std::memory_order_relaxed);
  if (n == 0) {
    int d = 0;
    (void)hipGetDevice(&d);
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, d) != hipSuccess || n <= 0) n = 256;
    cus.store(n, std::memory_order_relaxed);
  }
  return n;
}

struct Plan {
  int M, few, hw;      // rows of a tile; which kernel; heads of a workgroup
  int64_t items, slots;
  int chunk_min, split;
  int64_t part_bytes, info_bytes;
};

// Which kernel, how many items at most, and whether keys may be split.
Plan plan_of(const mi355_paged_attn_args* a) {
  Plan w;
  const int64_t G = a->H / a->Hk, rows = a->max_seqlen_q * G;
  const int64_t all_rows = (a->cu_seqlens_q ? a->Sq : a->Sq * a->B) * G;
  // three kinds of row tiles: 16, 64 with two waves for each row, 128 (two tiles of sixteen rows in the
  // first kernel gain nothing: 32 rows over 8 to 60 thousand keys take 33 and 116 us there, 21 and
  // 104 us with a tile of 64)
  w.few = rows <= 16;
  w.M = w.few ? 16 : rows <= 64 ? 64 : 128;
  // as many heads to a workgroup as share its four waves: what they read lies side by side
  w.hw = !w.few ? 1 : a->Hk % 4 == 0 ? 4 : a->Hk % 2 == 0 ? 2 : 1;
  const int64_t tiles = all_rows / w.M + a->B;  // row tiles: at most one not full for each sequence
  // Workgroups of one round: two a CU (many rows with heads of 64: three; 509 tokens behind 30k keys
  // 105 us, with two 115 us).  What is over one round waits for it: with few rows two rounds of half
  // the length take 50 us where one takes 44 (32 x 1 token, ragged).
  const int64_t want = (w.few ? 2 : a->D == 64 ? 3 : 2) * (int64_t)cu_count();
  const int64_t groups = a->Hk / w.hw;
  w.slots = (want + groups - 1) / groups;
  w.chunk_min = w.few ? (w.hw == 4 ? 1 : 4) : 4;
  // keys that a sequence's rows see, at most (were max_seqlen_q too small, more would be read in one piece)
  const int64_t room = a->table_width * a->block_size;
  const int64_t cap = a->window_left < 0 || a->window_left >= room
                          ? room : std::min(room, a->window_left + a->max_seqlen_q + KT);
  // (below that a piece costs less than the join's launch: 1 token over 100 keys 9.5 us, split 13; one
  // prompt of 500 tokens 19 us, split 30)
  w.split = cap > (w.few ? 4 * (4 / w.hw) : 8) * KT && (all_rows / w.M) * groups < 2 * want;
  // (find_item makes no more: with one lane for a sequence the chunks fit one or two rounds, else
  // there is at most one more than the work takes for each tile of rows)
  const int64_t chunks = a->B > 64 ? tiles + w.slots
                         : 5 * tiles <= 3 * w.slots ? w.slots : std::max(2 * w.slots, tiles + w.slots / 4);
  w.items = w.split ? chunks : tiles;
  w.part_bytes = w.split ? a->Hk * w.items * w.M * (a->D + 2) * (int64_t)sizeof(float) : 0;
  w.info_bytes = w.split ? a->B * 2 * (int64_t)sizeof(int32_t) : 0;
  return w;
}

int check(const mi355_paged_attn_args* a) {
  MI355_REQUIRE(a != nullptr, "paged_attn_fp8: null args");
  MI355_REQUIRE(a->D == 64 || a->D == 128, "paged_attn_fp8: head size %ld not in {64,128}", (long)a->D);
  MI355_REQUIRE(a->B >= 0 && a->B < (1 << 24) && a->Sq >= 0 && a->Sq < (1ll << 31) && a->H > 0 && a->H < 65536 &&
                    a->Hk > 0 && a->H % a->Hk == 0 && a->max_seqlen_q >= 0 && a->max_seqlen_q < (1ll << 31),
                "paged_attn_fp8: bad shape B=%ld Sq=%ld H=%ld Hk=%ld", (long)a->B, (long)a->Sq, (long)a->H,
                (long)a->Hk);
  const int64_t tokens = a->cu_seqlens_q ? a->Sq : a->Sq * a->B;
  MI355_REQUIRE(tokens < (1ll << 31) && tokens * (a->H / a->Hk) < (1ll << 31), "paged_attn_fp8: too many rows");
  MI355_REQUIRE(a->block_size >= 16 && a->block_size <= 1024 && (a->block_size & (a->block_size - 1)) == 0,
                "paged_attn_fp8: block size %ld must be a power of two in [16, 1024]", (long)a->block_size);
  MI355_REQUIRE(a->num_blocks >= 0 && a->num_blocks < (1ll << 31) && a->table_width >= 0 &&
                    a->table_width * a->block_size <= (1ll << 31) - 4096 && a->table_stride >= 0,
                "paged_attn_fp8: bad page table");
  MI355_REQUIRE(a->window_left < 0 || a->causal, "paged_attn_fp8: a window needs causal masking");
  return MI355_OK;
}

template <int D, int HALVES>
int launch_many(const PagedParams& p, dim3 grid, hipStream_t st) {
  constexpr int LDS = 4 * KT * D * 2;  // two stages of keys and values
  // the limit of dynamic LDS is an attribute of the function on each device
  static std::atomic<unsigned long long> known{0};
  int dev = 0;
  (void)hipGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(known.load(std::memory_order_acquire) & bit)) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(paged_many_rows_kernel<D, 4, HALVES>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) {
      mi355_set_error("paged_attn_fp8: cannot reserve %d B of LDS: %s", LDS, hipGetErrorString(e));
      return MI355_EHIP;
    }
    known.fetch_or(bit, std::memory_order_release);
  }
  hipLaunchKernelGGL((paged_many_rows_kernel<D, 4, HALVES>), grid, dim3(256), LDS, st, p);
  return MI355_OK;
}

template <int D>
int launch(const PagedParams& p, const Plan& w, hipStream_t st) {
  const dim3 grid((unsigned)(w.few ? (w.items + 7) / 8 * 8 * (p.Hk / w.hw) : w.items * p.Hk));
  if (w.few) {
    hipLaunchKernelGGL(paged_few_rows_kernel<D>, grid, dim3(256), 0, st, p);
  } else {
    if (int rc = w.M == 64 ? launch_many<D, 2>(p, grid, st) : launch_many<D, 1>(p, grid, st)) return rc;
  }
  MI355_CHECK_LAUNCH("paged_attn_fp8");
  if (w.split) {
    const int64_t tokens = (int64_t)p.Sq * (p.cu ? 1 : p.B), heads = p.Hk * p.G, head_groups = (heads + 3) / 4;
    // four waves for a row while there are few rows (4 x 1 token over 128k keys: 6.3 us, with one 9)
    if (tokens * heads <= 2048)
      hipLaunchKernelGGL(paged_join_kernel<D>, dim3((unsigned)(tokens * heads)), dim3(256), 0, st, p, w.M);
    else
      hipLaunchKernelGGL(paged_join_rows_kernel<D>, dim3((unsigned)((tokens * head_groups + 3) / 4)), dim3(256), 0, st, p,
                         w.M, tokens * head_groups, (int)head_groups);
    MI355_CHECK_LAUNCH("paged_attn_fp8 (join)");
  }
  return MI355_OK;
}

}  // namespace

extern "C" int64_t mi355_paged_attn_workspace_bytes(const mi355_paged_attn_args* a) {
  if (check(a) != MI355_OK) return MI355_EINVAL;
  if (a->B == 0 || a->Sq == 0) return 0;
  const Plan w = plan_of(a);
  return w.part_bytes + w.info_bytes;
}

extern "C" int mi355_paged_attn_fp8(const mi355_paged_attn_args* a, void* stream) {
  if (int rc = check(a)) return rc;
  if (a->B == 0 || a->Sq == 0) return MI355_OK;
  MI355_REQUIRE(a->q && a->out && a->cache_seqlens, "paged_attn_fp8: null pointer");
  MI355_REQUIRE(a->table_width == 0 || (a->page_table && a->num_blocks > 0 && a->k_cache && a->v_cache &&
                                        a->k_scale && a->v_scale),
                "paged_attn_fp8: null pointer or no blocks");
  const int64_t strides[] = {a->q_sb, a->q_ss, a->q_sh, a->o_sb, a->o_ss, a->o_sh};
  for (int64_t s : strides)
    MI355_REQUIRE(s % 8 == 0, "paged_attn_fp8: strides of q and out must be multiples of 8 elements");
  const int64_t cache_strides[] = {a->kc_sb, a->kc_st, a->kc_sh, a->vc_sb, a->vc_st, a->vc_sh};
  for (int64_t s : cache_strides)
    MI355_REQUIRE(s % 16 == 0, "paged_attn_fp8: strides of the caches must be multiples of 16 bytes");
  MI355_REQUIRE(a->kc_st >= 0 && a->kc_st < (1 << 24) && a->vc_st >= 0 && a->vc_st < (1 << 24),
                "paged_attn_fp8: token stride of a cache too large");
  MI355_REQUIRE(((uintptr_t)a->q | (uintptr_t)a->out | (uintptr_t)a->k_cache | (uintptr_t)a->v_cache) % 16 == 0,
                "paged_attn_fp8: q, out and the caches must be 16-byte aligned");
  const Plan w = plan_of(a);
  MI355_REQUIRE(w.items * a->Hk < (1ll << 31), "paged_attn_fp8: too many row tiles");
  MI355_REQUIRE(a->workspace_bytes >= w.part_bytes + w.info_bytes && (!w.split || a->workspace) &&
                    (uintptr_t)a->workspace % 16 == 0,
                "paged_attn_fp8: workspace of %ld bytes needed (16-byte aligned), %ld given",
                (long)(w.part_bytes + w.info_bytes), (long)a->workspace_bytes);
  const int64_t batch = a->cu_seqlens_q ? 1 : a->B;
  const mi355::Rows q = {a->q, 2 * a->D, {batch, a->Sq, a->H}, {2 * a->q_sb, 2 * a->q_ss, 2 * a->q_sh}},
                    out = {a->out, 2 * a->D, {batch, a->Sq, a->H}, {2 * a->o_sb, 2 * a->o_ss, 2 * a->o_sh}};
  MI355_REQUIRE(rows_distinct(out), "paged_attn_fp8: rows of out overlap each other");
  MI355_REQUIRE(rows_same(out, q) || rows_apart(out, q), "paged_attn_fp8: out overlaps q and is not the same rows");
  PagedParams p;
  p.q = (const unsigned short*)a->q;
  p.o = (unsigned short*)a->out;
  p.lse = a->lse;
  p.kc = (const unsigned char*)a->k_cache;
  p.vc = (const unsigned char*)a->v_cache;
  p.ks = a->k_scale;
  p.vs = a->v_scale;
  p.cu = a->cu_seqlens_q;
  p.lens = a->cache_seqlens;
  p.table = a->page_table;
  p.q_sb = a->q_sb; p.q_ss = a->q_ss; p.q_sh = a->q_sh;
  p.o_sb = a->o_sb; p.o_ss = a->o_ss; p.o_sh = a->o_sh;
  p.lse_sb = a->lse_sb; p.lse_sh = a->lse_sh;
  p.kc_sb = a->kc_sb; p.kc_st = (int)a->kc_st; p.kc_sh = a->kc_sh;
  p.vc_sb = a->vc_sb; p.vc_st = (int)a->vc_st; p.vc_sh = a->vc_sh;
  p.table_stride = a->table_stride;
  p.B = (int)a->B;
  p.Hk = (int)a->Hk;
  p.G = (int)(a->H / a->Hk);
  p.Sq = (int)a->Sq;
  p.cap = (int)(a->table_width * a->block_size);
  p.num_blocks = (int)a->num_blocks;
  p.lb = __builtin_ctzll((unsigned long long)a->block_size);
  p.causal = a->causal != 0;
  p.window = a->window_left < 0 || a->window_left >= p.cap ? -1 : (int)a->window_left;  // (beyond: hides nothing)
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.items = (int)w.items;
  p.slots = (float)w.slots;
  // written and read, against what the chip moves while a workgroup does a tile of keys (2 us)
  p.join_cost = (float)(a->Hk * w.M * (a->D + 2) * 8) / 7e6f;
  p.chunk_min = w.chunk_min;
  p.split = w.split;
  p.by_length = !w.few && !w.split && a->causal && a->B > 1 && a->B <= SORTED_SEQS;
  p.hw = w.hw;
  p.turns = w.few ? 4 / w.hw : 1;
  p.part = (float*)a->workspace;
  p.info = (int32_t*)((char*)a->workspace + w.part_bytes);
  return a->D == 128 ? launch<128>(p, w, (hipStream_t)stream) : launch<64>(p, w, (hipStream_t)stream);
}
