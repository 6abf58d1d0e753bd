// What stands around a paged 8-bit key/value cache, for gfx950: block tables and slot maps from
// request lengths, rotary positions from scaled frequencies, and the store that rounds keys and
// values into the cache.  The attention that reads the cache is in paged_attention.hip.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "overlap.h"

namespace {

constexpr int KV_BLOCK_MIN = 16, KV_BLOCK_MAX = 1024;
constexpr int SCALE_EXP_MIN = -64;  // exponent of the scale of a block without a nonzero value

inline bool block_size_ok(int64_t bs) {
  return bs >= KV_BLOCK_MIN && bs <= KV_BLOCK_MAX && (bs & (bs - 1)) == 0;
}
inline int log2_of(int64_t bs) { return __builtin_ctzll((unsigned long long)bs); }

// ------------------------------------------------------------------------------------ plan --
// One launch.  Every workgroup adds up the lengths of all requests for itself (B values out of
// L2 and one scan over 256 threads, about as long as the gap between two launches) and then
// fills the slots of its own 1024 tokens, so nothing has to be handed from one workgroup to
// another.  Entries of the table that a workgroup reads (blocks held before the call) and
// entries that any workgroup writes (fresh blocks) are different ones.
// Bound by its launch and three loads that hang on each other: 48 requests of one token 2.7 us, 500
// prompts of 147 thousand tokens (2.4 MB) 6.6 us.
constexpr int PLAN_THREADS = 256, PLAN_TOKENS = 1024;
constexpr int64_t PLAN_MAX_REQUESTS = 4096;  // three ints each in LDS: 48 KiB

struct PlanParams {
  const int32_t *context_lens, *new_lens, *free_blocks, *free_begin;
  int32_t *table, *cu, *seq_lens, *free_end, *status;
  int64_t *slots, *positions;
  int64_t table_stride, table_width, num_free, num_blocks, max_tokens;
  int B, lb;
};

// Sum over the lanes up to this one of values below 2^36, in two halves of 32-bit lane operations.
__device__ __forceinline__ int64_t wave_scan36(int64_t v) {
  return ((int64_t)wave_scan((int)(v >> 16)) << 16) + wave_scan((int)(v & 0xffff));
}

__global__ __launch_bounds__(PLAN_THREADS) void kv_block_plan_kernel(PlanParams p) {
  extern __shared__ int32_t lds_plan[];
  int32_t* cu = lds_plan;                  // [B] first token of a request
  int32_t* fresh_at = lds_plan + p.B;      // [B] its first entry among the fresh blocks
  int32_t* context = lds_plan + 2 * p.B;   // [B]
  __shared__ int64_t wave_tok[4], wave_fresh[4];
  __shared__ int wave_wide[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t bs = 1ll << p.lb;
  const int64_t begin = max(p.free_begin[0], 0);
  // a thread owns `per` requests that follow each other: one scan over the threads is enough.  At
  // most 16 requests of less than 2^31 tokens each: its sums stay below 2^36.
  const int per = (p.B + PLAN_THREADS - 1) / PLAN_THREADS;
  const int i0 = tid * per, i1 = min(p.B, i0 + per);
  int64_t tok = 0, fresh = 0;
  int wide = 0;
  for (int i = i0; i < i1; ++i) {
    const int64_t c = max(p.context_lens[i], 0), n = max(p.new_lens[i], 0);
    const int64_t held = (c + bs - 1) >> p.lb, need = (c + n + bs - 1) >> p.lb;
    context[i] = (int)c;
    tok += n;
    fresh += need - held;
    wide += need > p.table_width;
  }
  const int64_t tok_in = wave_scan36(tok), fresh_in = wave_scan36(fresh);  // inclusive over the wave
  wide = wave_scan(wide);
  if (lane == 63) {
    wave_tok[wave] = tok_in;
    wave_fresh[wave] = fresh_in;
    wave_wide[wave] = wide;
  }
  __syncthreads();
  int64_t tok_all = 0, fresh_all = 0, tok_at = tok_in - tok, fresh_from = fresh_in - fresh;
  int wide_all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) {
      tok_at += wave_tok[w];
      fresh_from += wave_fresh[w];
    }
    tok_all += wave_tok[w];
    fresh_all += wave_fresh[w];
    wide_all += wave_wide[w];
  }
  const int64_t lacking = max((int64_t)0, begin + fresh_all - p.num_free);
  const int64_t over = max((int64_t)0, tok_all - p.max_tokens);
  const bool good = lacking == 0 && over == 0 && wide_all == 0;
  const bool first_group = blockIdx.x == 0;
  for (int i = i0; i < i1; ++i) {
    const int64_t c = context[i], n = max(p.new_lens[i], 0);
    if (good) {  // the sums fit: tokens are below max_tokens, blocks below num_free
      cu[i] = (int)tok_at;
      fresh_at[i] = (int)fresh_from;
    }
    if (first_group) {
      p.cu[i] = good ? (int)tok_at : 0;
      p.seq_lens[i] = (int)(good ? c + n : c);
    }
    tok_at += n;
    fresh_from += ((c + n + bs - 1) >> p.lb) - ((c + bs - 1) >> p.lb);
  }
  if (first_group && tid == 0) {
    p.cu[p.B] = good ? (int)tok_all : 0;
    p.free_end[0] = (int)(begin + (good ? fresh_all : 0));
    p.status[0] = (int)min(lacking, (int64_t)INT32_MAX);
    p.status[1] = (int)min(over, (int64_t)INT32_MAX);
    p.status[2] = wide_all;
  }
  __syncthreads();
  // Tokens t0, t0 + 256, ...: four at a time, so that their searches and look-ups go on together.
  const int64_t t0 = (int64_t)blockIdx.x * PLAN_TOKENS + tid;
  auto fill = [&](auto count, int64_t from) {
    constexpr int N = decltype(count)::value;
    int lo[N], hi[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      lo[k] = 0;
      hi[k] = p.B;
    }
    // the last request that begins at or before t is the one that holds it
    for (int left = good ? p.B : 1; left > 1; left = (left + 1) >> 1) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int mid = (lo[k] + hi[k]) >> 1;
        const bool up = cu[mid] <= (int)(from + k * PLAN_THREADS);  // (mid is in [0, B))
        lo[k] = up ? mid : lo[k];
        hi[k] = up ? hi[k] : mid;
      }
    }
    int64_t place[N];
    int id[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t t = from + k * PLAN_THREADS;
      place[k] = 0;
      id[k] = -1;
      if (good && t < tok_all) {
        const int64_t c = context[lo[k]];
        place[k] = c + (t - cu[lo[k]]);
        const int64_t j = place[k] >> p.lb, held = (c + bs - 1) >> p.lb;
        id[k] = j < held ? p.table[lo[k] * p.table_stride + j] : p.free_blocks[begin + fresh_at[lo[k]] + (j - held)];
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t t = from + k * PLAN_THREADS;
      if (t >= p.max_tokens) continue;
      // a block's first token: never one held before
      if (good && t < tok_all && (place[k] & (bs - 1)) == 0)
        p.table[lo[k] * p.table_stride + (place[k] >> p.lb)] = id[k];
      p.slots[t] = id[k] >= 0 && id[k] < p.num_blocks ? ((int64_t)id[k] << p.lb) + (place[k] & (bs - 1)) : -1;
      p.positions[t] = place[k];
    }
  };
  if (p.max_tokens > 2 * PLAN_THREADS) {
    fill(std::integral_constant<int, 4>{}, t0);
  } else {
    for (int64_t t = t0; t - tid < p.max_tokens; t += PLAN_THREADS) fill(std::integral_constant<int, 1>{}, t);
  }
}

// ------------------------------------------------------------------------------------ rope --
struct Rope {
  const int64_t* positions;
  const void* inv_freq;  // [half], fp64 or fp32
  int f64, half, neox;
  double factor;
};

// cos and sin of position * frequency, times the factor.  The product is formed in quarter turns
// and in fp64 (a position of 10^6 leaves fp32 0.06 rad of it), reduced exactly to an eighth of a
// turn on either side of the nearest quarter, and evaluated there by the Taylor sums, in fp64 up to
// the terms that stay below 10^-11: rounded to fp32 they are as good as correctly rounded.  That is
// some twenty fp64 operations for a pair of a token, shared by all its heads (or by a block's rows).
__device__ __forceinline__ double rope_quarters(const Rope& r, int i) {  // turned for each position, in quarters
  return (r.f64 ? reinterpret_cast<const double*>(r.inv_freq)[i]
                : (double)reinterpret_cast<const float*>(r.inv_freq)[i]) * 0.63661977236758134308;  // 2 / pi
}
__device__ __forceinline__ float2 rope_cos_sin(const Rope& r, int64_t pos, double each) {
  const double quarters = (double)pos * each;
  const double whole = rint(quarters);
  const double a = (quarters - whole) * 1.57079632679489661923, a2 = a * a;
  const int quadrant = (int)(whole - 4.0 * floor(whole * 0.25));
  double s = fma(a2, -1.0 / 39916800.0, 1.0 / 362880.0);
  s = fma(a2, s, -1.0 / 5040.0);
  s = fma(a2, s, 1.0 / 120.0);
  s = fma(a2, s, -1.0 / 6.0);
  s = fma(a2 * a, s, a);
  double c = fma(a2, 1.0 / 479001600.0, -1.0 / 3628800.0);
  c = fma(a2, c, 1.0 / 40320.0);
  c = fma(a2, c, -1.0 / 720.0);
  c = fma(a2, c, 1.0 / 24.0);
  c = fma(a2, c, -0.5);
  c = fma(a2, c, 1.0);
  const double cq = quadrant & 1 ? s : c, sq = quadrant & 1 ? c : s;
  return make_float2((float)((quadrant == 1 || quadrant == 2 ? -cq : cq) * r.factor),
                     (float)((quadrant >= 2 ? -sq : sq) * r.factor));
}

__device__ __forceinline__ void unpack8(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = __uint_as_float(v[j] << 16);
    f[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  return u32x4{pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7])};
}
__device__ __forceinline__ void turn(float& a, float& z, float2 cs) {
  const float u = fmaf(-z, cs.y, __fmul_rn(a, cs.x));
  z = fmaf(a, cs.y, __fmul_rn(z, cs.x));
  a = u;
}

// Rows of one tensor: [tokens, heads, D] with its own strides, in and out (which may be the same).
struct RopeRows {
  const unsigned short* x;
  unsigned short* out;
  int64_t st, sh, ot, oh;
  int heads;
};

// One piece of a row.  Pieces [0, turned) hold pairs: 8 elements of each half (half layout) or 8
// neighbours (interleaved); the pieces behind them are copied as they are.
__device__ __forceinline__ void rope_piece(const Rope& r, const unsigned short* x, unsigned short* out,
                                           int piece, int turned, const float2* cs) {
  if (piece >= turned) {
    const int at = 2 * r.half + (piece - turned) * 8;
    *reinterpret_cast<u32x4*>(out + at) = *reinterpret_cast<const u32x4*>(x + at);
    return;
  }
  float f[8];
  if (r.neox) {
    float g[8];
    const int at = piece * 8;
    unpack8(*reinterpret_cast<const u32x4*>(x + at), f);
    unpack8(*reinterpret_cast<const u32x4*>(x + at + r.half), g);
#pragma unroll
    for (int j = 0; j < 8; ++j) turn(f[j], g[j], cs[at + j]);
    *reinterpret_cast<u32x4*>(out + at) = pack8(f);
    *reinterpret_cast<u32x4*>(out + at + r.half) = pack8(g);
  } else {
    unpack8(*reinterpret_cast<const u32x4*>(x + piece * 8), f);
#pragma unroll
    for (int j = 0; j < 4; ++j) turn(f[2 * j], f[2 * j + 1], cs[piece * 4 + j]);
    *reinterpret_cast<u32x4*>(out + piece * 8) = pack8(f);
  }
}

constexpr int ROPE_THREADS = 256, ROPE_MAX_HALF = 128, ROPE_MAX_TOKENS = 4;

// The rows of tokens [t0, t0 + nt) of two tensors (the second may have no heads).  Cosine and
// sine of a token are formed once for all its heads and kept in LDS: with 40 heads of 128 that
// is 1/40 of the fp64 products that forming them at each pair would take.  Bound by memory from some
// hundred tokens on: 8191 of 40 heads of 128, 168 MB in 35.8 us = 4.7 TB/s where nothing of it is in a
// cache (a large copy: 4.9), over the same memory again and again 28.7.
template <int THREADS>
__device__ __forceinline__ void rope_tokens(const Rope& r, const RopeRows& a, const RopeRows& b, int D,
                                            int64_t t0, int nt, float2* cs) {
  for (int i = threadIdx.x; i < nt * r.half; i += THREADS) {
    const int k = i / r.half;
    cs[i] = rope_cos_sin(r, r.positions[t0 + k], rope_quarters(r, i - k * r.half));
  }
  __syncthreads();
  const int turned = r.neox ? r.half / 8 : r.half / 4;
  const int copied = (D - 2 * r.half) / 8;
  const int pieces = turned + copied, heads = a.heads + b.heads;
  for (int i = threadIdx.x; i < nt * heads * pieces; i += THREADS) {
    const int piece = i % pieces, row = i / pieces, head = row % heads, k = row / heads;
    const RopeRows& m = head < a.heads ? a : b;
    const int h = head < a.heads ? head : head - a.heads;
    if (piece >= turned && m.x == m.out) continue;
    rope_piece(r, m.x + (t0 + k) * m.st + h * m.sh, m.out + (t0 + k) * m.ot + h * m.oh, piece, turned,
               cs + k * r.half);
  }
}

__global__ __launch_bounds__(ROPE_THREADS) void rope_scaled_kernel(Rope r, RopeRows q, RopeRows k, int D,
                                                                   int64_t tokens, int per_group) {
  __shared__ float2 cs[ROPE_MAX_TOKENS * ROPE_MAX_HALF];
  const int64_t t0 = (int64_t)blockIdx.x * per_group;
  rope_tokens<ROPE_THREADS>(r, q, k, D, t0, (int)min((int64_t)per_group, tokens - t0), cs);
}

// Tokens of one workgroup: one, until there are some thirty for each CU, since the last round of
// long workgroups leaves much of the chip idle (1714 tokens, 144 heads of 128: 34 us, by fours 55); then
// four, since very many small workgroups are held up by their own dispatch (60000 tokens, 3 heads of
// 64: 17 us, by ones 44; 8191 tokens, 40 heads of 128: 37.4 us, by ones 38.0, by eights 46.7).
inline int rope_group(int64_t tokens) { return tokens >= 7168 ? ROPE_MAX_TOKENS : 1; }

// ----------------------------------------------------------------------------------- store --
// A run is the tokens of a call that follow each other into one block, for one head and one of the
// two caches.  The workgroup among whose tokens a run begins (the token before it goes to another
// block) takes it; where a block has several (a token between them is skipped, or goes elsewhere), the
// one with the first takes them all, so no two of them write one block's scale.  A team holds a run: one wave up to 16 rows
// of 128, the whole workgroup beyond that, with as many threads as a block's rows ask for.  A row of
// D elements is held by D / 8 lanes, and the team holds HELD sets of rows in registers between the
// maximum and the rounding; longer runs are read a second time.  Cosines and sines of these rows
// are formed together and handed on through LDS.
// Keys come first in the grid, then values, then the queries' rotation: what takes longest begins
// first.
//
// 48 runs of one token take 6.4 us, bound by the chain slot, row and scale, maximum, code; 1200 of them
// 31 (run after run by whole workgroups: 106).  4602 tokens of 12 prompts (104 MB with 32 heads of
// queries) take 32 us = 3.3 TB/s, among other calls 39: 15 for the queries alone, and for keys and values
// the chain again, the look for tokens elsewhere (3) and the cosines, which each head forms for itself.
// Blocks of 256: 2420 tokens of 3 prompts 43 us (threads: 1842 tokens took 25 with 1024 and 70 with 256);
// blocks of 1024: 1400 tokens 126, read twice.  Measured and slower, where these 12 prompts took 38: keys
// and values in turn (44), queries in turn with both (52), 128 threads with eight rows each (53-62), 512
// with two (45), five or more waves a SIMD (52-80, more values in scratch memory; at four the instances
// of 256 and 512 threads keep theirs in 124 registers, that of 1024 puts six out).
constexpr int HELD = 4;
struct StoreParams {
  const unsigned short *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
  unsigned char *k_cache, *v_cache;
  int64_t kc_sb, kc_st, kc_sh, vc_sb, vc_st, vc_sh;
  float *k_scale, *v_scale;  // [blocks, heads]
  const int64_t* slots;
  int64_t tokens, num_blocks;
  int Hk, lb, group;
  unsigned kv_groups;  // workgroups before those that turn the queries; half of them keys'
  int q_group;
  Rope rope;           // positions == nullptr: keys are stored as they are
  RopeRows q;
};

__device__ __forceinline__ bool finite(float x) {
  return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
}

// 8 values times a power of two -> 8 e4m3 bytes, to the nearest, ties to even; what is not
// finite becomes NaN (e4m3 has no infinity)
__device__ __forceinline__ u32x2 round_fp8(const float (&f)[8], float inv) {
  u32x2 o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float g[4];
    unsigned bad = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = f[4 * h + j];
      if (!finite(x)) bad |= 0x7fu << (8 * j);
      g[j] = finite(x) ? clamp_fp8(x * inv, -FP8_E4M3_MAX, FP8_E4M3_MAX) : 0.f;
    }
    o[h] = cvt4_fp8(g[0], g[1], g[2], g[3]) | bad;
  }
  return o;
}

// THREADS that hold a run together.  A wave has room for the cosines of one set of rows (4 of 128, 8 of
// 64), a workgroup for those of 1024 / (D / 8) rows.
template <int D, int THREADS>
struct StoreLds {
  static constexpr int ROWS = THREADS / (D / 8);  // of a set
  static constexpr int TURNED = THREADS == 64 ? 1 : 1024 / THREADS;  // sets whose cosines there is room for
  float2 cs[TURNED * ROWS][D / 2];
  float top[THREADS / 64];
  int first[THREADS / 64];
};
// what one thread of a team wrote to LDS is there for the others
template <int THREADS>
__device__ __forceinline__ void team_sync() {
  if constexpr (THREADS > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// `len` tokens of one block: t0, t0 + 1, ..., or (LISTED) list[0], list[1], ...
template <int D, int THREADS, bool LISTED = false>
__device__ void store_run(const StoreParams& p, bool keys, int t0, const int* list, int len, int block, int head,
                          StoreLds<D, THREADS>& lds) {
  constexpr int LPR = D / 8, ROWS = StoreLds<D, THREADS>::ROWS, CHUNK = HELD * ROWS;
  const int lane = threadIdx.x & 63, wave = THREADS > 64 ? threadIdx.x >> 6 : 0;  // of the team
  const int c = lane % LPR, sub = (64 * wave + lane) / LPR;
  const int bs = 1 << p.lb;
  const Rope& r = p.rope;
  const bool turned = keys && r.positions;
  float* scale_at = (keys ? p.k_scale : p.v_scale) + (int64_t)block * p.Hk + head;
  const float old = *scale_at;
  u32x4 held[HELD];
  int place[HELD];  // in the block; bs: no row
  // CHUNK rows of the run, keys rotated.  The rotated key is a bf16 value before it is rounded to 8
  // bits, as it would be between the rotary operator and the store.
  const int64_t st = keys ? p.k_st : p.v_st;
  const unsigned short* rows_at = (keys ? p.k + head * p.k_sh : p.v + head * p.v_sh) + t0 * st;
  const int64_t* slots_at = p.slots + t0;
  const int64_t* positions_at = r.positions + t0;
  auto nth = [&](int row) {
    if constexpr (LISTED) return list[row];
    else return row;
  };
  auto fetch = [&](int row0) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int row = row0 + h * ROWS + sub;
      held[h] = u32x4{0, 0, 0, 0};
      place[h] = bs;
      if (row < len) {
        held[h] = *reinterpret_cast<const u32x4*>(rows_at + nth(row) * st + 8 * c);
        place[h] = (int)slots_at[nth(row)] & (bs - 1);
      }
    }
    if (!turned) return;
    constexpr int TURNED = StoreLds<D, THREADS>::TURNED;
#pragma unroll
    for (int h0 = 0; h0 < HELD; h0 += TURNED) {
      const int from = row0 + h0 * ROWS;
      if (h0 && from >= len) break;
      const int rows = min(TURNED * ROWS, len - from);
      team_sync<THREADS>();  // what was here before has been read
      // a lane keeps its pair, and goes over the rows
      const int side = 64 / r.half, pair = lane % r.half, k0 = wave * side + lane / r.half;
      if (lane < side * r.half) {
        const double each = rope_quarters(r, pair);
#pragma unroll 1
        for (int k = k0; k < rows; k += THREADS / 64 * side)
          lds.cs[k][pair] = rope_cos_sin(r, positions_at[nth(from + k)], each);
      }
      team_sync<THREADS>();
      const bool mine = 8 * c < 2 * r.half;
#pragma unroll
      for (int h = h0; h < h0 + TURNED; ++h) {
        float f[8];
        unpack8(held[h], f);
        const float2* cs = lds.cs[(h - h0) * ROWS + sub];
        if (r.neox) {
          // the other element of each pair is `half` away: half / 8 lanes, in the same row and wave
          const int away = r.half / 8;
          const bool second = c >= away;
          const int from = mine ? (second ? lane - away : lane + away) : lane;
          u32x4 other;
#pragma unroll
          for (int j = 0; j < 4; ++j) other[j] = __shfl(held[h][j], from, 64);
          float g[8];
          unpack8(other, g);
          if (mine && place[h] < bs) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 w = cs[(second ? c - away : c) * 8 + j];
              if (second) turn(g[j], f[j], w);
              else turn(f[j], g[j], w);
            }
          }
        } else if (mine && place[h] < bs) {
#pragma unroll
          for (int j = 0; j < 4; ++j) turn(f[2 * j], f[2 * j + 1], cs[c * 4 + j]);
        }
        held[h] = pack8(f);
      }
    }
  };
  // the largest finite magnitude and the smallest place in the block
  float top = 0.f;
  int first = bs;
  for (int row0 = 0; row0 < len; row0 += CHUNK) {
    fetch(row0);
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      float f[8];
      unpack8(held[h], f);
      first = min(first, place[h]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (finite(f[j])) top = fmaxf(top, fabsf(f[j]));  // rows behind the run are zeros
    }
  }
  top = group_max<64>(top);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
  team_sync<THREADS>();  // the run before has been read, and every thread has the old scale
  if constexpr (THREADS > 64) {
    if (lane == 0) {
      lds.top[wave] = top;
      lds.first[wave] = first;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      top = fmaxf(top, lds.top[w]);
      first = min(first, lds.first[w]);
    }
  }
  // the smallest power of two with top <= 448 * 2^e: 448 = 1.75 * 2^8
  const unsigned bits = __float_as_uint(top);
  const int e = max(SCALE_EXP_MIN, (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));
  float scale = __uint_as_float((unsigned)(e + 127) << 23);
  unsigned char* cache = (keys ? p.k_cache : p.v_cache) + (int64_t)block * (keys ? p.kc_sb : p.vc_sb) +
                         head * (keys ? p.kc_sh : p.vc_sh) + 8 * c;
  const int64_t row_bytes = keys ? p.kc_st : p.vc_st;
  if (first > 0) {
    if (old >= scale) {
      scale = old;
    } else if (old > 0.f) {  // the block's earlier tokens to the larger step
      const float shrink = old / scale;
      for (int i = sub; i < first; i += ROWS) {
        u32x2* at = reinterpret_cast<u32x2*>(cache + i * row_bytes);
        const u32x2 w = *at;
        u32x2 n;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[h], false);
          const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[h], true);
          unsigned nan = 0;  // NaN stays NaN
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (((w[h] >> (8 * j)) & 0x7f) == 0x7f) nan |= 0xffu << (8 * j);
          n[h] = (cvt4_fp8(lo[0] * shrink, lo[1] * shrink, hi[0] * shrink, hi[1] * shrink) & ~nan) | (nan & 0x7f7f7f7fu);
        }
        *at = n;
      }
    }
  }
  if (wave == 0 && lane == 0) *scale_at = scale;
  const float inv = 1.f / scale;  // exact: a power of two (a scale that a caller set may be any)
  for (int row0 = 0; row0 < len; row0 += CHUNK) {
    if (len > CHUNK) fetch(row0);
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      float f[8];
      unpack8(held[h], f);
      if (place[h] < bs) *reinterpret_cast<u32x2*>(cache + place[h] * row_bytes) = round_fp8(f, inv);
    }
  }
}

template <int D, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void kv_store_kernel(StoreParams p) {
  constexpr int WAVES = THREADS / 64;
  __shared__ union {
    float2 q[ROPE_MAX_HALF * ROPE_MAX_TOKENS];
    StoreLds<D, THREADS> kv;
    StoreLds<D, 64> wave[WAVES];
  } lds;
  if (blockIdx.x >= p.kv_groups) {
    const int64_t t0 = (int64_t)(blockIdx.x - p.kv_groups) * p.q_group;
    rope_tokens<THREADS>(p.rope, p.q, RopeRows{nullptr, nullptr, 0, 0, 0, 0, 0}, D, t0,
                         (int)min((int64_t)p.q_group, p.tokens - t0), lds.q);
    return;
  }
  // a workgroup: (group of tokens, head, keys or values); each wave finds the runs that begin there
  __shared__ unsigned long long apart[2];
  __shared__ int list[KV_BLOCK_MAX], listed;
  const unsigned half = p.kv_groups / 2;
  const bool keys = blockIdx.x < half;
  const unsigned part = keys ? blockIdx.x : blockIdx.x - half;
  const int head = (int)(part % p.Hk);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w0 = (int)(part / p.Hk) * p.group, t = w0 + lane;  // 64 slots: the group's and those behind it
  const int64_t limit = p.num_blocks << p.lb;
  const unsigned tokens = (unsigned)p.tokens;
  auto block_of = [&](unsigned token) {  // -1: none, or its slot is outside the pool
    const uint64_t s = p.slots[min(token, tokens - 1)];  // (no branch: loads go on side by side)
    return token < tokens && s < (uint64_t)limit ? (int)(s >> p.lb) : -1;
  };
  const int block = block_of(t), last = t ? block_of(t - 1) : -1;
  const unsigned long long begins = __ballot(lane < p.group && block >= 0 && last != block);
  if (!begins) return;
  // the run that begins at lane l: its block, and its length, to the first slot of another block, if
  // need be behind these 64
  int run_len = 0;  // of the run that begins at this lane
  for (unsigned long long todo = begins; todo; todo &= todo - 1) {
    const int l = __ffsll(todo) - 1, mine = __builtin_amdgcn_readlane(block, l);
    int len = 0;
    unsigned long long out = __ballot(lane >= l && block != mine);
    if (out) len = __ffsll(out) - 1 - l;
    for (int at = w0 + 64; !out; at += 64) {
      out = __ballot(block_of(at + lane) != mine);
      len = at - w0 - l + (out ? __ffsll(out) - 1 : 0);
    }
    if (lane == l) run_len = len;
  }
  // Runs that do not fill their block, and whose block has tokens elsewhere in the call (`more`; `earlier`:
  // before the run, which is the first one's then).  The low eleven bits of a block choose a bit of 64 x 32;
  // where another run begins in a block whose bit is set, ours are asked.  Without it 4602 tokens of 12
  // prompts take 30 us instead of 33, and 48 single tokens 6.3 instead of 6.4; more or fewer loads in flight
  // than 12, or fetched before the runs are measured, take as long.
  unsigned long long more = 0, earlier = 0;
  const unsigned long long partial = __ballot(run_len > 0 && run_len < (1 << p.lb));
  if (partial) {
    unsigned bits = 0, twice = 0;  // twice: two of ours have one bit
    for (unsigned long long todo = partial; todo; todo &= todo - 1) {
      const int mine = __builtin_amdgcn_readlane(block, __ffsll(todo) - 1);
      const unsigned bit = 1u << (mine & 31);
      twice |= (unsigned)__builtin_amdgcn_readlane((int)bits, (mine >> 5) & 63) & bit;
      if (lane == ((mine >> 5) & 63)) bits |= bit;
    }
    // N loads of 64 slots in flight, `step` slots apart
    auto search = [&](auto count, unsigned at0, unsigned step) {
      constexpr int N = decltype(count)::value;
#pragma unroll 1
      for (; at0 < tokens; at0 += N * step) {
        int theirs[N];
#pragma unroll
        for (int u = 0; u < N; ++u) theirs[u] = block_of(at0 + u * step + lane);
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const unsigned first = at0 + u * step;
          if (first >= tokens) break;
          const int before = __builtin_amdgcn_update_dpp(-2, theirs[u], 0x138, 0xf, 0xf, false);  // wave_shr:1
          const unsigned word = (unsigned)__shfl((int)bits, (theirs[u] >> 5) & 63, 64);
          const bool ours = !twice && first + lane - (unsigned)w0 < (unsigned)p.group;
          for (unsigned long long hits = __ballot(theirs[u] >= 0 && theirs[u] != before && !ours &&
                                                  ((word >> (theirs[u] & 31)) & 1));
               hits; hits &= hits - 1) {
            const int h = __ffsll(hits) - 1, at = (int)first + h;
            const bool same = run_len > 0 && block == __builtin_amdgcn_readlane(theirs[u], h);
            more |= __ballot(same && (at < t || at - t >= run_len)) & partial;
            earlier |= __ballot(same && at < t) & partial;
          }
        }
      }
    };
    // few tokens: every wave goes over all of them, in little code (eight loads in flight: 0.5 us more)
    if (tokens <= 256) {
      search(std::integral_constant<int, 1>{}, 0, 64);
    } else {
      if (threadIdx.x == 0) apart[0] = apart[1] = 0;
      search(std::integral_constant<int, 12>{}, 64 * wave, THREADS);
      __syncthreads();
      if (lane == 0 && more) {
        atomicOr(&apart[0], more);
        atomicOr(&apart[1], earlier);
      }
      __syncthreads();
      more = apart[0];
      earlier = apart[1];
    }
  }
  const unsigned long long runs = begins & ~more;
  // runs that a wave holds go to the waves in turn, the others to all of them together
  constexpr int FEW = HELD * StoreLds<D, 64>::ROWS;
  const unsigned long long few = runs & __ballot(run_len <= FEW);
  for (unsigned long long todo = runs & ~few; todo; todo &= todo - 1) {
    const int l = __ffsll(todo) - 1;
    store_run<D, THREADS>(p, keys, w0 + l, nullptr, __builtin_amdgcn_readlane(run_len, l),
                          __builtin_amdgcn_readlane(block, l), head, lds.kv);
  }
  if (few != runs) __syncthreads();  // (the LDS is used anew)
  int turn = 0;
  for (unsigned long long todo = few; todo; todo &= todo - 1, turn = turn + 1 == WAVES ? 0 : turn + 1) {
    if (turn != wave) continue;
    const int l = __ffsll(todo) - 1;
    store_run<D, 64>(p, keys, w0 + l, nullptr, __builtin_amdgcn_readlane(run_len, l),
                     __builtin_amdgcn_readlane(block, l), head, lds.wave[wave]);
  }
  // blocks whose tokens stand apart, with a list of them: one block after the other (500 x 8 tokens, 8 heads:
  // in order 23 us, every third one skipped 63, the sequences in turn 214)
  for (unsigned long long todo = more & ~earlier; todo; todo &= todo - 1) {
    const int mine = __builtin_amdgcn_readlane(block, __ffsll(todo) - 1);
    __syncthreads();
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    for (unsigned at = threadIdx.x; at < tokens; at += THREADS) {
      if (block_of(at) != mine) continue;
      const int i = atomicAdd(&listed, 1);
      if (i < KV_BLOCK_MAX) list[i] = (int)at;  // (more only if a slot is given twice)
    }
    __syncthreads();
    store_run<D, THREADS, true>(p, keys, 0, list, min(listed, 1 << p.lb), mine, head, lds.kv);
  }
}

using mi355::Rows;
// [tokens, heads, D] in bf16, strides in elements
Rows head_rows(const void* at, int64_t tokens, int64_t heads, int64_t D, int64_t st, int64_t sh) {
  return Rows{at, 2 * D, {1, tokens, heads}, {0, 2 * st, 2 * sh}};
}
// an output may be an input of its own, and must not touch it otherwise
bool same_or_apart(const Rows& out, const Rows& in) { return rows_same(out, in) || rows_apart(out, in); }

bool rope_args_ok(const char* what, int64_t head_size, int64_t rot_dim, const void* inv_freq,
                  const int64_t* positions, int64_t tokens) {
  if (tokens && (!positions || !inv_freq)) {
    mi355_set_error("%s: null pointer", what);
    return false;
  }
  if (rot_dim <= 0 || rot_dim % 16 != 0 || rot_dim > head_size) {
    mi355_set_error("%s: rot_dim %ld must be a multiple of 16 within the head size %ld", what,
                    (long)rot_dim, (long)head_size);
    return false;
  }
  return true;
}

}  // namespace

extern "C" int mi355_kv_block_plan(const int32_t* context_lens, const int32_t* new_lens, int64_t B,
                                   int32_t* block_table, int64_t table_stride, int64_t table_width,
                                   const int32_t* free_blocks, int64_t num_free,
                                   const int32_t* free_begin, int64_t block_size, int64_t num_blocks,
                                   int64_t* slot_mapping, int64_t* positions, int64_t max_tokens,
                                   int32_t* cu_seqlens_q, int32_t* seq_lens, int32_t* free_end,
                                   int32_t* status, void* stream) {
  MI355_REQUIRE(B >= 0 && B <= PLAN_MAX_REQUESTS, "kv_block_plan: %ld requests, at most %ld in one call",
                (long)B, (long)PLAN_MAX_REQUESTS);
  MI355_REQUIRE(block_size_ok(block_size), "kv_block_plan: block size %ld must be a power of two in [16, 1024]",
                (long)block_size);
  MI355_REQUIRE(max_tokens >= 0 && max_tokens <= (1ll << 31) - 4096 && num_free >= 0 && num_free < (1ll << 31) &&
                    num_blocks >= 0 && num_blocks < (1ll << 31) && table_width >= 0 && table_width < (1ll << 31) &&
                    table_width * block_size <= (1ll << 31) - 4096 && table_stride < (1ll << 40) &&
                    (B <= 1 || table_stride >= table_width),
                "kv_block_plan: bad size");
  MI355_REQUIRE(free_begin && cu_seqlens_q && free_end && status, "kv_block_plan: null pointer");
  MI355_REQUIRE(B == 0 || (context_lens && new_lens && seq_lens && (block_table || table_width == 0)),
                "kv_block_plan: null pointer");
  MI355_REQUIRE(max_tokens == 0 || (slot_mapping && positions), "kv_block_plan: null pointer");
  MI355_REQUIRE(num_free == 0 || free_blocks, "kv_block_plan: null pointer");
  // every workgroup reads the inputs, some while others write already
  struct Span {
    const void* at;
    int64_t bytes;
  };
  const Span in[] = {{context_lens, 4 * B}, {new_lens, 4 * B}, {free_blocks, 4 * num_free}, {free_begin, 4},
                     {block_table, B ? 4 * ((B - 1) * table_stride + table_width) : 0}};
  const Span out[] = {{cu_seqlens_q, 4 * (B + 1)}, {seq_lens, 4 * B}, {free_end, 4}, {status, 12},
                      {slot_mapping, 8 * max_tokens}, {positions, 8 * max_tokens}};
  auto apart = [](const Span& a, const Span& b) {
    return a.bytes == 0 || b.bytes == 0 || (uintptr_t)a.at + a.bytes <= (uintptr_t)b.at ||
           (uintptr_t)b.at + b.bytes <= (uintptr_t)a.at;
  };
  bool clear = apart(in[2], in[4]);  // the table is written as well
  for (const Span& o : out) {
    for (const Span& i : in) clear = clear && apart(o, i);
    for (const Span& o2 : out) clear = clear && (&o == &o2 || apart(o, o2));
  }
  MI355_REQUIRE(clear, "kv_block_plan: outputs must not share memory with inputs or with each other");
  PlanParams p = {context_lens, new_lens, free_blocks, free_begin, block_table, cu_seqlens_q, seq_lens,
                  free_end, status, slot_mapping, positions, table_stride, table_width, num_free, num_blocks,
                  max_tokens, (int)B, log2_of(block_size)};
  const int64_t groups = max_tokens ? (max_tokens + PLAN_TOKENS - 1) / PLAN_TOKENS : 1;
  const size_t lds = (size_t)(3 * B) * sizeof(int32_t);
  hipLaunchKernelGGL(kv_block_plan_kernel, dim3((unsigned)groups), dim3(PLAN_THREADS), lds,
                     (hipStream_t)stream, p);
  MI355_CHECK_LAUNCH("kv_block_plan");
  return MI355_OK;
}

extern "C" int mi355_rope_scaled(const int64_t* positions, const void* q, void* q_out, const void* k,
                                 void* k_out, int64_t tokens, int64_t Hq, int64_t Hk, int64_t head_size,
                                 int64_t rot_dim, int64_t q_st, int64_t q_sh, int64_t qo_st, int64_t qo_sh,
                                 int64_t k_st, int64_t k_sh, int64_t ko_st, int64_t ko_sh,
                                 const void* inv_freq, int inv_freq_is_f64, float attn_factor, int is_neox,
                                 void* stream) {
  MI355_REQUIRE(tokens >= 0 && Hq >= 0 && Hk >= 0 && tokens < (1ll << 31) && Hq < 65536 && Hk < 65536,
                "rope_scaled: bad shape");
  if (tokens == 0 || Hq + Hk == 0) return MI355_OK;
  MI355_REQUIRE(head_size > 0 && head_size % 8 == 0 && head_size <= 2 * ROPE_MAX_HALF,
                "rope_scaled: head size %ld must be a multiple of 8, at most 256", (long)head_size);
  if (!rope_args_ok("rope_scaled", head_size, rot_dim, inv_freq, positions, tokens)) return MI355_EINVAL;
  MI355_REQUIRE((Hq == 0 || (q && q_out)) && (Hk == 0 || (k && k_out)), "rope_scaled: null pointer");
  const int64_t strides[] = {q_st, q_sh, qo_st, qo_sh, k_st, k_sh, ko_st, ko_sh};
  for (int64_t s : strides)
    MI355_REQUIRE(s % 8 == 0, "rope_scaled: strides must be multiples of 8 elements");
  MI355_REQUIRE(((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)k_out) % 16 == 0,
                "rope_scaled: rows must be 16-byte aligned");
  const Rows q_in = head_rows(q, tokens, Hq, head_size, q_st, q_sh), k_in = head_rows(k, tokens, Hk, head_size, k_st, k_sh),
             q_to = head_rows(q_out, tokens, Hq, head_size, qo_st, qo_sh),
             k_to = head_rows(k_out, tokens, Hk, head_size, ko_st, ko_sh);
  MI355_REQUIRE(rows_distinct(q_to) && rows_distinct(k_to), "rope_scaled: rows of an output overlap each other");
  MI355_REQUIRE(same_or_apart(q_to, q_in) && same_or_apart(k_to, k_in),
                "rope_scaled: an output overlaps its input and is not the same rows");
  MI355_REQUIRE(rows_apart(q_to, k_in) && rows_apart(k_to, q_in) && rows_apart(q_to, k_to),
                "rope_scaled: an output overlaps the other tensor");
  Rope r = {positions, inv_freq, inv_freq_is_f64, (int)(rot_dim / 2), is_neox != 0, attn_factor};
  RopeRows a = {(const unsigned short*)q, (unsigned short*)q_out, q_st, q_sh, qo_st, qo_sh, (int)Hq};
  RopeRows b = {(const unsigned short*)k, (unsigned short*)k_out, k_st, k_sh, ko_st, ko_sh, (int)Hk};
  const int per = rope_group(tokens);
  hipLaunchKernelGGL(rope_scaled_kernel, dim3((unsigned)((tokens + per - 1) / per)), dim3(ROPE_THREADS), 0,
                     (hipStream_t)stream, r, a, b, (int)head_size, tokens, per);
  MI355_CHECK_LAUNCH("rope_scaled");
  return MI355_OK;
}

extern "C" int mi355_kv_store_fp8(const mi355_kv_store_args* a, void* stream) {
  MI355_REQUIRE(a != nullptr, "kv_store_fp8: null args");
  MI355_REQUIRE(a->D == 64 || a->D == 128, "kv_store_fp8: head size %ld not in {64,128}", (long)a->D);
  MI355_REQUIRE(block_size_ok(a->block_size), "kv_store_fp8: block size %ld must be a power of two in [16, 1024]",
                (long)a->block_size);
  MI355_REQUIRE(a->tokens >= 0 && a->tokens <= (1ll << 31) - 4096 && a->Hk > 0 && a->Hk < 65536 && a->Hq >= 0 &&
                    a->Hq < 65536 && a->num_blocks >= 0 && a->num_blocks < (1ll << 31),
                "kv_store_fp8: bad shape");
  if (a->tokens == 0) return MI355_OK;
  MI355_REQUIRE(a->k && a->v && a->slot_mapping, "kv_store_fp8: null pointer");
  MI355_REQUIRE(a->num_blocks == 0 || (a->k_cache && a->v_cache && a->k_scale && a->v_scale),
                "kv_store_fp8: null pointer");
  const int64_t strides[] = {a->k_st, a->k_sh, a->v_st, a->v_sh, a->kc_sb, a->kc_st, a->kc_sh, a->vc_sb,
                             a->vc_st, a->vc_sh, a->q_st, a->q_sh, a->qo_st, a->qo_sh};
  for (int64_t s : strides)
    MI355_REQUIRE(s % 8 == 0, "kv_store_fp8: strides must be multiples of 8 elements");
  MI355_REQUIRE(((uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q | (uintptr_t)a->q_out) % 16 == 0 &&
                    ((uintptr_t)a->k_cache | (uintptr_t)a->v_cache) % 8 == 0,
                "kv_store_fp8: rows must be 16-byte aligned (cache rows 8-byte)");
  const bool turn_keys = a->positions != nullptr;
  if (turn_keys &&
      !rope_args_ok("kv_store_fp8", a->D, a->rot_dim, a->inv_freq, a->positions, a->tokens))
    return MI355_EINVAL;
  MI355_REQUIRE(a->Hq == 0 || (turn_keys && a->q && a->q_out),
                "kv_store_fp8: queries need positions and both their pointers");
  const Rows q_in = head_rows(a->q, a->tokens, a->Hq, a->D, a->q_st, a->q_sh),
             q_to = head_rows(a->q_out, a->tokens, a->Hq, a->D, a->qo_st, a->qo_sh),
             k_in = head_rows(a->k, a->tokens, a->Hk, a->D, a->k_st, a->k_sh),
             v_in = head_rows(a->v, a->tokens, a->Hk, a->D, a->v_st, a->v_sh),
             kc = {a->k_cache, a->D, {a->num_blocks, a->block_size, a->Hk}, {a->kc_sb, a->kc_st, a->kc_sh}},
             vc = {a->v_cache, a->D, {a->num_blocks, a->block_size, a->Hk}, {a->vc_sb, a->vc_st, a->vc_sh}},
             ks = {a->k_scale, 4 * a->num_blocks * a->Hk, {1, 1, 1}, {0, 0, 0}},
             vs = {a->v_scale, 4 * a->num_blocks * a->Hk, {1, 1, 1}, {0, 0, 0}};
  MI355_REQUIRE(rows_distinct(q_to) && rows_distinct(kc) && rows_distinct(vc),
                "kv_store_fp8: rows of an output overlap each other");
  MI355_REQUIRE(same_or_apart(q_to, q_in) && rows_apart(q_to, k_in) && rows_apart(q_to, v_in),
                "kv_store_fp8: the queries' output overlaps keys, values or queries (and is not the same rows)");
  MI355_REQUIRE(rows_apart(kc, vc) && rows_apart(ks, vs), "kv_store_fp8: the caches or their scales overlap each other");
  StoreParams p;
  p.k = (const unsigned short*)a->k;
  p.v = (const unsigned short*)a->v;
  p.k_st = a->k_st; p.k_sh = a->k_sh; p.v_st = a->v_st; p.v_sh = a->v_sh;
  p.k_cache = (unsigned char*)a->k_cache;
  p.v_cache = (unsigned char*)a->v_cache;
  p.kc_sb = a->kc_sb; p.kc_st = a->kc_st; p.kc_sh = a->kc_sh;
  p.vc_sb = a->vc_sb; p.vc_st = a->vc_st; p.vc_sh = a->vc_sh;
  p.k_scale = a->k_scale;
  p.v_scale = a->v_scale;
  p.slots = a->slot_mapping;
  p.tokens = a->tokens;
  p.num_blocks = a->num_blocks;
  p.Hk = (int)a->Hk;
  p.lb = log2_of(a->block_size);
  // Threads for the rows that a run can have: 256 hold 64 rows of 128, 1024 hold 256.
  const int64_t rows = std::min(a->block_size, a->tokens), held = HELD * 256 * 8 / a->D;
  const int threads = rows > 2 * held ? 1024 : rows > held ? 512 : 256;
  // Tokens among which a workgroup looks for the beginning of a run: one for each of its waves while
  // there are few tokens (each may be a request of its own), then as many as keep the launch to about
  // twice the workgroups that the chip holds: most find no run where tokens follow each other, and
  // take a place for the while (4602 tokens of 12 prompts, 8 heads: groups of 64 43 us, of 32 53).
  const int64_t most = threads > 256 ? 1024 : 2048;
  p.group = threads / 64;
  while (p.group < 64 && (a->tokens + p.group - 1) / p.group * 2 * a->Hk > most) p.group *= 2;
  const int64_t units = (a->tokens + p.group - 1) / p.group * 2 * a->Hk;
  MI355_REQUIRE(units + a->tokens < (1ll << 31), "kv_store_fp8: too many tokens and heads for one call");
  p.kv_groups = (unsigned)units;
  // tokens of a workgroup that turns queries: with 256 threads two (8 x 600 tokens 37.8 us, one 39.6, four
  // 38.9), with more four (1842 tokens 24.9, one 29)
  p.q_group = a->tokens < 1024 ? 1 : threads > 256 ? 4 : 2;
  const unsigned q_groups = a->Hq ? (unsigned)((a->tokens + p.q_group - 1) / p.q_group) : 0;
  p.rope = Rope{a->positions, a->inv_freq, a->inv_freq_is_f64, (int)(a->rot_dim / 2), a->is_neox != 0,
                a->attn_factor};
  p.q = RopeRows{(const unsigned short*)a->q, (unsigned short*)a->q_out, a->q_st, a->q_sh, a->qo_st, a->qo_sh,
                 (int)a->Hq};
  const dim3 grid(p.kv_groups + q_groups);
  hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto threads) {
    constexpr int T = decltype(threads)::value;
    if (a->D == 128) hipLaunchKernelGGL((kv_store_kernel<128, T>), grid, dim3(T), 0, st, p);
    else hipLaunchKernelGGL((kv_store_kernel<64, T>), grid, dim3(T), 0, st, p);
  };
  if (threads == 1024) launch(std::integral_constant<int, 1024>{});
  else if (threads == 512) launch(std::integral_constant<int, 512>{});
  else launch(std::integral_constant<int, 256>{});
  MI355_CHECK_LAUNCH("kv_store_fp8");
  return MI355_OK;
}
