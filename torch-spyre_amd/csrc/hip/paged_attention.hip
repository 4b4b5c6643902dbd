// Attention of a step's new tokens over a paged KV cache: one decoded token per
// sequence, the tree of tokens that speculative decoding drafts, or a piece of a
// prompt, ragged over the batch.
//
// Sequence b holds len_b keys, the last n_b = starts[b + 1] - starts[b] of them
// its new tokens, whose queries are rows starts[b] ..; key x lies in page
// table[b][x / page] at x % page.  New token i sees the len_b - n_b keys before
// the step and of the new ones those that its mask row names (without a mask:
// those up to itself):
//
//   O = sum_x 2^(c s_x - m) v_x / sum_x 2^(c s_x - m),  s = q K^T, c = scale log2 e
//
// with a running maximum m and sum per row.  A row that sees nothing is 0, and so are rows
// that belong to no sequence.
//
// Layout of the work:
//   * A unit is (sequence, KV head, tile of rows): the G = H / Hkv query heads of
//     a KV head are rows of one tile (row r = new token r / G, head r % G), so K
//     and V are read once for all of them.  Where single tokens are decoded, a wave
//     takes 16 rows; the 4 waves of a workgroup take 1, 2 or 4 groups of rows, by the
//     rows that the sequence has, and split the keys 4, 2 or 1 ways.
//   * The lengths are known on the device only, so the launch has a fixed grid and
//     every workgroup works out its share: units cut into items of 128 keys,
//     an equal run of items for each workgroup.  A unit that ends up in several
//     workgroups leaves partial (m, l, O) in the workspace, which a second
//     kernel merges in a fixed order.  The same launch thus serves any
//     lengths (a captured graph's too).
//   * No LDS in that key loop.  S^T = K Q^T on 16x16x32 MFMAs: a lane's K
//     fragment is 16 bytes of a key row, loaded straight from the cache.  A lane then
//     holds scores of one query (column lane % 16) for keys 4 (lane / 16) + r,
//     which are the 8 values that O^T += V^T P^T wants from it, in registers:
//     the 32 slots of that product are the keys in the order {4 g + j, 16 + 4 g +
//     j}.  For V^T each lane loads D / 16 consecutive head dims of its 8 keys
//     (whole cache rows over 16 lanes) and turns the 8 x D / 16 block with byte
//     permutes; head dim D / 16 m + t is row m of the product's tile t.
//   * More tokens (128-row tiles, every wave 32 rows of its own) would ask the
//     caches for each key four times: their K and V pass through LDS, 64 keys a stage,
//     two stages, a row's 16-byte chunks swapped by the row's number so that
//     fragments are read without bank conflicts (V^T by transposing reads).
//   * A workgroup's next unit is looked up, and its first loads are under way, before
//     the results of the one before it leave.
//   * Probabilities round to the element type for the second product (the matrix cores take
//     both operands in one type): half a step of each key's share of O.  fp16 has that
//     step from 2^-14 on only and nothing below 2^-25, so there they are held 2^7 times as
//     large (at most 2^15, with 2^8 for a maximum that the reference does not follow; the
//     division by the sum, which holds the factor too, takes it out): half a step from 2^-21 of the
//     largest on, below it 2^-32 of the largest.  Scores, maxima, sums and O stay fp32; O rounds
//     once.
//
// What bounds it (32 query heads over 8 of 128): decoding and trees of one long sequence
// the bytes of K and V, 64 ragged sequences of up to 4000 keys 122 us (530 MB, 4.3
// TB/s), 131072 keys 105 us for a token and 115 for a tree of 16; four sequences of 1152
// keys the latency of two kernels, 18 us.  Pieces of prompts, 3 x 777 tokens over 2825 keys, 189 us
// (93 GFLOP, 24 us of it the merge), are bound by latency: scores, softmax and second product
// of a wave follow each other, two waves a SIMD, which issue vector instructions 40 % of the
// time and keep the matrix cores busy 25 %.  Whole prompts are bound by the planning: for each
// unit head_items and locate walk all tiles of a KV head, some 0.9 us a tile, 1.7 of the
// 2.06 ms of 8192 tokens and 0.27 of the 0.51 of four times 2048.
#include <algorithm>
#include <type_traits>

#include "gemm_common.h"

namespace sph {
namespace {

constexpr int PT = 256;                 // threads
constexpr int kItemKeys = 128;          // keys of one item
constexpr int kMaxSeqs = 4096;
constexpr int kMaxGrid = 512;             // two workgroups per CU
constexpr int kFewParts = 16;             // parts of a unit that one group of lanes merges
constexpr int32_t kPagedIndex = 3;      // error code: page, length or start out of range
constexpr float kLog2e = 1.4426950408889634f;
// s_waitcnt for vmcnt(0) alone (fields of gfx9: vmcnt [3:0] and [15:14], the others at their most)
constexpr int kWaitVmcnt0 = 0x0F70;

struct PagedArgs {
  const void* q;
  int64_t q_st, q_sh;
  const void* kc;
  int64_t k_sp, k_sh, k_ss;
  const void* vc;
  int64_t v_sp, v_sh, v_ss;
  const int64_t* table;
  int64_t ld_table, width, n_pages;
  int page;
  const int64_t* lens;
  const int64_t* starts;
  const uint8_t* mask;
  int64_t ld_mask;
  int mask_w;
  int64_t tokens;
  int batch, nkv, g;
  float scale_log2;
  void* o;        // [tokens, H, D]
  float* part;    // [grid][2] partial tiles
  int32_t* desc;  // [grid][8] the unit that begins in a workgroup and ends in another: tasks
                  // to merge it, workgroups, head, first row, rows, first token
  int32_t* err;
};

// The kernel's arguments, read again wherever they are asked for: held all
// through the key loop they would not fit the scalar registers, and came from vector
// registers and scratch memory instead (decoding 64 sequences 124 to 148 us).
typedef const __attribute__((address_space(4))) PagedArgs* ArgPtr;
__device__ inline ArgPtr args() {
  ArgPtr a = (ArgPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}

// Values that are the same in every lane, in scalar registers.
__device__ inline int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline int64_t uni(int64_t v) {
  const uint32_t lo = uni(static_cast<int>(v)), hi = uni(static_cast<int>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// What a workgroup has to know of one sequence.
struct Seq {
  int64_t start;
  int n, len, rows, rw, tiles;  // rw: groups of rows per workgroup
};

// Forms of the kernel: a wave takes 16 rows, or 32 of a 128-row tile whose keys pass through
// LDS.  Each serves any number.
enum { DECODE, WIDE };
constexpr int rows_of(int form) { return form == DECODE ? 16 : 32; }  // of a wave

template <int FORM>
__device__ inline Seq sequence(int b, bool report) {
  const ArgPtr p = args();
  const int64_t s0 = p->starts[b], s1 = p->starts[b + 1], len = p->lens[b];
  Seq s{s0, 0, 0, 0, 1, 0};
  if (s0 < 0 || s1 < s0 || s1 > p->tokens) {
    if (report && p->err != nullptr) *p->err = kPagedIndex;
    return s;
  }
  s.n = static_cast<int>(s1 - s0);
  const bool bad = len < s.n || len > p->width * p->page ||
                   (p->mask != nullptr && s.n > p->mask_w) || (s.n > 0 && p->n_pages == 0);
  s.len = bad ? 0 : static_cast<int>(len);
  if (bad && report && p->err != nullptr) *p->err = kPagedIndex;
  s.rows = s.n * p->g;
  constexpr int R = rows_of(FORM);
  s.rw = FORM == WIDE ? 4 : s.rows <= R ? 1 : s.rows <= 2 * R ? 2 : 4;
  s.tiles = (s.rows + R * s.rw - 1) / (R * s.rw);
  return s;
}
// (of a sequence that is the same in every lane)
__device__ inline Seq uni(const Seq& s) {
  return Seq{uni(s.start), uni(s.n), uni(s.len), uni(s.rows), uni(s.rw), uni(s.tiles)};
}

// Keys that the rows of a tile can see at most (causal: up to its last token).
template <int FORM>
__device__ inline int tile_keys(const Seq& s, int tile) {
  const ArgPtr p = args();
  if (p->mask != nullptr || s.len == 0) return s.len;
  const int last = min((tile + 1) * rows_of(FORM) * s.rw, s.rows) - 1;
  return s.len - s.n + last / p->g + 1;
}
template <int FORM>
__device__ inline int tile_items(const Seq& s, int tile) {
  return max(1, (tile_keys<FORM>(s, tile) + kItemKeys - 1) / kItemKeys);
}
// Items of one KV head of a sequence.
template <int FORM>
__device__ inline int64_t head_items(const Seq& s) {
  if (s.tiles <= 1 || args()->mask != nullptr)
    return s.tiles == 0 ? 0 : s.tiles * static_cast<int64_t>(tile_items<FORM>(s, 0));
  int64_t k = 0;
  for (int t = 0; t < s.tiles; ++t) k += tile_items<FORM>(s, t);
  return k;
}

__device__ inline float xor_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}

template <typename T>
__device__ inline bool not_finite(uint32_t two) {
  constexpr uint32_t e = __is_same(T, half_t) ? 0x7c00u : 0x7f80u;
  return (two & e) == e || ((two >> 16) & e) == e;
}

// Two floats rounded to the element type, lo in the low half.
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
template <typename T>
__device__ inline uint32_t pack2(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  if constexpr (__is_same(T, half_t))
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

typedef u32x2 u32x2_any __attribute__((aligned(2)));

// T, head dim, form, whether pages hold whole blocks of 16 keys.
template <typename T, int D, int FORM, bool P16>
__global__ void __launch_bounds__(PT) __attribute__((amdgpu_waves_per_eu(2)))
paged_attn_kernel(const PagedArgs) {
  constexpr int RT = FORM == DECODE ? 1 : 2;
  constexpr int KK = D / 32, DT = D / 16, R = 16 * RT, PITCH = D + 4;
  constexpr int VW = DT / 2;           // 32-bit words of a lane's share of a V row
  constexpr int KPB = P16 ? 16 : 1;    // keys per page look-up
  constexpr bool AHEAD = FORM == DECODE;  // (the others have no registers for it)
  constexpr int SK = 64, CPR = D / 8;  // keys of a stage, 16-byte chunks of a row
  constexpr int SR = PT / CPR, SP = SK / SR;  // rows and turns of a stage's loads
  constexpr int STAGE = SK * D * 2;    // bytes of a stage's K (or V)
  constexpr int MERGE = 4 * R * PITCH * 4, LDS = FORM == WIDE && 4 * STAGE > MERGE ? 4 * STAGE : MERGE;
  static_assert(SP <= KK, "a stage fits the registers of a step's keys");
  constexpr float kLift = __is_same(T, half_t) ? 7.f : 0.f;  // log2 of the probabilities' factor
  extern __shared__ int64_t prefix[];  // [batch + 1] items before a sequence
  __shared__ __attribute__((aligned(1024))) char lds[LDS];
  __shared__ float mg_m[4][R], mg_l[4][R];
  __shared__ int64_t scan[4];
  __shared__ uint8_t odd_rows[2][SK];  // keys of a stage with a value that is not finite
  auto merge = reinterpret_cast<float(*)[R][PITCH]>(lds);
  const int t = threadIdx.x, lane = t & 63;
  const int wave = uni(t >> 6);
  const int n16 = lane & 15, g4 = lane >> 4;
  // contiguous runs of workgroups to each of the 8 XCDs
  int wg = blockIdx.x;
  {
    const int total = gridDim.x, q = total >> 3, r = total & 7, x = wg & 7;
    wg = x * q + min(x, r) + (wg >> 3);
  }
  const int batch = args()->batch;
  // items before every sequence
  int64_t total = 0;
  for (int b0 = 0; b0 < batch; b0 += PT) {
    int64_t v = 0;
    if (b0 + t < batch) {
      const Seq s = sequence<FORM>(b0 + t, wg == 0);
      v = head_items<FORM>(s) * args()->nkv;
    }
    int64_t x = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t y = __shfl_up(x, off, 64);
      if (lane >= off) x += y;
    }
    if (lane == 63) scan[wave] = x;
    __syncthreads();
    int64_t base = total;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) base += scan[w];
      total += scan[w];
    }
    if (b0 + t < batch) prefix[b0 + t] = base + x - v;
    __syncthreads();
  }
  if (t == 0) {
    prefix[batch] = total;
    args()->desc[static_cast<int64_t>(wg) * 8] = 0;
  }
  __syncthreads();
  total = uni(total);
  const int64_t quota = uni(max(static_cast<int64_t>(1), (total + gridDim.x - 1) / gridDim.x));
  int64_t item = wg * quota;
  const int64_t end = min(item + quota, total);

  // The unit that holds an item, from there to its end or this workgroup's.
  struct Unit {
    Seq s;
    int b, h, tile, count;  // sequence, KV head, tile of rows, items of the tile
    int c0, c1, keys;       // this workgroup's items, keys that the tile's rows see at most
    int kbeg, kend, ctx;    // keys of the items, keys that every row sees
  };
  // (The compiler does not see that all of it is uniform across the loop.)
  auto scalar = [](const Unit& u) {
    return Unit{uni(u.s),    uni(u.b),  uni(u.h),    uni(u.tile), uni(u.count), uni(u.c0),
                uni(u.c1),   uni(u.keys), uni(u.kbeg), uni(u.kend), uni(u.ctx)};
  };
  auto locate = [&](int64_t at, int b) {
    Unit u;
    if (b < 0) {  // (the first: prefix[lo] <= at < prefix[hi])
      int lo = 0, hi = batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (uni(prefix[mid]) <= at) lo = mid;
        else hi = mid;
      }
      b = lo;
    }
    while (uni(prefix[b + 1]) <= at) ++b;
    u.b = b;
    u.s = uni(sequence<FORM>(b, false));
    const int64_t per_head = head_items<FORM>(u.s);
    int64_t rem = at - uni(prefix[b]);
    if (rem < per_head) {
      u.h = 0;
    } else if ((rem | per_head) >> 31 == 0) {
      u.h = uni(static_cast<int>(static_cast<uint32_t>(rem) / static_cast<uint32_t>(per_head)));
    } else {
      u.h = uni(static_cast<int>(rem / per_head));
    }
    rem -= u.h * per_head;
    u.tile = 0;
    u.count = tile_items<FORM>(u.s, 0);
    if (args()->mask != nullptr) {
      u.tile = rem < u.count ? 0 : uni(static_cast<int>(rem / u.count));
      rem -= static_cast<int64_t>(u.tile) * u.count;
    } else {
      while (rem >= u.count) {
        rem -= u.count;
        u.count = tile_items<FORM>(u.s, ++u.tile);
      }
    }
    u.c0 = static_cast<int>(rem);
    u.c1 = static_cast<int>(min(static_cast<int64_t>(u.count), u.c0 + (end - at)));
    u.keys = tile_keys<FORM>(u.s, u.tile);
    u.kbeg = u.c0 * kItemKeys;
    u.kend = min(u.keys, u.c1 * kItemKeys);
    u.ctx = u.s.len - u.s.n;
    return scalar(u);
  };
  auto step_of = [&](const Unit& u) { return FORM == WIDE ? SK : 32 * (4 / u.s.rw); };
  auto first_key = [&](const Unit& u) { return u.kbeg + 32 * (wave / u.s.rw); };  // of this wave (WIDE: 0)
  auto last_block = [&](const Unit& u) { return (max(u.keys, 1) - 1) / KPB; };
  // Page of the look-ups blk .. of a unit, one a lane.
  auto page_at = [&](const Unit& u, int blk) {
    const ArgPtr p = args();
    return p->table[u.b * p->ld_table + min(blk + lane, last_block(u)) * KPB / p->page];
  };
  // Those of its first keys.  (New tokens of a sequence that is out of range make a unit without
  // keys, for which nothing is looked up: the table may have no columns.)
  auto first_pages = [&](const Unit& u) {
    return u.keys > 0 ? page_at(u, first_key(u) / KPB) : int64_t{0};
  };

  u32x4 qf[RT][KK];
  int tok[RT];
  u32x4 kr[2][KK];
  uint32_t vr[8][VW];
  // Where a key's rows lie, in bytes from the head's first: lane l holds that of
  // 16-key block base + l (off P16: of key base + l); `ahead` are the pages after those.
  const char *Kh, *Vh;
  int base = 0;
  int64_t ko = 0, vo = 0, ahead = 0;
  auto turn_pages = [&](const Unit& u, int blk) {
    const ArgPtr p = args();
    base = blk;
    const int x = min(blk + lane, last_block(u)) * KPB;
    const bool ok = ahead >= 0 && ahead < p->n_pages;
    if (!ok && p->err != nullptr) *p->err = kPagedIndex;
    const int64_t pg = ok ? ahead : 0;
    const int at = x % p->page;
    ko = (pg * p->k_sp + at * p->k_ss) * 2;
    vo = (pg * p->v_sp + at * p->v_ss) * 2;
    ahead = page_at(u, blk + max(64, step_of(u) / KPB));
  };
  auto lane_of = [&](int64_t v, int i) {  // (i uniform)
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), i);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), i);
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
  };
  const uint32_t k_next = static_cast<uint32_t>(args()->k_ss) * 2;
  const uint32_t v_next = static_cast<uint32_t>(args()->v_ss) * 2;
  const uint32_t k_lane = (P16 ? n16 * k_next : 0u) + 16 * g4;
  const uint32_t v_lane = (P16 ? 4 * g4 * v_next : 0u) + 2 * DT * n16;
  // A step's 32 keys, as fragments.
  auto load_k = [&](const Unit& u, int kb) {
    const int last = last_block(u);
#pragma unroll
    for (int th = 0; th < 2; ++th) {
      const char* src;
      if constexpr (P16)
        src = Kh + lane_of(ko, min(kb / 16 + th, last) - base);
      else
        src = Kh + __shfl(ko, min(kb + 16 * th + n16, last) - base, 64);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        kr[th][kk] = *reinterpret_cast<const u32x4_any*>(src + k_lane + 64 * kk);
    }
  };
  auto load_v = [&](const Unit& u, int kb) {
    const int last = last_block(u);
#pragma unroll
    for (int th = 0; th < 2; ++th) {
      const char* src = Vh;
      if constexpr (P16) src += lane_of(vo, min(kb / 16 + th, last) - base);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* at = src;
        if constexpr (P16) at += j * v_next;
        else at += __shfl(vo, min(kb + 16 * th + 4 * g4 + j, last) - base, 64);
        at += v_lane;
        if constexpr (VW == 4) {
          const u32x4 w = *reinterpret_cast<const u32x4_any*>(at);
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[4 * th + j][e] = w[e];
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2_any*>(at);
          vr[4 * th + j][0] = w[0];
          vr[4 * th + j][1] = w[1];
        }
      }
    }
  };
  // A stage's 64 keys: this thread's chunk t % CPR of rows t / CPR + SR i, K in
  // kr[0], V in kr[1].
  const int srow = t / CPR, schunk = t % CPR;
  const uint32_t k_row = (P16 ? (srow & 15) * k_next : 0u) + 16 * schunk;
  const uint32_t v_row = (P16 ? (srow & 15) * v_next : 0u) + 16 * schunk;
  auto load_stage = [&](const Unit& u, int kb) {
    const int last = last_block(u);
#pragma unroll
    for (int i = 0; i < SP; ++i) {
      const char *k = Kh, *v = Vh;
      if constexpr (P16) {
        const int blk = min((kb + SR * i + uni(srow)) / 16, last) - base;
        k += lane_of(ko, blk);
        v += lane_of(vo, blk);
      } else {
        const int x = min(kb + srow + SR * i, last) - base;
        k += __shfl(ko, x, 64);
        v += __shfl(vo, x, 64);
      }
      kr[0][i] = *reinterpret_cast<const u32x4_any*>(k + k_row);
      kr[1][i] = *reinterpret_cast<const u32x4_any*>(v + v_row);
    }
  };
  // Queries of a unit and its first keys (its first pages are in `ahead`).
  auto begin = [&](const Unit& u) {
    const int row0 = u.tile * R * u.s.rw + (wave % u.s.rw) * R;
    const ArgPtr p = args();
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = min(row0 + 16 * i + n16, u.s.rows - 1);
      tok[i] = r / p->g;
      const T* q = static_cast<const T*>(p->q) + (u.s.start + tok[i]) * p->q_st +
                   static_cast<int64_t>(u.h * p->g + r % p->g) * p->q_sh;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        qf[i][kk] = *reinterpret_cast<const u32x4_any*>(q + 32 * kk + 8 * g4);
    }
    Kh = reinterpret_cast<const char*>(static_cast<const T*>(p->kc) + u.h * p->k_sh);
    Vh = reinterpret_cast<const char*>(static_cast<const T*>(p->vc) + u.h * p->v_sh);
    const int kb = first_key(u);
    if (kb < u.kend && (FORM == WIDE || row0 < u.s.rows)) {
      turn_pages(u, kb / KPB);
      if constexpr (FORM == WIDE) {
        load_stage(u, kb);
      } else {
        load_k(u, kb);
        load_v(u, kb);
      }
    }
  };

  Unit u{}, next{};
  if (item < end) {
    u = locate(item, -1);
    ahead = first_pages(u);
    begin(u);
  }
  while (item < end) {
    u = scalar(u);
    item = uni(item);
    const bool more_units = AHEAD && item + (u.c1 - u.c0) < end;
    int64_t ahead_next = 0;
    if (more_units) {
      next = locate(item + (u.c1 - u.c0), u.b);
      ahead_next = first_pages(next);
    }
    const int tile0 = u.tile * R * u.s.rw, row0 = tile0 + (wave % u.s.rw) * R;
    const int kend = u.kend, ctx = u.ctx;
    // Keys that all rows of this wave (of the tile) see: without a mask also new ones, up to the
    // first row's token.
    const bool masked = args()->mask != nullptr;
    const int seen = masked ? ctx : ctx + row0 / args()->g + 1;
    const int seen_tile = masked ? ctx : ctx + tile0 / args()->g + 1;
    f32x4 o[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float c = args()->scale_log2;

    // Scores of 32 keys from kb on that a row does not see.
    auto hide = [&](f32x4 (&sc)[RT][2], int kb) {
      const ArgPtr p = args();
      const int k0 = kb + 4 * g4;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        uint8_t named[8];
        if (p->mask != nullptr) {
          const uint8_t* mr = p->mask + (u.s.start + tok[i]) * p->ld_mask;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            named[j] = mr[max(0, min(k0 + 16 * (j >> 2) + (j & 3) - ctx, u.s.n - 1))];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) named[j] = k0 + 16 * (j >> 2) + (j & 3) - ctx <= tok[i];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = k0 + 16 * (j >> 2) + (j & 3);
          const bool see = key < kend && (key < ctx || named[j] != 0);
          sc[i][j >> 2][j & 3] = see ? sc[i][j >> 2][j & 3] : -INFINITY;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // Scores to probabilities, in place and as the fragment of the second product.
    auto softmax = [&](f32x4 (&sc)[2], int i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, sc[j >> 2][j & 3]);
      mx *= c;
      // the reference follows the maximum only when it is passed by more than
      // 8: a probability is then at most 2^8
      if (__ballot(mx > m[i] + 8.f) != 0) {
        mx = xor_max(mx);
        const float to = fmaxf(m[i], mx);
        const float a = m[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[i] - to);
        l[i] *= a;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[i][d] *= a;
        m[i] = to;
      }
      const float ref = m[i] == -INFINITY ? 0.f : kLift - m[i];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float pr = __builtin_amdgcn_exp2f(fmaf(sc[j >> 2][j & 3], c, ref));
        sc[j >> 2][j & 3] = pr;
        l[i] += pr;
      }
      u32x4 pf;
#pragma unroll
      for (int e = 0; e < 4; ++e) pf[e] = pack2<T>(sc[e >> 1][2 * (e & 1)], sc[e >> 1][2 * (e & 1) + 1]);
      return pf;
    };
    // Values that are not finite, of new keys that some rows do not see: a probability of
    // 0 would not cancel them in the product, so they were taken out of it and are
    // added here to the rows that see them.  bits: of the 32 keys from kb on; dim(d, r): where
    // o[.][d][r] lies.
    auto add_odd = [&](f32x4 (&sc)[RT][2], int kb, uint32_t bits, auto dim) {
#pragma unroll 1
      for (int x = 0; x < 32; ++x) {
        if ((bits >> x & 1u) == 0) continue;
        const ArgPtr p = args();
        const int key = kb + x, j = 4 * (x >> 4) + (x & 3);
        const int64_t pg = p->table[u.b * p->ld_table + key / p->page];
        const T* v = reinterpret_cast<const T*>(Vh) + (pg >= 0 && pg < p->n_pages ? pg : 0) * p->v_sp +
                     (key % p->page) * p->v_ss;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          float w = 0.f;
#pragma unroll
          for (int y = 0; y < 8; ++y) w = y == j ? sc[i][y >> 2][y & 3] : w;
          w = __shfl(w, n16 + 16 * (x >> 2 & 3), 64);
          if (w == 0.f) continue;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i][d][r] = fmaf(w, Num<T>::to_f(v[dim(d, r)]), o[i][d][r]);
            __builtin_amdgcn_sched_barrier(0);  // (few registers are left)
          }
        }
      }
    };

    // Queries and first keys have landed.  (Else the compiler waits for the queries where the
    // key loop uses them, in every step, and so for all loads in flight there.)
    __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
    if constexpr (FORM != WIDE) {
      const int step = step_of(u);
      int kb = first_key(u);
      // One step of 32 keys; EDGE: some of them are not seen by every row.  (The last step as a
      // third variant, so that the loads ahead are certain and the keys need not be
      // waited for together with the values, costs more in code than it saves.)
      auto one = [&](auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        f32x4 sc[RT][2];
#pragma unroll
        for (int th = 0; th < 2; ++th)
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) a = mfma16<T>(kr[th][kk], qf[i][kk], a);
            sc[i][th] = a;
          }
        const bool more = kb + step < kend;
        uint32_t bits = 0;
        if constexpr (EDGE) {
          hide(sc, kb);
          // (slots past the end may hold anything, too)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = kb + 4 * g4 + 16 * (j >> 2) + (j & 3);
            bool bad = false;
#pragma unroll
            for (int e = 0; e < VW; ++e) bad = bad || not_finite<T>(vr[j][e]);
            bad = bad && key < kend && key >= seen;
            const uint64_t all = __ballot(bad);  // (16 lanes hold a key)
#pragma unroll
            for (int g = 0; g < 4; ++g)
              bits |= ((all >> 16 * g & 0xffffu) != 0 ? 1u : 0u) << (16 * (j >> 2) + 4 * g + (j & 3));
            const bool drop = key >= kend || (all >> (16 * g4) & 0xffffu) != 0;
#pragma unroll
            for (int e = 0; e < VW; ++e) vr[j][e] = drop ? 0u : vr[j][e];
          }
        }
        if (more) {
          if (kb + step + 32 > (base + 64) * KPB) turn_pages(u, (kb + step) / KPB);
          load_k(u, kb + step);
        }
        __builtin_amdgcn_sched_barrier(0);
        u32x4 pf[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) pf[i] = softmax(sc[i], i);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          // dims DT n16 + d of this lane's 8 keys
          u32x4 vf;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            vf[e] = __builtin_amdgcn_perm(vr[2 * e + 1][d >> 1], vr[2 * e][d >> 1],
                                          d & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int i = 0; i < RT; ++i) o[i][d] = mfma16<T>(vf, pf[i], o[i][d]);
        }
        if constexpr (EDGE) {
          if (bits != 0) add_odd(sc, kb, bits, [&](int d, int r) { return DT * (4 * g4 + r) + d; });
        }
        if (more) load_v(u, kb + step);
        __builtin_amdgcn_sched_barrier(0);
        kb += step;
      };
      if (row0 < u.s.rows) {
        while (kb + 32 <= min(kend, seen)) one(std::false_type{});
        while (kb < kend) one(std::true_type{});
      }
    } else {
      // Stages of 64 keys in LDS: [stage][K, V][key][chunk ^ key].
      static_assert(SR % CPR == 0, "a turn further, the swap is the same");
      const int put_at = (srow * CPR + (schunk ^ (srow & (CPR - 1)))) * 16;
      auto put = [&](int kb, int slot) {
        char* to = lds + slot * 2 * STAGE;
        const bool edge = kb + SK > seen_tile || kb + SK > kend;
#pragma unroll
        for (int i = 0; i < SP; ++i) {
          const int row = srow + SR * i, at = put_at + SR * i * CPR * 16;
          u32x4 v = kr[1][i];
          if (edge) {
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) bad = bad || not_finite<T>(v[e]);
            bad = bad && kb + row < kend && kb + row >= seen_tile;
            bad = (__ballot(bad) >> (lane & ~(CPR - 1)) & ((1ull << CPR) - 1)) != 0;
            if (schunk == 0) odd_rows[slot][row] = bad;
            if (bad || kb + row >= kend) v = u32x4{0u, 0u, 0u, 0u};
          }
          *reinterpret_cast<u32x4*>(to + at) = kr[0][i];
          *reinterpret_cast<u32x4*>(to + STAGE + at) = v;
        }
      };
      auto fetch = [&](int kb) {
        if (kb >= kend) return;
        if (kb + SK > (base + 64) * KPB) turn_pages(u, kb / KPB);
        load_stage(u, kb);
      };
      // Fragments' places in a stage: the lane's row and swapped chunk; what is added to
      // the row (16, 32) does not change the swap.
      uint32_t k_at[KK], v_at[DT];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        k_at[kk] = (n16 * CPR + ((4 * kk + g4) ^ (n16 & (CPR - 1)))) * 16;
      // V^T of dims 16 d .., keys 4 g4 + (0 .. 3): lane 4 e + q of 16 points at row e,
      // values 4 q ..
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int row = 4 * g4 + (n16 >> 2), q = n16 & 3;
        v_at[d] = (row * CPR + ((2 * d + (q >> 1)) ^ (row & (CPR - 1)))) * 16 + 8 * (q & 1);
      }
      const bool here = row0 < u.s.rows;
      __syncthreads();  // (the buffer is the merge's, too)
      if (u.kbeg < kend) put(u.kbeg, 0);
      fetch(u.kbeg + SK);
      __syncthreads();
      for (int kb0 = u.kbeg, slot = 0; kb0 < kend; kb0 += SK, slot ^= 1) {
        if (here) {
#pragma unroll 1
          for (int sub = 0; sub < 2; ++sub) {
            const int kb = kb0 + 32 * sub;
            if (kb >= kend) break;
            const char* sk = lds + slot * 2 * STAGE + 32 * sub * D * 2;
            const SPH_LDS char* sv = (const SPH_LDS char*)(sk + STAGE);
            f32x4 sc[RT][2];
#pragma unroll
            for (int th = 0; th < 2; ++th) {
              u32x4 kf[KK];
#pragma unroll
              for (int kk = 0; kk < KK; ++kk)
                kf[kk] = *reinterpret_cast<const u32x4*>(sk + k_at[kk] + 16 * th * D * 2);
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) a = mfma16<T>(kf[kk], qf[i][kk], a);
                sc[i][th] = a;
              }
            }
            if (kb + 32 > seen || kb + 32 > kend) hide(sc, kb);
            u32x4 pf[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) pf[i] = softmax(sc[i], i);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              u32x2 half[2];  // keys 4 g4 .. and 16 more
#pragma unroll
              for (int th = 0; th < 2; ++th)
                half[th] = __builtin_bit_cast(
                    u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                               (SPH_LDS s16x4*)(sv + v_at[d] + 16 * th * D * 2)));
              const u32x4 vf = __builtin_shufflevector(half[0], half[1], 0, 1, 2, 3);
#pragma unroll
              for (int i = 0; i < RT; ++i) o[i][d] = mfma16<T>(vf, pf[i], o[i][d]);
            }
            if (kb + 32 > seen_tile) {
              const uint32_t bits =
                  static_cast<uint32_t>(__ballot(odd_rows[slot][32 * sub + (lane & 31)] != 0));
              if (bits != 0) add_odd(sc, kb, bits, [&](int d, int r) { return 16 * d + 4 * g4 + r; });
            }
          }
        }
        if (kb0 + SK < kend) put(kb0 + SK, slot ^ 1);
        fetch(kb0 + 2 * SK);
        __syncthreads();
      }
    }

    // The waves' states meet in LDS: rows of wave group wave % rw, from 4 / rw waves.
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      l[i] += __shfl_xor(l[i], 16, 64);
      l[i] += __shfl_xor(l[i], 32, 64);
      const int r = 16 * i + n16;
      if (g4 == 0) {
        mg_m[wave][r] = m[i];
        mg_l[wave][r] = l[i];
      }
      if constexpr (FORM == WIDE) {
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&merge[wave][r][16 * d + 4 * g4]) = o[i][d];
      } else {
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
#pragma unroll
          for (int d = 0; d < DT; d += 4)
            *reinterpret_cast<f32x4*>(&merge[wave][r][DT * (4 * g4 + rr) + d]) =
                f32x4{o[i][d][rr], o[i][d + 1][rr], o[i][d + 2][rr], o[i][d + 3][rr]};
      }
    }
    if (more_units) {
      ahead = ahead_next;
      begin(next);
    }
    __syncthreads();
    const bool whole = u.c0 == 0 && u.c1 == u.count;
    const int rw = u.s.rw, kw = 4 / rw;
    const int live = min(R * rw, u.s.rows - tile0);
    const ArgPtr p = args();
    float* slot = p->part + (static_cast<int64_t>(wg) * 2 + (u.c0 > 0 ? 0 : 1)) * (4 * R) * (D + 4);
    constexpr int LR = D / 8, RP = PT / LR;  // lanes per row, rows at a time
#pragma unroll 1
    for (int r = t / LR; r < live; r += RP) {
      const int w0 = r / R, rr = r % R, cc = (t % LR) * 8;
      float M = -INFINITY, sum = 0.f, acc[8] = {};
      for (int k = 0; k < kw; ++k) M = fmaxf(M, mg_m[w0 + k * rw][rr]);
      for (int k = 0; k < kw; ++k) {
        const int w = w0 + k * rw;
        if (mg_m[w][rr] == -INFINITY && mg_l[w][rr] == 0.f) continue;  // saw nothing
        const float a = __builtin_amdgcn_exp2f(mg_m[w][rr] - (M == -INFINITY ? 0.f : M));
        sum = fmaf(a, mg_l[w][rr], sum);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(a, merge[w][rr][cc + e], acc[e]);
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= inv;
        const int row = tile0 + r;
        store8u<T>(static_cast<T*>(p->o) +
                       ((u.s.start + row / p->g) * p->nkv * p->g + u.h * p->g + row % p->g) * D + cc,
                   acc);
      } else {
        float* to = slot + r * (D + 4);
        if (cc == 0) {
          to[0] = M;
          to[1] = sum;
        }
        store8<float>(to + 4 + cc, acc);
      }
    }
    if (t == 0 && u.c0 == 0 && u.c1 < u.count) {
      // this workgroup holds the unit's beginning: the merge kernel finds here what it needs
      int32_t* d = p->desc + static_cast<int64_t>(wg) * 8;
      const int parts = static_cast<int>((item + u.count - 1) / quota - wg) + 1;
      d[0] = parts > kFewParts ? live : (live + 7) / 8;  // rows, or groups of 8, to merge
      d[1] = parts;
      d[2] = u.h;
      d[3] = tile0;
      d[4] = live;
      d[5] = static_cast<int32_t>(u.s.start);
    }
    item += u.c1 - u.c0;
    if constexpr (AHEAD) {
      u = next;
    } else if (item < end) {
      u = locate(item, u.b);
      ahead = first_pages(u);
      begin(u);
    }
    __syncthreads();
  }

  {  // rows that belong to no sequence
    const ArgPtr p = args();
    const int64_t none = 0;
    const int64_t before = min(max(p->starts[0], none), p->tokens);
    const int64_t behind = min(max(p->starts[batch], none), p->tokens);
    const int64_t rest = before + p->tokens - behind;
    const int64_t width = static_cast<int64_t>(p->g) * p->nkv * D;
    for (int64_t x = wg; x < rest; x += gridDim.x) {
      T* o = static_cast<T*>(p->o) + (x < before ? x : behind + x - before) * width;
      const float z[8] = {};
      for (int64_t c = t * 8; c < width; c += PT * 8) store8u<T>(o + c, z);
    }
  }
}

// Units that several workgroups hold: the one in which a unit begins has its first part
// in its second slot, those behind it have theirs in their first.  8 groups of D / 4
// lanes: with few parts each takes a row, else all of them one row, a run of the parts
// each, always in the same order.  Every workgroup looks all of them up and takes
// its turn.  (Two workgroups per unit and a row per wave took 180 of 330 us for one
// sequence of 131072 keys with 16 new tokens: 8 units of 64 parts and 64 rows.)
template <typename T, int D, int FORM>
__global__ void __launch_bounds__(PT) paged_attn_merge(const PagedArgs p, int grid) {
  constexpr int R4 = 4 * rows_of(FORM), L = D / 4, NB = 8;
  constexpr int G8 = 8;  // groups of lanes
  __shared__ int first[kMaxGrid + 1];  // tasks before a workgroup's
  __shared__ int info[kMaxGrid][5];
  __shared__ int scan[4];
  __shared__ float ms[G8], ls[G8];
  __shared__ __attribute__((aligned(16))) float os[G8][D];
  const int t = threadIdx.x, lane = t & 63, wave = uni(t >> 6);
  int total = 0;
  for (int g0 = 0; g0 < grid; g0 += PT) {
    int v = 0;
    if (g0 + t < grid) {
      const int32_t* d = p.desc + static_cast<int64_t>(g0 + t) * 8;
      v = d[0];
#pragma unroll
      for (int i = 0; i < 5; ++i) info[g0 + t][i] = d[1 + i];
    }
    int x = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(x, off, 64);
      if (lane >= off) x += y;
    }
    if (lane == 63) scan[wave] = x;
    __syncthreads();
    int base = total;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) base += scan[w];
      total += scan[w];
    }
    if (g0 + t < grid) first[g0 + t] = base + x - v;
    __syncthreads();
  }
  total = uni(total);
  const int g = t / L, c = (t % L) * 4;  // (D = 64: 16 groups, the last 8 idle)
  for (int task = blockIdx.x; task < total; task += gridDim.x) {
    int lo = 0, hi = grid;  // the last workgroup with first <= task: it has tasks
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (uni(first[mid]) <= task) lo = mid;
      else hi = mid;
    }
    const int parts = uni(info[lo][0]), h = info[lo][1], tile0 = info[lo][2], live = info[lo][3];
    const bool few = parts <= kFewParts;
    const int r = (task - uni(first[lo])) * (few ? 8 : 1) + (few ? g : 0);
    const int k0 = few ? 0 : g, dk = few ? 1 : G8;
    float M = -INFINITY, sum = 0.f, acc[4] = {};
    const bool mine = g < G8 && r < live;
    if (mine) {
      for (int k1 = k0; k1 < parts; k1 += dk * NB) {
        float m[NB], l[NB];
        f32x4 o[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const int at = min(k1 + dk * k, parts - 1);
          const int64_t slot = (static_cast<int64_t>(lo) + at) * 2 + (at == 0 ? 1 : 0);
          const float* x = p.part + (slot * R4 + r) * (D + 4);
          m[k] = x[0];
          l[k] = x[1];
          o[k] = *reinterpret_cast<const f32x4*>(x + 4 + c);
        }
        float to = M;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          if (k1 + dk * k >= parts) {
            m[k] = -INFINITY;
            l[k] = 0.f;
          }
          to = fmaxf(to, m[k]);
        }
        const float ref = to == -INFINITY ? 0.f : to;
        const float a = M == -INFINITY ? (sum == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(M - ref);
        sum *= a;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] *= a;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          if (m[k] == -INFINITY && l[k] == 0.f) continue;  // saw nothing
          const float w = __builtin_amdgcn_exp2f(m[k] - ref);
          sum = fmaf(w, l[k], sum);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, o[k][e], acc[e]);
        }
        M = to;
      }
    }
    if (!few) {
      if (g < G8) {
        if (c == 0) {
          ms[g] = M;
          ls[g] = sum;
        }
        *reinterpret_cast<f32x4*>(&os[g][c]) = f32x4{acc[0], acc[1], acc[2], acc[3]};
      }
      __syncthreads();
      M = -INFINITY;
      for (int k = 0; k < G8; ++k) M = fmaxf(M, ms[k]);
      const float ref = M == -INFINITY ? 0.f : M;
      sum = 0.f;
      for (int e = 0; e < 4; ++e) acc[e] = 0.f;
      for (int k = 0; k < G8; ++k) {
        if (ms[k] == -INFINITY && ls[k] == 0.f) continue;
        const float a = __builtin_amdgcn_exp2f(ms[k] - ref);
        sum = fmaf(a, ls[k], sum);
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(a, os[k][c + e], acc[e]);
      }
      __syncthreads();
    }
    if (mine && (few || g == 0)) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int at = tile0 + r;
      T* to = static_cast<T*>(p.o) + ((static_cast<int64_t>(info[lo][4]) + at / p.g) * p.nkv * p.g +
                                      h * p.g + at % p.g) * D + c;
      u32x2 w;
      w[0] = pack2<T>(acc[0] * inv, acc[1] * inv);
      w[1] = pack2<T>(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<u32x2_any*>(to) = w;
    }
  }
}

// The host knows how many tokens come, not whose they are.  One a sequence at most: the form
// for them (64 ragged sequences of up to 4000 keys 123 us, 142 in the other; as many heads of
// keys as of queries 100 and 104; 131072 keys 105 and 110).  More are trees or pieces of
// prompts, perhaps among single tokens: 16 tokens of 131072 keys take 183 and 115, 63 single tokens
// beside a piece of 40 / 150 / 512 / 900 (2000 keys each) 145 / 206 / 261 / 333 and 113 / 125 /
// 153 / 180.  Where every sequence brings 2 to 4 tokens the form for single ones would be
// ahead: 64 ragged ones of 2 127 and 150, of 4 132 and 165, of 6 160 and 170.
int form_of(int64_t tokens, int64_t batch, int64_t g) {
  return tokens <= batch && g <= 16 ? DECODE : WIDE;
}
// Workgroups: what the chip holds at once, or fewer when the shapes cannot hold as many items.
int64_t paged_grid(int64_t tokens, int64_t batch, int64_t n_kv, int64_t g, int64_t max_keys) {
  const int64_t tiles = std::min(tokens, tokens * g / rows_of(form_of(tokens, batch, g)) + batch);
  const double items = static_cast<double>(tiles) * n_kv *
                       static_cast<double>(std::max<int64_t>(1, ceil_div(max_keys, kItemKeys)));
  return items < kMaxGrid ? std::max<int64_t>(1, static_cast<int64_t>(items)) : kMaxGrid;
}
int64_t paged_part_floats(int64_t tokens, int64_t batch, int64_t g, int64_t head_dim) {
  return 2 * 4 * rows_of(form_of(tokens, batch, g)) * (head_dim + 4);
}

}  // namespace
}  // namespace sph

extern "C" int64_t sph_paged_attention_workspace_bytes(int64_t tokens, int64_t batch,
                                                       int64_t n_heads, int64_t n_kv_heads,
                                                       int64_t head_dim, int64_t max_keys) {
  using namespace sph;
  if (tokens <= 0 || batch <= 0 || n_kv_heads <= 0 || n_heads < n_kv_heads || head_dim <= 0 ||
      max_keys < 0)
    return 0;
  const int64_t g = n_heads / n_kv_heads;
  const int64_t grid = paged_grid(tokens, batch, n_kv_heads, g, max_keys);
  return grid * 32 + grid * paged_part_floats(tokens, batch, g, head_dim) * 4;
}

extern "C" int sph_paged_attention(
    sph_dtype dtype, int64_t tokens, int64_t batch, int64_t n_heads, int64_t n_kv_heads,
    int64_t head_dim, const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k_cache,
    int64_t k_stride_p, int64_t k_stride_h, int64_t k_stride_s, const void* v_cache,
    int64_t v_stride_p, int64_t v_stride_h, int64_t v_stride_s, int64_t n_pages, int64_t page_size,
    const int64_t* block_table, int64_t ld_table, int64_t table_width, const int64_t* seq_lens,
    const int64_t* q_starts, const uint8_t* mask, int64_t ld_mask, int64_t mask_width, float scale,
    void* o, void* workspace, int64_t workspace_bytes, int32_t* error_word, sph_stream_t stream) {
  using namespace sph;
  SPH_REQUIRE(dtype == SPH_F16 || dtype == SPH_BF16, SPH_ERR_UNSUPPORTED,
              "paged attention: dtype must be F16 or BF16");
  SPH_REQUIRE(head_dim == 64 || head_dim == 128, SPH_ERR_UNSUPPORTED,
              "paged attention: head_dim must be 64 or 128");
  SPH_REQUIRE(tokens >= 0 && batch >= 0 && n_heads > 0 && n_kv_heads > 0 && n_pages >= 0 &&
                  page_size > 0 && table_width >= 0 && mask_width >= 0,
              SPH_ERR_INVALID_ARG, "paged attention: bad sizes");
  SPH_REQUIRE(n_heads % n_kv_heads == 0, SPH_ERR_UNSUPPORTED,
              "paged attention: query heads must be a multiple of the KV heads");
  SPH_REQUIRE(scale > 0.f && scale < INFINITY, SPH_ERR_INVALID_ARG,
              "paged attention: scale must be positive and finite");
  if (tokens == 0) return SPH_OK;
  SPH_REQUIRE(batch > 0, SPH_ERR_INVALID_ARG, "paged attention: tokens without sequences");
  SPH_REQUIRE(batch <= kMaxSeqs, SPH_ERR_TOO_LARGE, "paged attention: at most 4096 sequences");
  SPH_REQUIRE(n_heads < (1 << 20) && tokens < (1LL << 24) && tokens * n_heads < (1LL << 26),
              SPH_ERR_TOO_LARGE, "paged attention: at most 2^26 query rows");
  SPH_REQUIRE(page_size < (1LL << 30) && n_pages < (1LL << 31) && table_width < (1LL << 30) &&
                  table_width * page_size < (1LL << 30),
              SPH_ERR_TOO_LARGE, "paged attention: at most 2^30 keys a sequence, 2^31 pages");
  SPH_REQUIRE(k_stride_s >= 0 && v_stride_s >= 0 && k_stride_s < (1 << 26) && v_stride_s < (1 << 26),
              SPH_ERR_TOO_LARGE, "paged attention: rows of a page at most 2^26 elements apart");
  SPH_REQUIRE(q != nullptr && o != nullptr && seq_lens != nullptr && q_starts != nullptr &&
                  (block_table != nullptr || table_width == 0) &&
                  ((k_cache != nullptr && v_cache != nullptr) || n_pages == 0),
              SPH_ERR_INVALID_ARG, "paged attention: null pointer");
  SPH_REQUIRE(mask == nullptr || (mask_width < (1LL << 30) && (tokens == 1 || ld_mask >= mask_width)),
              SPH_ERR_INVALID_ARG, "paged attention: mask rows overlap");
  const int64_t max_keys = table_width * page_size;
  const int64_t need = sph_paged_attention_workspace_bytes(tokens, batch, n_heads, n_kv_heads,
                                                           head_dim, max_keys);
  SPH_REQUIRE(workspace != nullptr && workspace_bytes >= need &&
                  reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
              SPH_ERR_INVALID_ARG, "paged attention: workspace too small or not 16-byte aligned");
  const int64_t g = n_heads / n_kv_heads;
  const int form = form_of(tokens, batch, g);
  const int64_t grid = paged_grid(tokens, batch, n_kv_heads, g, max_keys);
  PagedArgs a{};
  a.q = q;
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.kc = k_cache;
  a.k_sp = k_stride_p;
  a.k_sh = k_stride_h;
  a.k_ss = k_stride_s;
  a.vc = v_cache;
  a.v_sp = v_stride_p;
  a.v_sh = v_stride_h;
  a.v_ss = v_stride_s;
  a.table = block_table;
  a.ld_table = ld_table;
  a.width = table_width;
  a.n_pages = n_pages;
  a.page = static_cast<int>(page_size);
  a.lens = seq_lens;
  a.starts = q_starts;
  a.mask = mask;
  a.ld_mask = ld_mask;
  a.mask_w = static_cast<int>(mask_width);
  a.tokens = tokens;
  a.batch = static_cast<int>(batch);
  a.nkv = static_cast<int>(n_kv_heads);
  a.g = static_cast<int>(g);
  a.scale_log2 = scale * kLog2e;
  a.o = o;
  a.desc = static_cast<int32_t*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + grid * 32);
  a.err = error_word;
  hipStream_t st = as_stream(stream);
  const unsigned mgrid = static_cast<unsigned>(std::min<int64_t>(1024, tokens * n_heads));
  const size_t lds = static_cast<size_t>(batch + 1) * 8;
  auto go = [&](auto tt, auto dd, auto rr, auto pp) {
    using T = decltype(tt);
    constexpr int D = decltype(dd)::value, FORM = decltype(rr)::value;
    paged_attn_kernel<T, D, FORM, decltype(pp)::value><<<dim3(grid), PT, lds, st>>>(a);
    if (grid > 1) paged_attn_merge<T, D, FORM><<<dim3(mgrid), PT, 0, st>>>(a, static_cast<int>(grid));
  };
  auto by_page = [&](auto tt, auto dd, auto rr) {
    if (page_size % 16 == 0) go(tt, dd, rr, std::true_type{});
    else go(tt, dd, rr, std::false_type{});
  };
  auto by_rows = [&](auto tt, auto dd) {
    if (form == DECODE) by_page(tt, dd, std::integral_constant<int, DECODE>{});
    else by_page(tt, dd, std::integral_constant<int, WIDE>{});
  };
  auto by_dim = [&](auto tt) {
    if (head_dim == 128) by_rows(tt, std::integral_constant<int, 128>{});
    else by_rows(tt, std::integral_constant<int, 64>{});
  };
  if (dtype == SPH_F16) by_dim(half_t{});
  else by_dim(bf16_t{});
  return check_launch("sph_paged_attention");
}
