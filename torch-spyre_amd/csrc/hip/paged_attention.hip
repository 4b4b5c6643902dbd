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
//     and V are read once for all of them.  A wave takes 16 RT rows; the 4 waves of
//     a workgroup take RW = 1, 2 or 4 groups of rows, by the rows that the
//     sequence has, and split the keys 4 / RW ways.
//   * The lengths are known on the device only, so the launch has a fixed grid and
//     every workgroup works out its share: units cut into items of 128 keys,
//     an equal run of items for each workgroup.  A unit that ends up in several
//     workgroups leaves partial (m, l, O) in the workspace, which a second
//     kernel merges in a fixed order.  The same launch thus serves any
//     lengths (a captured graph's too).
//   * No LDS in the key loop.  S^T = K Q^T on 16x16x32 MFMAs: a lane's K
//     fragment is 16 bytes of a key row, loaded straight from the cache.  A lane then
//     holds scores of one query (column lane % 16) for keys 4 (lane / 16) + r,
//     which are the 8 values that O^T += V^T P^T wants from it, in registers:
//     the 32 slots of that product are the keys in the order {4 g + j, 16 + 4 g +
//     j}.  For V^T each lane loads D / 16 consecutive head dims of its 8 keys
//     (whole cache rows over 16 lanes) and turns the 8 x D / 16 block with byte
//     permutes; head dim D / 16 m + t is row m of the product's tile t.
//   * Probabilities round to the element type for the second product; scores,
//     maxima, sums and O stay fp32; O rounds once.
#include <algorithm>

#include "gemm_common.h"

namespace sph {
namespace {

constexpr int PT = 256;                 // threads
constexpr int kItemKeys = 128;          // keys of one item
constexpr int kMaxSeqs = 4096;
constexpr int32_t kPagedIndex = 3;      // error code: page, length or start out of range
constexpr float kLog2e = 1.4426950408889634f;

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
  int32_t* desc;  // [grid][8]
  int32_t* err;
};

// What a workgroup has to know of one sequence.
struct Seq {
  int64_t start;
  int n, len, rows, rw, tiles;  // rw: groups of rows per workgroup
};

template <int RT>
__device__ inline Seq sequence(const PagedArgs& p, int b, bool report) {
  const int64_t s0 = p.starts[b], s1 = p.starts[b + 1], len = p.lens[b];
  Seq s{s0, 0, 0, 0, 1, 0};
  if (s0 < 0 || s1 < s0 || s1 > p.tokens) {
    if (report && p.err != nullptr) *p.err = kPagedIndex;
    return s;
  }
  s.n = static_cast<int>(s1 - s0);
  const bool bad = len < s.n || len > p.width * p.page || (p.mask != nullptr && s.n > p.mask_w) ||
                   (len > 0 && p.n_pages == 0);
  s.len = bad ? 0 : static_cast<int>(len);
  if (bad && report && p.err != nullptr) *p.err = kPagedIndex;
  s.rows = s.n * p.g;
  constexpr int R = 16 * RT;
  s.rw = s.rows <= R ? 1 : s.rows <= 2 * R ? 2 : 4;
  s.tiles = (s.rows + R * s.rw - 1) / (R * s.rw);
  return s;
}

// Keys that the rows of a tile can see at most (causal: up to its last token).
template <int RT>
__device__ inline int tile_keys(const PagedArgs& p, const Seq& s, int tile) {
  if (p.mask != nullptr) return s.len;
  const int last = min((tile + 1) * 16 * RT * s.rw, s.rows) - 1;
  return s.len == 0 ? 0 : s.len - s.n + last / p.g + 1;
}
template <int RT>
__device__ inline int tile_items(const PagedArgs& p, const Seq& s, int tile) {
  return max(1, (tile_keys<RT>(p, s, tile) + kItemKeys - 1) / kItemKeys);
}
// Items of one KV head of a sequence.
template <int RT>
__device__ inline int64_t head_items(const PagedArgs& p, const Seq& s) {
  int64_t k = 0;
  if (p.mask != nullptr) return s.tiles * static_cast<int64_t>(s.tiles ? tile_items<RT>(p, s, 0) : 0);
  for (int t = 0; t < s.tiles; ++t) k += tile_items<RT>(p, s, t);
  return k;
}

// Values that are the same in every lane, in scalar registers.
__device__ inline int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline int64_t uni(int64_t v) {
  const uint32_t lo = uni(static_cast<int>(v)), hi = uni(static_cast<int>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
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

// (uniform) index of a 16-key block's page and the position in it, for 64 blocks at once:
// lane l holds block first + l.
struct Blocks {
  int page, at;
};
__device__ inline Blocks blocks(const PagedArgs& p, const int64_t* row, int first, int last) {
  const int x = min(first + static_cast<int>(threadIdx.x & 63), last) * 16;
  Blocks b;
  const int i = x / p.page;
  const int64_t pg = row[i];
  const bool ok = pg >= 0 && pg < p.n_pages;
  if (!ok && p.err != nullptr) *p.err = kPagedIndex;
  b.page = ok ? static_cast<int>(pg) : 0;
  b.at = x - i * p.page;
  return b;
}

// T, head dim, groups of 16 rows per wave, whether pages hold whole blocks of 16 keys.
template <typename T, int D, int RT, bool P16>
__global__ void __launch_bounds__(PT) paged_attn_kernel(const PagedArgs p) {
  constexpr int KK = D / 32, DT = D / 16, R = 16 * RT, PITCH = D + 4;
  constexpr int VW = DT / 2;  // 32-bit words of a lane's share of a V row
  extern __shared__ int64_t prefix[];  // [batch + 1] items before a sequence
  __shared__ __attribute__((aligned(16))) float merge[4][R][PITCH];
  __shared__ float mg_m[4][R], mg_l[4][R];
  __shared__ int64_t scan[4];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n16 = lane & 15, g4 = lane >> 4;
  // contiguous runs of workgroups to each of the 8 XCDs
  int wg = blockIdx.x;
  {
    const int total = gridDim.x, q = total >> 3, r = total & 7, x = wg & 7;
    wg = x * q + min(x, r) + (wg >> 3);
  }

  // rows that belong to no sequence
  const int64_t before = min(max(p.starts[0], static_cast<int64_t>(0)), p.tokens);
  const int64_t behind = min(max(p.starts[p.batch], static_cast<int64_t>(0)), p.tokens);
  {
    const int64_t rest = before + p.tokens - behind;
    const int chunks = p.g * p.nkv * D / 8;
    for (int64_t x = wg; x < rest; x += gridDim.x) {
      T* o = static_cast<T*>(p.o) + (x < before ? x : behind + x - before) * p.g * p.nkv * D;
      const float z[8] = {};
      for (int c = t; c < chunks; c += PT) store8u<T>(o + c * 8, z);
    }
  }

  // items before every sequence
  int64_t total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += PT) {
    int64_t v = 0;
    if (b0 + t < p.batch) {
      const Seq s = sequence<RT>(p, b0 + t, wg == 0);
      v = head_items<RT>(p, s) * p.nkv;
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
    if (b0 + t < p.batch) prefix[b0 + t] = base + x - v;
    __syncthreads();
  }
  if (t == 0) prefix[p.batch] = total;
  __syncthreads();
  total = uni(total);
  const int64_t quota = uni(max(static_cast<int64_t>(1), (total + gridDim.x - 1) / gridDim.x));
  int64_t item = wg * quota;
  const int64_t end = min(item + quota, total);
  int32_t* desc = p.desc + static_cast<int64_t>(wg) * 8;
  if (t == 0) desc[0] = 0;
  int b = 0;
  if (item < end) {  // the sequence that holds the first item
    int lo = 0, hi = p.batch;  // prefix[lo] <= item < prefix[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= item) lo = mid;
      else hi = mid;
    }
    b = uni(lo);
  }

  while (item < end) {
    while (uni(prefix[b + 1]) <= item) ++b;
    Seq s = sequence<RT>(p, b, false);
    s = Seq{uni(s.start), uni(s.n), uni(s.len), uni(s.rows), uni(s.rw), uni(s.tiles)};
    const int64_t per_head = head_items<RT>(p, s);
    int64_t rem = item - uni(prefix[b]);
    const int h = uni(static_cast<int>(rem / per_head));
    rem -= h * per_head;
    int tile = 0, count = tile_items<RT>(p, s, 0);
    if (p.mask != nullptr) {
      tile = static_cast<int>(rem / count);
      rem -= static_cast<int64_t>(tile) * count;
    } else {
      while (rem >= count) {
        rem -= count;
        count = tile_items<RT>(p, s, ++tile);
      }
    }
    tile = uni(tile);
    const int c0 = uni(static_cast<int>(rem));
    const int c1 = static_cast<int>(min(static_cast<int64_t>(count), c0 + (end - item)));
    const int keys = tile_keys<RT>(p, s, tile);
    const int kbeg = c0 * kItemKeys, kend = min(keys, c1 * kItemKeys);
    const int ctx = s.len - s.n;  // keys that every row sees
    const int rw = s.rw, kw = 4 / rw;
    const int tile0 = tile * R * rw, row0 = tile0 + (wave % rw) * R;
    const int step = 32 * kw;

    // this lane's queries
    int tok[RT];
    u32x4 qf[RT][KK];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = min(row0 + 16 * i + n16, s.rows - 1);
      tok[i] = r / p.g;
      const T* q = static_cast<const T*>(p.q) + (s.start + tok[i]) * p.q_st +
                   static_cast<int64_t>(h * p.g + r % p.g) * p.q_sh;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        qf[i][kk] = *reinterpret_cast<const u32x4_any*>(q + 32 * kk + 8 * g4);
    }
    const bool rows_here = row0 < s.rows;

    f32x4 o[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const T* Kh = static_cast<const T*>(p.kc) + h * p.k_sh;
    const T* Vh = static_cast<const T*>(p.vc) + h * p.v_sh;
    const int64_t* trow = p.table + b * p.ld_table;
    const int last_block = (max(keys, 1) - 1) / 16;
    int first_block = -1;
    Blocks tab{0, 0};
    u32x4 kr[2][KK];
    uint32_t vr[8][VW];
    // The page and position of key block `blk` (16 keys) or, off P16, of this lane's own key.
    auto load_k = [&](int kb) {
#pragma unroll
      for (int th = 0; th < 2; ++th) {
        const T* src;
        if constexpr (P16) {
          const int i = min(kb / 16 + th, last_block) - first_block;
          const int pg = __builtin_amdgcn_readlane(tab.page, i);
          const int at = __builtin_amdgcn_readlane(tab.at, i);
          src = Kh + pg * p.k_sp + at * p.k_ss + n16 * p.k_ss;
        } else {
          const int i = min(kb + 16 * th + n16, keys - 1) - first_block;
          src = Kh + __shfl(tab.page, i, 64) * p.k_sp + __shfl(tab.at, i, 64) * p.k_ss;
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          kr[th][kk] = *reinterpret_cast<const u32x4_any*>(src + 32 * kk + 8 * g4);
      }
    };
    auto load_v = [&](int kb) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int th = j >> 2, in = 4 * g4 + (j & 3);
        const T* src;
        if constexpr (P16) {
          const int i = min(kb / 16 + th, last_block) - first_block;
          const int pg = __builtin_amdgcn_readlane(tab.page, i);
          const int at = __builtin_amdgcn_readlane(tab.at, i);
          src = Vh + pg * p.v_sp + at * p.v_ss + in * p.v_ss;
        } else {
          const int i = min(kb + 16 * th + in, keys - 1) - first_block;
          src = Vh + __shfl(tab.page, i, 64) * p.v_sp + __shfl(tab.at, i, 64) * p.v_ss;
        }
        src += DT * n16;
        if constexpr (VW == 4) {
          const u32x4 w = *reinterpret_cast<const u32x4_any*>(src);
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[j][e] = w[e];
        } else {
          typedef u32x2 u32x2_any __attribute__((aligned(2)));
          const u32x2 w = *reinterpret_cast<const u32x2_any*>(src);
          vr[j][0] = w[0];
          vr[j][1] = w[1];
        }
      }
    };
    // 64 blocks of 16 keys (off P16: 64 keys) from kb on
    auto pages_for = [&](int kb) {
      constexpr int span = P16 ? 1024 : 64;
      if (first_block >= 0 && kb + 32 <= (P16 ? 16 : 1) * first_block + span) return;
      if constexpr (P16) {
        first_block = kb / 16;
        tab = blocks(p, trow, first_block, last_block);
      } else {
        first_block = kb;
        const int x = min(kb + lane, keys - 1), i = x / p.page;
        const int64_t pg = trow[i];
        const bool ok = pg >= 0 && pg < p.n_pages;
        if (!ok && p.err != nullptr) *p.err = kPagedIndex;
        tab.page = ok ? static_cast<int>(pg) : 0;
        tab.at = x - i * p.page;
      }
    };

    int kb = kbeg + 32 * (wave / rw);
    if (rows_here && kb < kend) {
      pages_for(kb);
      load_k(kb);
      load_v(kb);
    }
    for (; rows_here && kb < kend; kb += step) {
      f32x4 sc[RT][2];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int th = 0; th < 2; ++th) {
          f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) a = mfma16<T>(kr[th][kk], qf[i][kk], a);
          sc[i][th] = a;
        }
      const bool more = kb + step < kend;
      const bool edge = kb + 32 > ctx;  // keys that not every row sees
      uint32_t odd = 0;  // keys of this lane's group with a value that is not finite
      if (edge) {
        const int k0 = kb + 4 * g4;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int th = 0; th < 2; ++th)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int key = k0 + 16 * th + r, j = key - ctx;
              bool see = key < kend;
              if (j >= 0)
                see = see && (p.mask != nullptr
                                  ? p.mask[(s.start + tok[i]) * p.ld_mask + j] != 0
                                  : j <= tok[i]);
              if (!see) sc[i][th][r] = -INFINITY;
            }
        // Slots past the end may hold anything, and a new key that some rows do
        // not see may hold infinities or NaN, which a probability of 0 would not cancel in
        // the product: they are taken out here and added below to the rows
        // that see them.
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = k0 + 16 * (j >> 2) + (j & 3);
          bool drop = key >= kend;
          if (!drop && key >= ctx) {
            bool bad = false;
#pragma unroll
            for (int e = 0; e < VW; ++e) bad = bad || not_finite<T>(vr[j][e]);
            // (any lane of this key's 16)
            bad = (__ballot(bad) >> (16 * g4) & 0xffffu) != 0;
            if (bad) odd |= 1u << j;
            drop = bad;
          }
          if (drop) {
#pragma unroll
            for (int e = 0; e < VW; ++e) vr[j][e] = 0;
          }
        }
      }
      const bool odd_any = edge && __ballot(odd != 0) != 0;
      if (more) {
        pages_for(kb + step);
        load_k(kb + step);
      }
      u32x4 pf[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int th = 0; th < 2; ++th)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sc[i][th][r] *= p.scale_log2;
            mx = fmaxf(mx, sc[i][th][r]);
          }
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
        const float ref = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
        for (int th = 0; th < 2; ++th)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sc[i][th][r] = __builtin_amdgcn_exp2f(sc[i][th][r] - ref);
            l[i] += sc[i][th][r];
          }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const T lo = Num<T>::from_f(sc[i][e >> 1][2 * (e & 1)]);
          const T hi = Num<T>::from_f(sc[i][e >> 1][2 * (e & 1) + 1]);
          pf[i][e] = __builtin_bit_cast(uint16_t, lo) |
                     static_cast<uint32_t>(__builtin_bit_cast(uint16_t, hi)) << 16;
        }
      }
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
      if (odd_any) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          for (int gg = 0; gg < 4; ++gg) {
            if ((__builtin_amdgcn_readlane(odd, 16 * gg) >> j & 1u) == 0) continue;
            const int key = kb + 16 * (j >> 2) + 4 * gg + (j & 3);
            const int64_t pg = trow[key / p.page];
            const T* v = Vh + (pg >= 0 && pg < p.n_pages ? pg : 0) * p.v_sp +
                         static_cast<int64_t>(key % p.page) * p.v_ss;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              const float pk = __shfl(sc[i][j >> 2][j & 3], n16 + 16 * gg, 64);
              if (pk == 0.f) continue;
#pragma unroll
              for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  o[i][d][r] = fmaf(pk, Num<T>::to_f(v[DT * (4 * g4 + r) + d]), o[i][d][r]);
            }
          }
      }
      if (more) load_v(kb + step);
    }

    // The waves' states meet in LDS: rows of wave group wave % rw, from kw waves.
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      l[i] += __shfl_xor(l[i], 16, 64);
      l[i] += __shfl_xor(l[i], 32, 64);
      const int r = 16 * i + n16;
      if (g4 == 0) {
        mg_m[wave][r] = m[i];
        mg_l[wave][r] = l[i];
      }
#pragma unroll
      for (int rr = 0; rr < 4; ++rr)
#pragma unroll
        for (int d = 0; d < DT; d += 4)
          *reinterpret_cast<f32x4*>(&merge[wave][r][DT * (4 * g4 + rr) + d]) =
              f32x4{o[i][d][rr], o[i][d + 1][rr], o[i][d + 2][rr], o[i][d + 3][rr]};
    }
    __syncthreads();
    const bool whole = c0 == 0 && c1 == count;
    const int live = min(R * rw, s.rows - tile0);
    float* slot = p.part + (static_cast<int64_t>(wg) * 2 + (c0 > 0 ? 0 : 1)) * (4 * R) * (D + 2);
    constexpr int LR = D / 8, RP = PT / LR;  // lanes per row, rows at a time
    for (int r = t / LR; r < live; r += RP) {
      const int w0 = r / R, rr = r % R, c = (t % LR) * 8;
      float M = -INFINITY, sum = 0.f, acc[8] = {};
      for (int k = 0; k < kw; ++k) M = fmaxf(M, mg_m[w0 + k * rw][rr]);
      for (int k = 0; k < kw; ++k) {
        const int w = w0 + k * rw;
        if (mg_m[w][rr] == -INFINITY && mg_l[w][rr] == 0.f) continue;  // saw nothing
        const float a = __builtin_amdgcn_exp2f(mg_m[w][rr] - (M == -INFINITY ? 0.f : M));
        sum = fmaf(a, mg_l[w][rr], sum);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(a, merge[w][rr][c + e], acc[e]);
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= inv;
        const int row = tile0 + r;
        store8u<T>(static_cast<T*>(p.o) +
                       ((s.start + row / p.g) * p.nkv * p.g + h * p.g + row % p.g) * D + c,
                   acc);
      } else {
        float* to = slot + r * (D + 2);
        if (c == 0) {
          to[0] = M;
          to[1] = sum;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) to[2 + c + e] = acc[e];
      }
    }
    if (t == 0 && c0 == 0 && c1 < count) {
      // this workgroup holds the unit's beginning: the merge kernel finds here what it needs
      const int64_t unit_end = item + count;
      desc[0] = static_cast<int32_t>((unit_end - 1) / quota - wg) + 1;  // workgroups of the unit
      desc[1] = h;
      desc[2] = tile0;
      desc[3] = live;
      desc[4] = static_cast<int32_t>(s.start);
    }
    item += c1 - c0;
    __syncthreads();
  }
}

// Units that several workgroups hold: workgroup wg0's beginning and the runs of those
// behind it, a row per wave's turn, in the order of the keys.
template <typename T, int D, int RT>
__global__ void __launch_bounds__(PT) paged_attn_merge(const PagedArgs p) {
  constexpr int R4 = 4 * 16 * RT, V = D / 64;
  const int32_t* desc = p.desc + static_cast<int64_t>(blockIdx.x) * 8;
  const int parts = desc[0];
  if (parts == 0) return;
  const int h = desc[1], tile0 = desc[2], live = desc[3];
  const int64_t start = desc[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int r = blockIdx.y * (PT / 64) + wave; r < live; r += gridDim.y * (PT / 64)) {
    auto part = [&](int k) {
      const int64_t slot = (static_cast<int64_t>(blockIdx.x) + k) * 2 + (k == 0 ? 1 : 0);
      return p.part + (slot * R4 + r) * (D + 2);
    };
    float M = -INFINITY;
    for (int k = lane; k < parts; k += 64) M = fmaxf(M, part(k)[0]);
    M = wave_reduce<MaxOp>(M);
    const float ref = M == -INFINITY ? 0.f : M;
    float sum = 0.f, acc[V] = {};
#pragma unroll 8
    for (int k = 0; k < parts; ++k) {
      const float* x = part(k);
      const bool nothing = x[0] == -INFINITY && x[1] == 0.f;
      const float a = nothing ? 0.f : __builtin_amdgcn_exp2f(x[0] - ref);
      sum = fmaf(a, x[1], sum);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(a, nothing ? 0.f : x[2 + V * lane + v], acc[v]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int row = tile0 + r;
    T* o = static_cast<T*>(p.o) +
           ((start + row / p.g) * p.nkv * p.g + h * p.g + row % p.g) * D + V * lane;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = Num<T>::from_f(acc[v] * inv);
  }
}

// Groups of 16 rows per wave: 1 where a sequence's rows fit 16 on average.
int row_groups(int64_t tokens, int64_t batch, int64_t g) {
  return tokens * g <= 16 * batch ? 1 : 2;
}
// Workgroups: what the chip holds at once, or fewer when the shapes cannot hold as many items.
int64_t paged_grid(int64_t tokens, int64_t batch, int64_t n_kv, int64_t g, int64_t max_keys) {
  const int rt = row_groups(tokens, batch, g);
  const int64_t most = rt == 1 ? 768 : 512;
  const int64_t tiles = std::min(tokens, tokens * g / (16 * rt) + batch);
  const double items = static_cast<double>(tiles) * n_kv *
                       static_cast<double>(std::max<int64_t>(1, ceil_div(max_keys, kItemKeys)));
  return items < most ? std::max<int64_t>(1, static_cast<int64_t>(items)) : most;
}
int64_t paged_part_floats(int64_t tokens, int64_t batch, int64_t g, int64_t head_dim) {
  return 2 * 64 * row_groups(tokens, batch, g) * (head_dim + 2);
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
  const int rt = row_groups(tokens, batch, g);
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
  const size_t lds = static_cast<size_t>(batch + 1) * 8;
  auto go = [&](auto tt, auto dd, auto rr, auto pp) {
    using T = decltype(tt);
    constexpr int D = decltype(dd)::value, RT = decltype(rr)::value;
    paged_attn_kernel<T, D, RT, decltype(pp)::value><<<dim3(grid), PT, lds, st>>>(a);
    if (grid > 1) paged_attn_merge<T, D, RT><<<dim3(grid, 2), PT, 0, st>>>(a);
  };
  auto by_page = [&](auto tt, auto dd, auto rr) {
    if (page_size % 16 == 0) go(tt, dd, rr, std::true_type{});
    else go(tt, dd, rr, std::false_type{});
  };
  auto by_rows = [&](auto tt, auto dd) {
    if (rt == 1) by_page(tt, dd, std::integral_constant<int, 1>{});
    else by_page(tt, dd, std::integral_constant<int, 2>{});
  };
  auto by_dim = [&](auto tt) {
    if (head_dim == 128) by_rows(tt, std::integral_constant<int, 128>{});
    else by_rows(tt, std::integral_constant<int, 64>{});
  };
  if (dtype == SPH_F16) by_dim(half_t{});
  else by_dim(bf16_t{});
  return check_launch("sph_paged_attention");
}
