// Tokens drawn from logits, with temperature, top-k, top-p and min-p, from given
// random numbers.
//
// For a row l[0 .. V) with maximum M and temperature t > 0 a token weighs
//   w_i = exp((l_i - M) / t)
// Tokens stand in the order of falling logits, equal ones by their index.
//   top-k   the first k stay
//   top-p   of those, the shortest run from the first on that holds p of their weight
//   min-p   of all, those with w_i >= min-p (the largest weight is 1)
// The token drawn is the first by index at which the weights of what stays, added up
// by index, exceed u times their sum.  t = 0: the largest logit, the lowest index first.
// NaN counts as -inf; a row without a value above -inf gives -1; beside +inf only
// +inf counts.
//
// A row has as many borders between tokens as it has tokens, so a relative error
// e of the weights turns over one drawn token in 1 / (V e): 32-bit weights would err once
// in some hundred rows.  Weights are therefore formed in 64 bits and held as
// whole multiples of 2^-shift, shift = 62 - log2 V (at most 51): their sums in 64-bit
// integers are exact and do not depend on the order of additions.
//
// A weight is formed in eleven 64-bit operations (2^y by a table of 256 steps and the series to
// the third power).  They bound the kernel: a 64-bit operation takes twice a 32-bit one's
// time, rows are read at the speed of the cache.  So as few weights as possible are formed:
//
//   * top-k of at most 1024: k of the 1024 threads' own maxima reach down to some value,
//     so the k largest do; what reaches it is listed in LDS (hardly more than k),
//     ranked by counting, and top-p, min-p and the draw run over the k first.
//   * else a cut (top-k by counts, top-p by weights) is found by histograms: over
//     2048 equal steps of the logit below the maximum (each holds few tokens, so the
//     atomics seldom meet), then over the ordered bit patterns of the step that the cut
//     falls into.  What is cut is described by that pattern and by how many of the
//     tokens with it stay; what stays is listed if there is room.  (Of a list the step's
//     tokens are few, and each is weighed by a thread of its own, which adds up those before it:
//     24 rows of top-p 50 us with the histograms of patterns, 41.5 so.)  The draw needs
//     the sums of all 512-token pieces and then one wave in the piece that holds the token.
//
// One workgroup per row, which reads it again where it is needed, a turn of loads ahead.  (Four
// turns ahead, the loops four times as long, doubled every pass's time: most
// instructions run a few times only, so fetching them counts.)  Several workgroups a row, in
// four launches (maxima, sums, lists, the rest), took 38.7 us for 42.4 at 24 rows of top-p,
// but 22.6 for 14.2 with top-k.
//
// Measured: 1 row of 49155 with every filter 14.3 us, 24 rows of top-p 0.9 41.5 us, 256
// rows of 131072 fp32 logits without filters 48.9 us (2.7 TB/s; 24 of it the weights).
#include <algorithm>
#include <type_traits>

#include "sph_common.h"

namespace sph {
namespace {

constexpr int ST = 1024;             // threads
constexpr int WAVES = ST / 64;
constexpr int TILE = ST * 8;         // tokens of a turn of the workgroup
constexpr int BINS = 2048;
constexpr int LIST = 14336;          // tokens that are listed in LDS
constexpr int64_t kMaxVocab = 1 << 20;
constexpr int MAX_PIECES = kMaxVocab / 512;
static_assert(MAX_PIECES <= BINS, "a piece per entry of the histogram");

struct alignas(8) Item {
  float value;
  int at;
};

struct SampleArgs {
  const void* logits;
  int64_t ld;
  int vocab, shift;
  const float* uniform;
  const float* temperature;
  const int64_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t* tokens;
};

// Order of the values as an order of unsigned integers.
__device__ inline uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct Shared {
  alignas(16) uint64_t hist[BINS];
  uint32_t count[BINS];
  Item list[LIST];
  double exp2[256];  // 2^(j / 256 + shift)
  uint64_t wave64[WAVES];
  float wmax[WAVES];
  int widx[WAVES];
  uint32_t few[ST];  // keys of a step's tokens
  uint32_t listed, in_few, kmin, kmax;
  int bin;
  uint64_t before, total;
};

// A row's weights.
struct Row {
  float top;     // M
  float floor;   // a value that has no weight for sure
  double rate;   // 256 log2 e / t
  const double* table;
  // 256 log2 of the weight; at least -26000, where it has none (NaN: -inf times 0)
  __device__ double log_of(float f) const {
    return fmax((static_cast<double>(f) - top) * rate, -26000.0);
  }
  // The weight times 2^shift, to the nearest whole number: y = 256 n + j + r, |r| <= 1/2, by
  // a sum with 1.5 2^52, whose low bits then hold 256 n + j; the series of 2^(r / 256)
  // to the third power (the next term is 1.4e-13 at most); n joins the exponent, and a sum
  // with 2^52 leaves the whole number in the low bits (shift <= 51).  NaN and -inf: 0.
  __device__ uint64_t weight(float f) const {
    constexpr double L = 0.0027076061740622863;  // ln 2 / 256
    const double y = (static_cast<double>(fmaxf(f, floor)) - top) * rate;
    const double s = y + 0x1.8p52;
    const int k = static_cast<int>(__builtin_bit_cast(uint64_t, s));
    const double r = y - (s - 0x1.8p52);
    double q = fma(L * L * L / 6, r, L * L / 2);
    q = fma(q, r, L);
    const double t = table[k & 255];
    uint64_t bits = __builtin_bit_cast(uint64_t, fma(t, q * r, t));
    bits += static_cast<uint64_t>(static_cast<uint32_t>(k >> 8) << 20) << 32;
    const double x = __builtin_bit_cast(double, bits) + 0x1p52;
    return __builtin_bit_cast(uint64_t, x) & 0xfffffffffffffull;
  }
};

// Inclusive sums over a wave, by lane moves inside rows of 16 and broadcasts of their ends.
template <int CTRL, int ROWS>
__device__ inline uint64_t moved(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ inline uint64_t wave_scan(uint64_t v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
__device__ inline uint32_t wave_scan(uint32_t v) {
  auto moved32 = [&](auto ctrl, auto rows) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  v += moved32(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  v += moved32(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  v += moved32(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  v += moved32(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  v += moved32(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  v += moved32(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return v;
}
__device__ inline uint64_t lane_xor(uint64_t v, int off) {
  const uint32_t lo = __shfl_xor(static_cast<int>(v), off, 64);
  const uint32_t hi = __shfl_xor(static_cast<int>(v >> 32), off, 64);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ inline uint64_t last_lane(uint64_t v) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), 63);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
// Over the workgroup's threads; total: of all.
__device__ inline uint64_t scan64(uint64_t v, Shared& s, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) s.wave64[wave] = v;
  __syncthreads();
  const uint64_t all = wave_scan(lane < WAVES ? s.wave64[lane] : 0);
  total = last_lane(all);
  const uint32_t lo = __shfl(static_cast<int>(all), max(wave - 1, 0), 64);
  const uint32_t hi = __shfl(static_cast<int>(all >> 32), max(wave - 1, 0), 64);
  return v + (wave == 0 ? 0 : static_cast<uint64_t>(hi) << 32 | lo);
}

// The first entry of s.hist at which cross(sum up to it, sum of all) holds: s.bin, with the
// sum before it in s.before and all in s.total.  Every thread calls it; without such an entry
// s.bin stays as it is.
template <typename F>
__device__ inline void find(Shared& s, F cross) {
  const int t = threadIdx.x;
  const uint64_t a = s.hist[2 * t], b = s.hist[2 * t + 1];
  uint64_t total;
  const uint64_t incl = scan64(a + b, s, total), e0 = incl - a - b, e1 = e0 + a;
  if (cross(e1, total) && (t == 0 || !cross(e0, total))) {
    s.bin = 2 * t;
    s.before = e0;
  } else if (cross(incl, total) && !cross(e1, total)) {
    s.bin = 2 * t + 1;
    s.before = e1;
  }
  if (t == 0) s.total = total;
  __syncthreads();
}

__device__ inline void add(uint64_t* to, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(to), static_cast<unsigned long long>(v));
}

// The number that the sums have to exceed.
__device__ inline uint64_t target_of(double u, uint64_t total) {
  const uint64_t x = u > 0.0 ? static_cast<uint64_t>(fmin(u, 1.0) * static_cast<double>(total)) : 0;
  return min(x, total - 1);
}

template <typename T>
__global__ void __launch_bounds__(ST) sample_kernel(const SampleArgs p) {
  __shared__ Shared s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + r * p.ld;
  const int V = p.vocab;
  const float temp = p.temperature != nullptr ? p.temperature[r] : 1.f;
  const int64_t k = p.top_k != nullptr ? p.top_k[r] : 0;
  const float share = p.top_p != nullptr ? p.top_p[r] : 1.f;
  const float min_p = p.min_p != nullptr ? p.min_p[r] : 0.f;
  const double u = p.uniform[r];
  if (t < 256) s.exp2[t] = exp2(t / 256.0 + p.shift);

  // 8 values from token i on, as they lie in memory; past the row's end -inf
  constexpr int RAW = sizeof(T) / 2;
  struct Eight {
    u32x4 w[RAW];
  };
  auto fetch = [&](int i) {
    Eight g;
    if (i + 8 <= V) {
#pragma unroll
      for (int j = 0; j < RAW; ++j) g.w[j] = *reinterpret_cast<const u32x4_any*>(x + i + j * 16 / sizeof(T));
    } else {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = i + j < V ? x[i + j] : Num<T>::from_f(-INFINITY);
      __builtin_memcpy(&g, e, sizeof(g));
    }
    return g;
  };
  // (beside +inf, which becomes 0, there is only -inf)
  bool top_inf = false;
  auto values = [&](const Eight& g, float (&v)[8]) {
    T e[8];
    __builtin_memcpy(e, &g, sizeof(g));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = Num<T>::to_f(e[j]);
    if (top_inf) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] == INFINITY ? 0.f : -INFINITY;
    }
  };
  // f(index of the turn's first, values, index of the first) for this thread's 8
  // tokens of every turn
  auto groups = [&](auto f) {
    Eight now = fetch(t * 8);
#pragma unroll 1
    for (int i0 = 0; i0 < V; i0 += TILE) {
      float v[8];
      values(now, v);
      now = fetch(i0 + TILE + t * 8);
      f(i0, v, i0 + t * 8);
    }
  };

  // ---- maximum (of this thread first); a row at no temperature: its first index
  float mine = -INFINITY;
  if (!(temp > 0.f)) {
    int at = 0x7fffffff;
    groups([&](int, const float (&v)[8], int i) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v[e] > mine) {
          mine = v[e];
          at = i + e;
        }
    });
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float om = __shfl_xor(mine, off, 64);
      const int oa = __shfl_xor(at, off, 64);
      if (om > mine || (om == mine && oa < at)) {
        mine = om;
        at = oa;
      }
    }
    if (lane == 0) {
      s.wmax[wave] = mine;
      s.widx[wave] = at;
    }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w)
      if (s.wmax[w] > mine || (s.wmax[w] == mine && s.widx[w] < at)) {
        mine = s.wmax[w];
        at = s.widx[w];
      }
    if (t == 0) p.tokens[r] = mine == -INFINITY ? -1 : at;
    return;
  }
  groups([&](int, const float (&v)[8], int) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mine = fmaxf(mine, v[e]);
  });
  {
    const float m = wave_reduce<MaxOp>(mine);
    if (lane == 0) s.wmax[wave] = m;
  }
  for (int i = t; i < BINS; i += ST) {
    s.hist[i] = 0;
    s.count[i] = 0;
  }
  if (t == 0) s.listed = 0;
  __syncthreads();
  float mx = s.wmax[0];
  for (int w = 1; w < WAVES; ++w) mx = fmaxf(mx, s.wmax[w]);
  if (mx == -INFINITY) {
    if (t == 0) p.tokens[r] = -1;
    return;
  }
  top_inf = mx == INFINITY;
  if (top_inf) mine = mine == INFINITY ? 0.f : -INFINITY;
  Row row;
  row.top = top_inf ? 0.f : mx + 0.f;  // (+ 0: one zero)
  row.rate = 256 * 1.4426950408889634074 / static_cast<double>(temp);
  row.table = s.exp2;
  {
    const float f = fmaxf(row.top - 72.f * temp, -3.402823466e38f);
    uint32_t key = key_of(f);  // (where t is small beside the last bit of M: one below it)
    while (key > 0x800000u && row.log_of(value_of(key)) > -25000.0 && key + 2 > key_of(f)) --key;
    row.floor = row.log_of(value_of(key)) > -25000.0 ? -INFINITY : value_of(key);
    // (there it is a value or two below M: whatever makes nothing of them will do)
    if (row.floor > -INFINITY)
      row.rate = fmin(row.rate, 32000.0 / (static_cast<double>(row.top) - row.floor));
  }
  // (a temperature at which -3.4e38 has weight: values are looked at one by one)
  const bool flat = row.floor == -INFINITY;
  // (no branch around a weight: eight in a row run side by side)
  auto weight = [&](float f) {
    const uint64_t w = row.weight(f);
    return f > -INFINITY ? w : 0;
  };
  // From 44 t below the maximum on a weight is less than half a unit.
  const float range = 44.f * temp;
  const float steps = range > 0.f && range < INFINITY ? (BINS - 1) / range : 0.f;
  auto step_of = [&](float f) {
    return static_cast<int>(fminf((row.top - f) * steps, static_cast<float>(BINS - 1)));
  };
  const double log_min = min_p > 0.f ? 256 * log2(static_cast<double>(fminf(min_p, 1.f))) : -30000.0;
  // Appends the tokens from lo to hi (lo > -inf) to the list, as far as there is room, and
  // counts them in s.listed.
  auto list_tokens = [&](float lo, float hi) {
    groups([&](int, const float (&v)[8], int i) {
      float most = v[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) most = fmaxf(most, v[e]);
      if (__ballot(most >= lo) == 0) return;
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m |= (v[e] >= lo && v[e] <= hi ? 1u : 0u) << e;
      if (__ballot(m != 0) == 0) return;
      const uint32_t n = __popc(m), upto = wave_scan(n);
      uint32_t at = 0;
      if (lane == 63) at = atomicAdd(&s.listed, upto);
      at = __builtin_amdgcn_readlane(at, 63) + upto - n;
      if (at >= LIST) return;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (m >> e & 1u) {
          if (at < LIST) s.list[at] = {v[e] + 0.f, i + e};
          ++at;
        }
    });
    __syncthreads();
  };
  auto clear = [&] {
    __syncthreads();
    for (int i = t; i < BINS; i += ST) s.hist[i] = 0;
    if (t == 0) s.listed = 0;
    __syncthreads();
  };

  // ---- few tokens stay: in order by counting
  if (k > 0 && k <= ST) {
    // k of the threads' maxima reach the least of those up to some step
    if (mine > -INFINITY) add(&s.hist[step_of(mine)], 1);
    if (t == 0) s.kmin = 0xffffffffu;
    __syncthreads();
    find(s, [&](uint64_t sum, uint64_t all) { return sum >= min(all, static_cast<uint64_t>(k)); });
    const bool enough = s.total >= static_cast<uint64_t>(k);
    if (mine > -INFINITY && step_of(mine) <= s.bin) atomicMin(&s.kmin, key_of(mine + 0.f));
    __syncthreads();
    // (fewer maxima than k: some threads have no tokens, so every token may be among the first)
    const float from = enough ? value_of(s.kmin) : -3.402823466e38f;
    if (enough || V <= LIST) list_tokens(from, INFINITY);
    const uint32_t n = s.listed;
    if ((enough || V <= LIST) && n <= ST) {
      // value and index in one number, larger for those that come first
      uint64_t mine64 = 0;
      if (t < static_cast<int>(n))
        mine64 = static_cast<uint64_t>(key_of(s.list[t].value)) << 32 |
                 ~static_cast<uint32_t>(s.list[t].at);
      s.hist[t] = mine64;
      __syncthreads();
      if (mine64 != 0) {
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < n; ++j) rank += s.hist[j] > mine64;
        s.hist[ST + rank] = mine64;
      }
      __syncthreads();
      const bool in = t < static_cast<int>(n) && t < k;
      mine64 = in ? s.hist[ST + t] : 0;
      const float f = value_of(static_cast<uint32_t>(mine64 >> 32));
      const int at = static_cast<int>(~static_cast<uint32_t>(mine64));
      uint64_t w = in ? weight(f) : 0;
      uint64_t total;
      const uint64_t upto = scan64(w, s, total);
      const double want = fmax(static_cast<double>(share), 0.0) * static_cast<double>(total);
      if (share < 1.f && t > 0 && !(static_cast<double>(upto - w) < want)) w = 0;
      if (in && row.log_of(f) < log_min) w = 0;
      __syncthreads();  // (the order above has been read)
      s.hist[2 * t] = w;
      s.hist[2 * t + 1] = at;
      scan64(w, s, total);
      const int m = __popcll(__ballot(w != 0));  // (what stays are the first)
      if (lane == 0) s.widx[wave] = m;
      __syncthreads();
      int stay = 0;
      for (int i = 0; i < WAVES; ++i) stay += s.widx[i];
      const uint64_t target = target_of(u, total);
      if (w != 0) {
        uint64_t upper = 0;  // weight up to this token by index
#pragma unroll 8
        for (int j = 0; j < stay; ++j) {
          const uint64_t other = s.hist[2 * j];
          upper += static_cast<int>(s.hist[2 * j + 1]) <= at ? other : 0;
        }
        if (upper > target && upper - w <= target) p.tokens[r] = at;
      }
      return;
    }
    clear();
  }

  // What stays: keys above cut, and the first `ties` tokens of those equal to it.
  uint32_t cut = key_of(-INFINITY);
  uint32_t ties = 0;
  bool listed = false;  // the list holds all that stays

  // f(value) for every token of the list or the row
  auto tokens = [&](bool of_list, auto f) {
    if (of_list) {
      const int n = static_cast<int>(s.listed);
      for (int i = t; i < n; i += ST) f(s.list[i].value);
    } else {
      groups([&](int, const float (&v)[8], int) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f(v[e]);
      });
    }
  };
  // Moves the cut to the first place in the order at which the amounts summed up to it
  // reach want_of(all of them); amount(f) of a token.  Of the tokens with the value at that
  // place as many stay as it takes.  (s.hist is 0.)
  auto move_cut = [&](auto amount, auto want_of) {
    const float cutv = value_of(cut);
    const uint32_t low_ties = ties;
    tokens(listed, [&](float f) {
      const uint64_t a = amount(f);
      if (f > cutv && a != 0) add(&s.hist[step_of(f)], a);
    });
    if (low_ties > 0 && t == 0) add(&s.hist[step_of(cutv)], amount(cutv) * low_ties);
    __syncthreads();
    find(s, [&](uint64_t sum, uint64_t all) { return static_cast<double>(sum) >= want_of(all); });
    const double want = want_of(s.total);
    const int bin = s.bin;
    uint64_t before = s.before;
    auto empty = [&] {
      __syncthreads();
      for (int i = t; i < BINS; i += ST) s.hist[i] = 0;
      __syncthreads();
    };
    const bool all_stay = static_cast<double>(s.total) < want;
    if (t == 0) {
      s.kmin = 0xffffffffu;
      s.kmax = 0;
      s.in_few = 0;
      if (!listed) s.listed = 0;
    }
    empty();
    if (all_stay) return;
    bool stepped = listed;  // the list holds the tokens of that step
    if (!listed) {
      // a list of what lies above the end of that step, or of the step alone (with room
      // for rounding)
      const float slack = 1e-6f * (fabsf(row.top) + (bin + 1) / steps);
      const float down = steps > 0.f && bin < BINS - 1
                             ? fmaxf(row.top - (bin + 1) / steps - slack, -3.402823466e38f)
                             : -3.402823466e38f;
      const float up = steps > 0.f ? row.top - bin / steps + slack : INFINITY;
      list_tokens(down, INFINITY);
      listed = stepped = s.listed <= LIST;
      if (!listed && up < row.top) {
        __syncthreads();
        if (t == 0) s.listed = 0;
        __syncthreads();
        list_tokens(down, up);
        stepped = s.listed <= LIST;
      }
    }
    const uint32_t low = cut;
    const bool cut_here = low_ties > 0 && step_of(cutv) == bin;
    // Few tokens in that step, as a rule: each thread weighs one and adds up what comes before.
    tokens(stepped, [&](float f) {
      if (!(f > cutv && step_of(f) == bin)) return;
      const uint32_t i = atomicAdd(&s.in_few, 1u);
      if (i < ST) s.few[i] = key_of(f + 0.f);
    });
    __syncthreads();
    const uint32_t n = s.in_few;
    if (n < 512) {
      // (2^parts threads a token, each with its part of the others)
      const int parts = min(__clz(n | 1) - 22, 6), token = t >> parts;
      const bool own = token < static_cast<int>(n), other = token == static_cast<int>(n) && cut_here;
      const uint32_t key = own ? s.few[token] : other ? low : 0;
      const uint64_t single = key != 0 ? amount(value_of(key)) : 0;
      if (token <= static_cast<int>(n)) {
        s.hist[2 * token] = own ? single : single * low_ties;
        s.hist[2 * token + 1] = key;
      }
      __syncthreads();
      uint64_t above = 0;
#pragma unroll 4
      for (uint32_t j = t & ((1 << parts) - 1); j <= n; j += 1 << parts) {
        const uint64_t w = s.hist[2 * j];
        above += static_cast<uint32_t>(s.hist[2 * j + 1]) > key ? w : 0;
      }
      for (int off = 1; off < 1 << parts; off *= 2) above += lane_xor(above, off);
      // the last key before which the amount is not reached
      const bool first = (t & ((1 << parts) - 1)) == 0 && single != 0;
      if (first && (above == 0 || static_cast<double>(before + above) < want)) atomicMin(&s.kmin, key);
      __syncthreads();
      cut = s.kmin;
      if (first && key == cut) {
        atomicAdd(&s.kmax, own ? 1u : low_ties);
        s.before = before + above;  // (all write the same)
        s.total = single;
      }
      __syncthreads();
      const double more = ceil((want - static_cast<double>(s.before)) / static_cast<double>(s.total));
      ties = min(s.kmax, static_cast<uint32_t>(fmax(more, 1.0)));
      empty();
      return;
    }
    auto in_step = [&](float f) { return f > cutv && step_of(f) == bin && amount(f) != 0; };
    uint32_t lo = 0xffffffffu, hi = 0;
    tokens(stepped, [&](float f) {
      if (!in_step(f)) return;
      lo = min(lo, key_of(f + 0.f));
      hi = max(hi, key_of(f + 0.f));
    });
    if (hi != 0) {
      atomicMin(&s.kmin, lo);
      atomicMax(&s.kmax, hi);
    }
    __syncthreads();
    lo = s.kmin;
    hi = s.kmax;
    if (cut_here) {
      lo = min(lo, low);
      hi = max(hi, low);
    }
    for (;;) {
      const uint32_t span = hi - lo;
      const int shift = span < BINS ? 0 : 32 - __clz(span) - 11;
      tokens(stepped, [&](float f) {
        if (!in_step(f)) return;
        const uint32_t key = key_of(f + 0.f);
        if (key >= lo && key <= hi) add(&s.hist[(hi - key) >> shift], amount(f));
      });
      if (t == 0 && cut_here && low >= lo && low <= hi)
        add(&s.hist[(hi - low) >> shift], amount(cutv) * low_ties);
      __syncthreads();
      find(s, [&](uint64_t sum, uint64_t) { return static_cast<double>(before + sum) >= want; });
      const uint32_t b = s.bin;
      const uint64_t all = s.hist[b];
      before += s.before;
      empty();
      if (shift == 0) {
        cut = hi - b;
        const uint64_t single = amount(value_of(cut));
        const double more = ceil((want - static_cast<double>(before)) / static_cast<double>(single));
        ties = min(static_cast<uint32_t>(all / single), static_cast<uint32_t>(fmax(more, 1.0)));
        return;
      }
      const uint32_t top = hi - (b << shift);
      lo = max(lo, top - ((1u << shift) - 1));
      hi = top;
    }
  };
  if (k > 0 && k < V)
    move_cut([](float) { return uint64_t{1}; }, [&](uint64_t) { return static_cast<double>(k); });
  if (share < 1.f)
    move_cut([&](float f) { return weight(f); },
             [&](uint64_t all) {
               // (one unit at least: of the first steps some may be empty, at a temperature
               // too small for them even that of the largest logit)
               return fmax(static_cast<double>(share) * static_cast<double>(all), 1.0);
             });
  // The least value that min-p lets through (the largest weight is 1), to the last bit.
  float least = -INFINITY;
  if (min_p > 0.f) {
    uint32_t lo = key_of(-3.402823466e38f), hi = key_of(row.top);  // (the largest passes)
    while (lo < hi) {  // 64 places at a time
      const uint32_t gap = (hi - lo) / 64 + 1, at = min(lo + lane * gap, hi);
      const uint64_t pass = __ballot(row.log_of(value_of(at)) >= log_min);
      const uint32_t l = pass != 0 ? __builtin_ctzll(pass) : 64;
      hi = pass != 0 ? min(lo + l * gap, hi) : hi;
      lo = l == 0 ? lo : lo + (l - 1) * gap + 1;
    }
    least = value_of(lo) + 0.f;
  }
  if (least > value_of(cut)) {
    cut = key_of(least) - (least == 0.f ? 2 : 1);  // (below 0 comes -0, which equals it)
    ties = 0;
  }

  // ---- the draw: weight above the cut and tokens at the cut in each piece of 512
  // (s.hist and s.count are 0)
  const float cutv = value_of(cut);
  const uint64_t tie_units = ties > 0 ? weight(cutv) : 0;
  if (!listed && cut != key_of(-INFINITY)) {
    __syncthreads();
    if (t == 0) s.listed = 0;
    __syncthreads();
    list_tokens(ties > 0 ? cutv : value_of(cut + 1), INFINITY);
    listed = s.listed <= LIST;
  }
  if (listed) {
    // each thread a run of an odd length (neighbours are of one piece, mostly)
    const int n = static_cast<int>(s.listed), run = n / ST | 1;
    uint64_t sum = 0;
    int piece = -1;
    auto leave = [&] {
      if (sum != 0) add(&s.hist[piece], sum);
      sum = 0;
    };
    for (int j = 0; j < n; j += run * ST)
      for (int i = j + t * run; i < min(j + (t + 1) * run, n); ++i) {
        const float f = s.list[i].value;
        const int at = s.list[i].at / 512;
        if (f > cutv) {
          if (at != piece) leave();
          piece = at;
          sum += weight(f);
        } else if (ties > 0 && f == cutv) {
          atomicAdd(&s.count[at], 1u);
        }
      }
    leave();
  } else if (cut == key_of(-INFINITY) && !flat) {
    groups([&](int i0, const float (&v)[8], int) {
      uint64_t sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += row.weight(v[e]);
      sum = wave_scan(sum);
      if (lane == 63) s.hist[i0 / 512 + wave] = sum;
    });
  } else {
    groups([&](int i0, const float (&v)[8], int) {
      uint64_t sum = 0;
      uint32_t n = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum += weight(v[e] > cutv ? v[e] : -INFINITY);
        n += ties > 0 && v[e] == cutv;
      }
      sum = wave_scan(sum);
      const uint64_t m = ties > 0 ? wave_scan(n) : 0;
      if (lane == 63) {
        s.hist[i0 / 512 + wave] = sum;
        s.count[i0 / 512 + wave] = static_cast<uint32_t>(m);
      }
    });
  }
  __syncthreads();
  if (wave != 0) return;
  // Each lane a run of the pieces, in order.  (Tokens at the cut stay by their index.)
  const int pieces = (V + 511) / 512, run = (pieces + 63) / 64;
  const int p0 = min(lane * run, pieces), p1 = min(p0 + run, pieces);
  uint64_t first = 0;
  if (ties > 0) {
    uint64_t n = 0;
    for (int i = p0; i < p1; ++i) n += s.count[i];
    first = wave_scan(n) - n;
    uint64_t seen = first;
    for (int i = p0; i < p1; ++i) {
      const uint32_t c = s.count[i];
      const uint64_t stay = seen >= ties ? 0 : min(static_cast<uint64_t>(c), ties - seen);
      s.hist[i] += stay * tie_units;
      s.count[i] = static_cast<uint32_t>(seen);
      seen += c;
    }
  }
  uint64_t sum = 0;
  for (int i = p0; i < p1; ++i) sum += s.hist[i];
  const uint64_t upto = wave_scan(sum);
  const uint64_t target = target_of(u, last_lane(upto));
  {
    uint64_t before = upto - sum;
    if (upto > target && before <= target) {  // (one lane)
      int i = p0;
      while (before + s.hist[i] <= target) before += s.hist[i++];
      s.bin = i;
      s.before = before;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int piece = s.bin, i = piece * 512 + lane * 8;
  float v[8];
  values(fetch(i), v);
  uint64_t n = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    n += ties > 0 && v[e] == cutv;
  }
  uint64_t tie = wave_scan(n) - n + (ties > 0 ? s.count[piece] : 0);
  uint64_t w[8], all = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    w[e] = v[e] > cutv ? weight(v[e]) : 0;
    if (ties > 0 && v[e] == cutv) w[e] = tie++ < ties ? tie_units : 0;
    all += w[e];
  }
  const uint64_t up = s.before + wave_scan(all);
  uint64_t at = up - all;
  if (up > target && at <= target) {
    int token = i;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (at <= target && at + w[e] > target) token = i + e;
      at += w[e];
    }
    p.tokens[r] = token;
  }
}

}  // namespace
}  // namespace sph

extern "C" int sph_sample(sph_dtype dtype, int64_t rows, int64_t vocab, const void* logits,
                          int64_t ld, const float* uniform, const float* temperature,
                          const int64_t* top_k, const float* top_p, const float* min_p,
                          int64_t* tokens, sph_stream_t stream) {
  using namespace sph;
  SPH_REQUIRE(dtype == SPH_F16 || dtype == SPH_BF16 || dtype == SPH_F32, SPH_ERR_UNSUPPORTED,
              "sample: logits must be F16, BF16 or F32");
  SPH_REQUIRE(rows >= 0 && vocab > 0, SPH_ERR_INVALID_ARG, "sample: bad sizes");
  if (rows == 0) return SPH_OK;
  SPH_REQUIRE(vocab <= kMaxVocab, SPH_ERR_TOO_LARGE, "sample: at most 2^20 tokens");
  SPH_REQUIRE(rows < (1 << 22), SPH_ERR_TOO_LARGE, "sample: at most 2^22 - 1 rows");
  SPH_REQUIRE(logits != nullptr && uniform != nullptr && tokens != nullptr, SPH_ERR_INVALID_ARG,
              "sample: null pointer");
  SPH_REQUIRE(rows == 1 || ld >= 0, SPH_ERR_INVALID_ARG, "sample: negative leading dimension");
  int bits = 0;
  while ((int64_t{1} << bits) < vocab) ++bits;
  const SampleArgs a{logits, ld, static_cast<int>(vocab), std::min(62 - bits, 51), uniform, temperature,
                     top_k, top_p, min_p, tokens};
  const dim3 grid(static_cast<unsigned>(rows));
  hipStream_t st = as_stream(stream);
  if (dtype == SPH_F16) sample_kernel<half_t><<<grid, ST, 0, st>>>(a);
  else if (dtype == SPH_BF16) sample_kernel<bf16_t><<<grid, ST, 0, st>>>(a);
  else sample_kernel<float><<<grid, ST, 0, st>>>(a);
  return check_launch("sph_sample");
}
