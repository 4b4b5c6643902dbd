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
// whole multiples of 2^-shift, shift = 62 - log2 V: their sums in 64-bit
// integers are exact and do not depend on the order of additions.
//
// One workgroup per row.  A cut (top-k by counts, top-p by weights) is found by
// histograms: first over 2048 equal steps of the logit between the maximum and the least logit
// that has weight (each step holds few tokens, so the atomics seldom meet), then
// within the step that the cut falls into, over ranges of the ordered bit patterns until
// one pattern is left.  What is cut is described by that pattern and by how
// many of the tokens with it stay.  The draw needs the sums of all 512-token
// pieces and then one wave in the piece that holds the token.
#include "sph_common.h"

namespace sph {
namespace {

constexpr int ST = 1024;             // threads
constexpr int WAVES = ST / 64;
constexpr int TILE = ST * 8;         // tokens of a turn of the workgroup
constexpr int BINS = 2048;
constexpr int LIST = 2048;           // tokens of a step that are kept in LDS
constexpr int64_t kMaxVocab = 1 << 20;
static_assert(kMaxVocab / 512 <= BINS, "a piece per entry of the scan");

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

struct Row {
  float top;        // M (0 where it is +inf)
  bool top_inf;
  double rate;      // 1 / t
  double unit;      // 2^shift
  __device__ float clean(float f) const {  // (+ 0: one zero)
    if (top_inf) return f == INFINITY ? 0.f : -INFINITY;
    return f != f ? -INFINITY : f + 0.f;
  }
  __device__ double weight(float f) const {
    return f == -INFINITY ? 0.0 : exp((static_cast<double>(f) - top) * rate);
  }
  __device__ uint64_t units(double w) const { return static_cast<uint64_t>(fma(w, unit, 0.5)); }
};

struct Shared {
  uint64_t hist[BINS];
  uint32_t count[BINS];
  float list[LIST];
  uint64_t wave64[WAVES];
  float wmax[WAVES], wmin[WAVES];
  int widx[WAVES];
  uint32_t listed, kmin, kmax;
  int bin;
  uint64_t before, total;
};

// Inclusive sums of a 64-bit value over the workgroup's threads; total: of all.
__device__ inline uint64_t scan64(uint64_t v, Shared& s, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t y = __shfl_up(v, off, 64);
    if (lane >= off) v += y;
  }
  __syncthreads();
  if (lane == 63) s.wave64[wave] = v;
  __syncthreads();
  uint64_t base = 0;
  total = 0;
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) base += s.wave64[w];
    total += s.wave64[w];
  }
  return base + v;
}

// The first entry of s.hist at which cross(sum up to it) holds: s.bin, with the sum before it
// in s.before and all in s.total.  Every thread calls it; cross holds for the whole sum.
template <typename F>
__device__ inline void find(Shared& s, F cross) {
  const int t = threadIdx.x;
  const uint64_t a = s.hist[2 * t], b = s.hist[2 * t + 1];
  uint64_t total;
  const uint64_t incl = scan64(a + b, s, total), e0 = incl - a - b, e1 = e0 + a;
  if (cross(e1) && (t == 0 || !cross(e0))) {
    s.bin = 2 * t;
    s.before = e0;
  } else if (cross(incl) && !cross(e1)) {
    s.bin = 2 * t + 1;
    s.before = e1;
  }
  if (t == 0) s.total = total;
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(ST) sample_kernel(const SampleArgs p) {
  __shared__ Shared s;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(p.logits) + r * p.ld;
  const int V = p.vocab;

  // f(tile, values, index of the first) for this thread's 8 tokens of every turn
  auto groups = [&](auto f) {
    for (int i0 = 0; i0 < V; i0 += TILE) {
      const int i = i0 + t * 8;
      float v[8];
      if (i + 8 <= V) load8u<T>(x + i, v);
      else load8_partial<T>(x + i, i < V ? V - i : 0, -INFINITY, v);
      f(i0, v, i);
    }
  };

  // ---- maximum, its first index, least finite value
  float mx = -INFINITY, mn = INFINITY;
  int at = 0x7fffffff;
  groups([&](int, const float (&v)[8], int i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (v[e] > mx) {
        mx = v[e];
        at = i + e;
      }
      if (v[e] > -INFINITY) mn = fminf(mn, v[e]);
    }
  });
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float om = __shfl_xor(mx, off, 64);
    const int oa = __shfl_xor(at, off, 64);
    if (om > mx || (om == mx && oa < at)) {
      mx = om;
      at = oa;
    }
    mn = fminf(mn, __shfl_xor(mn, off, 64));
  }
  if (lane == 0) {
    s.wmax[wave] = mx;
    s.widx[wave] = at;
    s.wmin[wave] = mn;
  }
  __syncthreads();
  for (int w = 0; w < WAVES; ++w) {
    if (s.wmax[w] > mx || (s.wmax[w] == mx && s.widx[w] < at)) {
      mx = s.wmax[w];
      at = s.widx[w];
    }
    mn = fminf(mn, s.wmin[w]);
  }
  const float temp = p.temperature != nullptr ? p.temperature[r] : 1.f;
  if (mx == -INFINITY || !(temp > 0.f)) {
    if (t == 0) p.tokens[r] = mx == -INFINITY ? -1 : at;
    return;
  }
  Row row;
  row.top_inf = mx == INFINITY;
  row.top = row.top_inf ? 0.f : mx;
  row.rate = 1.0 / static_cast<double>(temp);
  row.unit = ldexp(1.0, p.shift);
  // From 44 t below the maximum on a weight is less than half a unit.
  const float range = row.top_inf ? 0.f : fminf(mx - mn, 44.f * temp);
  const float steps = range > 0.f && range < INFINITY ? (BINS - 1) / range : 0.f;
  auto step_of = [&](float f) {
    return static_cast<int>(fminf((row.top - f) * steps, static_cast<float>(BINS - 1)));
  };

  // What stays: keys above cut, and the first `ties` tokens of those equal to it.
  uint32_t cut = key_of(-INFINITY);
  uint32_t ties = 0;

  // Moves the cut up to where cross(sum of amount over the order) first holds; amount(f) of a
  // token, `whole` times it for the tokens at the cut.  left(before, amount of one,
  // how many) gives the number that stays of the tokens where it holds.
  auto move_cut = [&](auto amount, auto cross, auto left) {
    // steps of the logit
    auto clear = [&] {
      __syncthreads();
      for (int i = t; i < BINS; i += ST) s.hist[i] = 0;
      if (t == 0) {
        s.listed = 0;
        s.kmin = 0xffffffffu;
        s.kmax = 0;
      }
      __syncthreads();
    };
    const float cutv = value_of(cut);
    const bool have = ties > 0;
    clear();
    groups([&](int, const float (&v)[8], int) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = row.clean(v[e]);
        if (f > -INFINITY && key_of(f) > cut) {
          const uint64_t a = amount(f);
          if (a != 0) atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[step_of(f)]), a);
        }
      }
    });
    if (have && t == 0)
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[step_of(cutv)]), amount(cutv) * ties);
    __syncthreads();
    find(s, [&](uint64_t sum) { return cross(sum, uint64_t{0}); });
    if (!cross(s.total, uint64_t{0})) return;  // all of it stays
    const int bin = s.bin;
    uint64_t before = s.before;
    const uint32_t low = cut;
    clear();
    // the keys of that step
    auto in_step = [&](float f) {
      return f > -INFINITY && key_of(f) > low && step_of(f) == bin && amount(f) != 0;
    };
    groups([&](int, const float (&v)[8], int) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = row.clean(v[e]);
        if (in_step(f)) {
          const uint32_t n = atomicAdd(&s.listed, 1u);
          if (n < LIST) s.list[n] = f;
          atomicMin(&s.kmin, key_of(f));
          atomicMax(&s.kmax, key_of(f));
        }
      }
    });
    const bool cut_here = have && step_of(cutv) == bin;
    __syncthreads();
    uint32_t lo = s.kmin, hi = s.kmax;
    const uint32_t listed = s.listed;
    if (cut_here) {
      lo = min(lo, low);
      hi = max(hi, low);
    }
    // f(value) for the tokens of the step
    auto step_tokens = [&](auto f) {
      if (listed <= LIST) {
        for (uint32_t i = t; i < listed; i += ST) f(s.list[i]);
      } else {
        groups([&](int, const float (&v)[8], int) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = row.clean(v[e]);
            if (in_step(y)) f(y);
          }
        });
      }
    };
    for (;;) {
      const uint32_t span = hi - lo;
      const int shift = span < BINS ? 0 : 32 - __clz(span) - 11;
      __syncthreads();
      for (int i = t; i < BINS; i += ST) s.hist[i] = 0;
      __syncthreads();
      step_tokens([&](float f) {
        const uint32_t k = key_of(f);
        if (k >= lo && k <= hi)
          atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[(hi - k) >> shift]), amount(f));
      });
      if (t == 0 && cut_here && low >= lo && low <= hi)
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.hist[(hi - low) >> shift]),
                  amount(cutv) * ties);
      __syncthreads();
      find(s, [&](uint64_t sum) { return cross(sum, before); });
      const uint32_t b = s.bin;
      if (shift == 0) {
        const uint32_t k = hi - b;
        const uint64_t one = amount(value_of(k)), all = s.hist[b];
        ties = left(before + s.before, one, static_cast<uint32_t>(all / one));
        cut = k;
        return;
      }
      before += s.before;
      const uint32_t top = hi - (b << shift);
      lo = max(lo, top - ((1u << shift) - 1));
      hi = top;
    }
  };

  if (p.top_k != nullptr) {
    const int64_t k = p.top_k[r];
    if (k > 0 && k < V) {
      const uint64_t want = k;
      move_cut([](float) { return uint64_t{1}; },
               [&](uint64_t sum, uint64_t before) { return before + sum >= want; },
               [&](uint64_t before, uint64_t, uint32_t n) {
                 return min(n, static_cast<uint32_t>(want - before));
               });
    }
  }
  if (p.top_p != nullptr && p.top_p[r] < 1.f) {
    const double share = fmax(static_cast<double>(p.top_p[r]), 0.0);
    // the weight of all that stays so far
    uint64_t mine = 0, total;
    groups([&](int, const float (&v)[8], int) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float f = row.clean(v[e]);
        if (f > -INFINITY && key_of(f) > cut) mine += row.units(row.weight(f));
      }
    });
    if (t == 0 && ties > 0) mine += row.units(row.weight(value_of(cut))) * ties;
    scan64(mine, s, total);
    const double want = share * static_cast<double>(total);
    move_cut([&](float f) { return row.units(row.weight(f)); },
             [&](uint64_t sum, uint64_t before) { return static_cast<double>(before + sum) >= want; },
             [&](uint64_t before, uint64_t one, uint32_t n) {
               const double more = ceil((want - static_cast<double>(before)) / static_cast<double>(one));
               return min(n, static_cast<uint32_t>(fmax(more, 1.0)));
             });
  }
  double least = 0.0;
  if (p.min_p != nullptr && p.min_p[r] > 0.f) least = fminf(p.min_p[r], 1.f);

  // ---- the draw: weight above the cut and tokens at the cut in each piece of 512
  __syncthreads();
  for (int i = t; i < BINS; i += ST) {
    s.hist[i] = 0;
    s.count[i] = 0;
  }
  __syncthreads();
  const double wc = ties > 0 ? row.weight(value_of(cut)) : 0.0;
  const uint64_t tie_units = wc >= least ? row.units(wc) : 0;
  auto units_above = [&](float f) -> uint64_t {
    if (!(f > -INFINITY) || key_of(f) <= cut) return 0;
    const double w = row.weight(f);
    return w >= least ? row.units(w) : 0;
  };
  groups([&](int i0, const float (&v)[8], int) {
    uint64_t sum = 0;
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = row.clean(v[e]);
      sum += units_above(f);
      n += ties > 0 && f > -INFINITY && key_of(f) == cut;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      sum += __shfl_xor(sum, off, 64);
      n += __shfl_xor(n, off, 64);
    }
    if (lane == 0) {
      s.hist[i0 / 512 + wave] = sum;
      s.count[i0 / 512 + wave] = n;
    }
  });
  __syncthreads();
  uint64_t total;
  {  // tokens at the cut stay by their index
    const uint32_t a = s.count[2 * t], b = s.count[2 * t + 1];
    const uint64_t incl = scan64(static_cast<uint64_t>(a) + b, s, total);
    const uint64_t e0 = incl - a - b, e1 = e0 + a;
    auto stay = [&](uint64_t first, uint32_t n) {
      return first >= ties ? 0u : min(n, static_cast<uint32_t>(ties - first));
    };
    s.hist[2 * t] += stay(e0, a) * tie_units;
    s.hist[2 * t + 1] += stay(e1, b) * tie_units;
    s.count[2 * t] = static_cast<uint32_t>(e0);
    s.count[2 * t + 1] = static_cast<uint32_t>(e1);
  }
  __syncthreads();
  {
    uint64_t mine = s.hist[2 * t] + s.hist[2 * t + 1];
    scan64(mine, s, total);
  }
  const double u = p.uniform[r];
  uint64_t target = u > 0.0 ? static_cast<uint64_t>(fmin(u, 1.0) * static_cast<double>(total)) : 0;
  target = min(target, total - 1);
  find(s, [&](uint64_t sum) { return sum > target; });
  if (wave != 0) return;
  const int piece = s.bin;
  const int i = piece * 512 + lane * 8;
  float v[8];
  if (i + 8 <= V) load8u<T>(x + i, v);
  else load8_partial<T>(x + i, i < V ? V - i : 0, -INFINITY, v);
  uint32_t n = 0;
  uint64_t sum = 0;
  for (int e = 0; e < 8; ++e) {
    v[e] = row.clean(v[e]);
    n += ties > 0 && v[e] > -INFINITY && key_of(v[e]) == cut;
  }
  uint32_t first = n;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t y = __shfl_up(first, off, 64);
    if (lane >= off) first += y;
  }
  first += s.count[piece] - n;
  uint64_t w[8];
  for (int e = 0; e < 8; ++e) {
    w[e] = units_above(v[e]);
    if (ties > 0 && v[e] > -INFINITY && key_of(v[e]) == cut) w[e] = first++ < ties ? tie_units : 0;
    sum += w[e];
  }
  uint64_t run = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t y = __shfl_up(run, off, 64);
    if (lane >= off) run += y;
  }
  const uint64_t upto = s.before + run;
  run = upto - sum;
  if (upto > target && run <= target) {
    int token = i;
    for (int e = 0; e < 8; ++e) {
      run += w[e];
      if (run > target) {
        token = i + e;
        break;
      }
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
  const SampleArgs a{logits, ld, static_cast<int>(vocab), 62 - bits, uniform, temperature,
                     top_k, top_p, min_p, tokens};
  const dim3 grid(static_cast<unsigned>(rows));
  hipStream_t st = as_stream(stream);
  if (dtype == SPH_F16) sample_kernel<half_t><<<grid, ST, 0, st>>>(a);
  else if (dtype == SPH_BF16) sample_kernel<bf16_t><<<grid, ST, 0, st>>>(a);
  else sample_kernel<float><<<grid, ST, 0, st>>>(a);
  return check_launch("sph_sample");
}
