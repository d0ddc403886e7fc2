// Drafted tokens held against the target's probabilities, from given random numbers: how many of a request's drafts are kept, and
// the token that follows them.
//
//   p_i = softmax(logits_i / t), q_i = softmax(draft_logits_i / t), or all of q_i on the drafted token where no draft model is given
//   draft d_i is kept while u_i q_i(d_i) < p_i(d_i); the first that is not ends the walk at i = kept
//   the next token is drawn from max(p - q, 0) at `kept` (from p where that is nothing, or where every draft was kept): the lowest
//   id whose cumulative weight exceeds u_last times the whole, or the last id of any weight
//   t <= 0: a draft is kept where it is the target's largest logit (ties: the lowest id), and the next token is the largest
//
// The rows are read once, a block two parts of kPart logits held in registers (`parts_kernel`: the largest, and each part's sum of
// exponentials below it).  A second launch (`choose_kernel`) decides - every block of a request for itself, from the parts' few
// numbers -, sums the weights of its part of the row that is drawn from, and the request's last block finds the part and the id.
// Everything that is compared with a random number is summed in 64 bits: the draw looks for a place among up to 151,936 cumulative
// weights, and sums in 32 bits, off by 1e-7, would choose another id for one draw in thirty; off by 1e-13, for none.  The vector units
// have 64-bit products at the rate of 32-bit ones, so that the exponentials cost nine operations each and not much more time than
// the reads: 64 requests of five rows and four draft rows of 151,936 logits (350 MB) take 75 us, 4.7 TB/s of the 6.2 that plain reads
// reach, and the second launch, which reads two rows of each request again (78 MB), 30 us; a single request 5.3 and 6.5 us, which are a
// launch's way to the first data and back.  Two parts a block: with one the first launch takes 78 us (its ends are paid twice as often),
// while parts of twice the size cost the second launch 17 us more, since one block ends with a whole part.

#include "common.h"
#include "api_rounds.h"

using namespace akv;

namespace {

constexpr int kThreads = 256;
constexpr int kChooseThreads = 512;
constexpr int kPart = 4096;                          // logits a part
constexpr int kPerBlock = 2;                         // parts a block of the first launch
constexpr int kMostPlaces = 64;                      // rows a request
constexpr int kMostParts = 64;                       // a lane each

// What a part of a row leaves.
struct Part {
  double sum;        // of exp((x - top) / t)
  float top;
  int best;          // the lowest id of the largest logit, where nothing is drawn
  int nan;
  int pad;
};

struct Verify {
  const float* logits;         // [rows, vocab]
  const float* draft;          // null, or request r's logits of place i at r * draft_request + i * draft_place
  const int *tokens, *q_start;
  const float *temperature, *uniforms;
  int *kept, *chosen;
  Part* parts;                 // [requests][places (targets), places - 1 (drafts)][parts]
  double* weights;             // [requests][parts]
  unsigned* arrivals;          // [requests]
  long draft_request, draft_place;
  int rows, vocab, requests, places, part_count;
};

// e^z for z <= 0.  2^f for |f| <= 1/2 by its series in f ln 2 up to the tenth power (the rest is below 2.3e-13 of it), the whole part
// of the exponent by scaling.
__device__ __forceinline__ double exp_of(double z) {
  const double y = fmax(z * 1.4426950408889634074, -1100.0);
  const double k = rint(y), f = (y - k) * 0.69314718055994530942;
  double v = 1.0 / 3628800.0;
  v = fma(v, f, 1.0 / 362880.0);
  v = fma(v, f, 1.0 / 40320.0);
  v = fma(v, f, 1.0 / 5040.0);
  v = fma(v, f, 1.0 / 720.0);
  v = fma(v, f, 1.0 / 120.0);
  v = fma(v, f, 1.0 / 24.0);
  v = fma(v, f, 1.0 / 6.0);
  v = fma(v, f, 0.5);
  v = fma(v, f, 1.0);
  v = fma(v, f, 1.0);
  return ldexp(v, static_cast<int>(k));
}

// e^((x - offset) / t) for what is done to whole rows, in nine operations of 64 bits.  In units of 1/32 of a power of two the exponent is
// x by + B, by = 32 log2(e) / t, B = -offset by.  B's whole part goes into the number that rounds: adding C = 1.5 * 2^52 + rint(B) to
// x by leaves the whole number k in the sum's lowest bits, and x by - (that - C) is the rest f, |f| <= 1/2, exactly - a fused product
// rounds once.  2^(k / 32) is one of 32 powers (`powers`: in LDS, a bank pair each, so that lanes do not wait for each other) with k's upper
// bits added to its exponent; the entries' exponents have k's lower five bits subtracted, so that k is added whole.  2^(f / 32) is
// a polynomial of degree 4, the series to the fifth with its last term spread over the others by the fifth Chebyshev polynomial (off by
// 8e-14).  With an offset that makes B whole that is all; what another one leaves is a factor, `rest`.  A logit is held above 680 t
// below the row's largest, rounded towards the largest (the next float may be half as far away: weights of 1e-147 and less, and whatever
// is less than kLeast counts as nothing where an id is picked).  Where that is the largest itself, the next float below it
// is more than 680 t away and only logits equal to it have any weight: `near` is false, and the logits are replaced
// by 0, the largest, and minus infinity.
constexpr int kPowers = 32;
constexpr double kMagic = 6755399441055744.0;
constexpr double kLeast = 1e-130;
constexpr float kWarmest = 1e28f;        // temperatures above it are taken as it: 680 t stays below the steps of the largest floats
struct Scale {
  double by, shift, origin;
  float lowest;
  bool near;
};
// `inverse` = 1 / t, a division that a block does once.  The offset is the one next to the largest logit for which B is whole.
__device__ __forceinline__ Scale scale_of(float t, double inverse, float top) {
  Scale s{kPowers * 1.4426950408889634074 * inverse, kMagic, 0.0, 0.f, true};
  const double deepest = static_cast<double>(top) - 680.0 * t;
  s.lowest = static_cast<float>(deepest);
  if (static_cast<double>(s.lowest) < deepest) s.lowest = nextafterf(s.lowest, INFINITY);
  s.near = s.lowest < top;
  if (s.near) s.origin = static_cast<double>(top);
  else s.lowest = -680.f * t;
  s.shift += rint(-s.origin * s.by);
  return s;
}
// The offset `above` beyond the largest logit.
__device__ __forceinline__ Scale scale_of(float t, double inverse, float top, double above, double& rest) {
  Scale s = scale_of(t, inverse, top);
  const double offset = s.origin + above;
  const double b = -offset * s.by, lost = fma(-offset, s.by, -b), whole = rint(b);
  rest = exp2(((b - whole) + lost) * (1.0 / kPowers));
  s.shift = kMagic + whole;
  return s;
}
template <int COUNT> __device__ __forceinline__ void only_largest(float (&v)[COUNT], float top) {
#pragma unroll
  for (int e = 0; e < COUNT; ++e) v[e] = v[e] == top ? 0.f : -INFINITY;
}
// (by a block's first 32 threads; `factor`: every weight's)
__device__ __forceinline__ void fill_powers(double* powers, double factor) {
  if (threadIdx.x < kPowers) {
    const double power = exp2(threadIdx.x * (1.0 / kPowers)) * factor;
    powers[threadIdx.x] = __hiloint2double(__double2hiint(power) - (static_cast<int>(threadIdx.x) << 15), __double2loint(power));
  }
}
__device__ __forceinline__ double split_exp(float x, const Scale& s, const double* powers, double& power) {
  constexpr double kStep = 0.69314718055994530942 / kPowers, kReach = kStep / 2;
  const double wide = static_cast<double>(fmaxf(x, s.lowest));
  const double rounded = fma(wide, s.by, s.shift);
  const int k = __double2loint(rounded);
  const double f = fma(wide, s.by, -(rounded - s.shift));
  double v = kStep * kStep * kStep * kStep / 24.0;
  v = fma(v, f, kStep * kStep * kStep * (1.0 / 6.0 + kReach * kReach * 20.0 / (16.0 * 120.0)));
  v = fma(v, f, kStep * kStep / 2.0);
  v = fma(v, f, kStep * (1.0 - kReach * kReach * kReach * kReach * 5.0 / (16.0 * 120.0)));
  power = powers[k & (kPowers - 1)];
  power = __hiloint2double(__double2hiint(power) + (k << 15), __double2loint(power));
  return fma(v, f, 1.0);
}
__device__ __forceinline__ double add_exp(double sum, float x, const Scale& s, const double* powers) {
  double power;
  const double v = split_exp(x, s, powers, power);
  return fma(v, power, sum);
}
__device__ __forceinline__ double just_exp(float x, const Scale& s, const double* powers) {
  double power;
  const double v = split_exp(x, s, powers, power);
  return v * power;
}

// a - b, not contracted with the products that they are: 0 where they are equal, not what the rounding of one leaves.
__device__ __forceinline__ double difference(double a, double b) {
#pragma clang fp contract(off)
  return a - b;
}

// Sums over the lanes up to each, and over all of them, inside the vector unit: four shifts within rows of 16 lanes, two broadcasts of
// a row's last lane to the rows behind it (an exchange through LDS takes some hundred cycles, and a sum of 64 bits twelve of them).
template <int CTRL, int ROWS> __device__ __forceinline__ double moved(double v) {
  const int low = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, false);
  const int high = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, false);
  return __hiloint2double(high, low);
}
__device__ __forceinline__ double sums_up_to(double v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ double of_lane(double v, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}
__device__ __forceinline__ double wave_sum64(double v) { return of_lane(sums_up_to(v), kWave - 1); }

// The largest value of a wave, and the lowest index of those that have it.
template <int CTRL, int ROWS> __device__ __forceinline__ float larger(float v) {
  const int low = __float_as_int(-INFINITY);
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(low, __float_as_int(v), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_top(float v) {
  v = larger<0x111, 0xf>(v);
  v = larger<0x112, 0xf>(v);
  v = larger<0x114, 0xf>(v);
  v = larger<0x118, 0xf>(v);
  v = larger<0x142, 0xa>(v);
  v = larger<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), kWave - 1));
}
template <int CTRL, int ROWS> __device__ __forceinline__ int lower(int v) {
  return min(v, __builtin_amdgcn_update_dpp(0x7fffffff, v, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_lowest(int v) {
  v = lower<0x111, 0xf>(v);
  v = lower<0x112, 0xf>(v);
  v = lower<0x114, 0xf>(v);
  v = lower<0x118, 0xf>(v);
  v = lower<0x142, 0xa>(v);
  v = lower<0x143, 0xc>(v);
  return __builtin_amdgcn_readlane(v, kWave - 1);
}

// IDS ids of a row from `begin` on in a block's registers: piece u of a thread is x[begin + 4 (u * threads + thread) ..], ids beyond the
// row minus infinity.  `whole`: rows of whole 16-byte pieces on 16-byte boundaries.
template <int THREADS, int IDS>
__device__ __forceinline__ void fetch_run(const float* x, int vocab, int begin, bool whole, float (&v)[IDS / 4 / THREADS][4]) {
  constexpr int kLoads = IDS / 4 / THREADS;
  const int first = begin + 4 * threadIdx.x;
  if (whole) {
    float4 fetched[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) fetched[u] = *reinterpret_cast<const float4*>(x + min(first + u * THREADS * 4, vocab - 4));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const bool inside = first + u * THREADS * 4 < vocab;
      v[u][0] = inside ? fetched[u].x : -INFINITY;
      v[u][1] = inside ? fetched[u].y : -INFINITY;
      v[u][2] = inside ? fetched[u].z : -INFINITY;
      v[u][3] = inside ? fetched[u].w : -INFINITY;
    }
  } else {
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[u][j] = x[min(first + u * THREADS * 4 + j, vocab - 1)];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (first + u * THREADS * 4 + j >= vocab) v[u][j] = -INFINITY;
  }
}

__device__ __forceinline__ bool whole_pieces(const Verify& a, const float* x) {
  return (a.vocab & 3) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

// A request's rows: those that q_start gives it, within the logits and the places there are.
__device__ __forceinline__ int rows_of(const Verify& a, int request, int& first) {
  first = a.q_start[request];
  const int end = a.q_start[request + 1];
  if (first < 0 || end > a.rows) return 0;
  return max(0, min(end - first, a.places));
}

__device__ __forceinline__ float temperature_of(const Verify& a, int request) {
  const float t = a.temperature[request];
  return t > kWarmest ? kWarmest : t;
}

// grid (blocks a row, 2 * places - 1, requests): rows 0 .. places - 1 are the target's, the others the draft's.  A block takes
// kPerBlock parts at once, and its waves do not wait for each other until the end.
__global__ __launch_bounds__(kThreads) void parts_kernel(Verify a) {
  constexpr int kWaves = kThreads / kWave, kPieces = kPart / 4 / kThreads;        // 16-byte pieces of a part a thread
  __shared__ Part of_waves[kPerBlock][kWaves];
  __shared__ double offsets[kPerBlock][kWaves];
  __shared__ double powers[kPowers];
  const int request = blockIdx.z, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const bool target = static_cast<int>(blockIdx.y) < a.places;
  const int place = target ? blockIdx.y : blockIdx.y - a.places;
  const int begin = blockIdx.x * kPerBlock;
  if (begin == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    __hip_atomic_store(a.arrivals + request, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);     // for the launch behind this one
  int first;
  const int rows = rows_of(a, request, first);
  const float t = temperature_of(a, request);
  const bool drawn = t > 0.f;
  if (place >= (target ? rows : rows - 1) || (!target && !drawn)) return;
  const float* x = target ? a.logits + static_cast<size_t>(first + place) * a.vocab
                          : a.draft + request * a.draft_request + place * a.draft_place;
  float v[kPerBlock * kPieces][4];
  fetch_run<kThreads, kPerBlock * kPart>(x, a.vocab, begin * kPart, whole_pieces(a, x), v);
  if (drawn) fill_powers(powers, 1.0);
  const double inverse = 1.0 / static_cast<double>(t);
  __syncthreads();
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < kPerBlock * kPieces; ++u) {
    nan |= __builtin_isunordered(v[u][0], v[u][1]) || __builtin_isunordered(v[u][2], v[u][3]);
    top = fmaxf(fmaxf(fmaxf(top, v[u][0]), v[u][1]), fmaxf(v[u][2], v[u][3]));
  }
  top = wave_top(top);
  nan = __any(nan);
  double sums[kPerBlock] = {}, offset = static_cast<double>(top);
  int best = 0x7fffffff;
  if (!drawn) {
#pragma unroll
    for (int u = kPerBlock * kPieces - 1; u >= 0; --u)
#pragma unroll
      for (int j = 3; j >= 0; --j)
        if (v[u][j] == top) best = begin * kPart + (u * kThreads + static_cast<int>(threadIdx.x)) * 4 + j;
    best = wave_lowest(best);
  } else if (top > -INFINITY && top < INFINITY && !nan) {
    const Scale scale = scale_of(t, inverse, top);
    if (scale.near) {
      offset = -(scale.shift - kMagic) * (t * (0.69314718055994530942 / kPowers));
    } else {
#pragma unroll
      for (int u = 0; u < kPerBlock * kPieces; ++u) only_largest(v[u], top);
    }
#pragma unroll
    for (int i = 0; i < kPerBlock; ++i) {
      double sum = 0.0, other = 0.0;     // (two sums: an addition does not wait for the one before it)
#pragma unroll
      for (int u = i * kPieces; u < (i + 1) * kPieces; ++u) {
        sum = add_exp(sum, v[u][0], scale, powers);
        other = add_exp(other, v[u][1], scale, powers);
        sum = add_exp(sum, v[u][2], scale, powers);
        other = add_exp(other, v[u][3], scale, powers);
      }
      sums[i] = wave_sum64(sum + other);
    }
  }
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < kPerBlock; ++i) {
      of_waves[i][wave] = Part{sums[i], top, best, nan ? 1 : 0, 0};
      offsets[i][wave] = offset;
    }
  __syncthreads();
  const int mine = static_cast<int>(threadIdx.x);
  if (mine < kPerBlock && begin + mine < a.part_count) {
    Part joined = of_waves[mine][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      const Part one = of_waves[mine][w];
      joined.nan |= one.nan;
      if (one.top > joined.top || (one.top == joined.top && one.best < joined.best)) { joined.top = one.top; joined.best = one.best; }
    }
    joined.sum = 0.0;
    if (drawn && joined.top > -INFINITY && joined.top < INFINITY) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (of_waves[mine][w].top > -INFINITY)
          joined.sum += of_waves[mine][w].sum * exp_of((offsets[mine][w] - static_cast<double>(joined.top)) * inverse);
    }
    a.parts[(static_cast<size_t>(request) * (2 * a.places - 1) + blockIdx.y) * a.part_count + begin + mine] = joined;
  }
}

// What a whole row's parts say.
struct Row {
  double sum, top;
  int best;
  bool fine;      // it has a next token: no NaN, something above minus infinity, nothing at plus infinity where it is drawn from
};

// By one wave, a lane a part.
__device__ __forceinline__ Row gather_row(const Part& part, double inverse, bool drawn) {
  const float top = wave_top(part.top);
  Row row{0.0, static_cast<double>(top), 0x7fffffff, !__any(part.nan != 0) && top > -INFINITY && !(drawn && top == INFINITY)};
  if (!drawn) row.best = wave_lowest(part.top == top ? part.best : 0x7fffffff);
  else if (row.fine) row.sum = wave_sum64(part.top > -INFINITY ? part.sum * exp_of((static_cast<double>(part.top) - row.top) * inverse) : 0.0);
  return row;
}

// grid (blocks a request, requests): a request's blocks share the parts of the row that is drawn from.
// (512 threads: what a request waits for is one block's chain of 64-bit operations; blocks of 256 and 1,024 were slower)
__global__ __launch_bounds__(kChooseThreads) void choose_kernel(Verify a) {
  constexpr int kThreads = kChooseThreads, kWaves = kThreads / kWave, kLoads = kPart / 4 / kThreads;
  __shared__ Row target[kMostPlaces], draft[kMostPlaces];
  __shared__ unsigned char fine[kMostPlaces];                // 1: the place's draft is kept if all before it are; 2: its number is NaN
  __shared__ double sums[kWaves], powers[kPowers], draft_powers[kPowers];
  __shared__ int of_waves[kWaves];
  __shared__ int is_last;
  const int block = blockIdx.x, request = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & (kWave - 1), wave = tid / kWave;
  int first;
  const int rows = rows_of(a, request, first);
  const float t = temperature_of(a, request);
  const bool drawn = t > 0.f;
  const double inverse = drawn ? 1.0 / static_cast<double>(t) : 1.0;
  const Part* parts = a.parts + static_cast<size_t>(request) * (2 * a.places - 1) * a.part_count;
  const int drafts = a.draft != nullptr && drawn ? rows - 1 : 0;
  auto part_of = [&](int i) {
    Part part{0.0, -INFINITY, 0x7fffffff, 0, 0};
    if (i < rows + drafts && lane < a.part_count) part = parts[static_cast<size_t>(i < rows ? i : a.places + i - rows) * a.part_count + lane];
    return part;
  };
  // (what place `tid`'s draft is decided by, and the rows' parts, are on their way together)
  const float last_number = a.uniforms[static_cast<size_t>(request) * a.places + a.places - 1];
  Part ahead = part_of(wave);
  int drafted = -1;
  float its_logit = 0.f, its_draft_logit = 0.f, its_number = 0.f;
  if (tid < rows - 1) {
    drafted = a.tokens[first + tid + 1];
    if (drawn && drafted >= 0 && drafted < a.vocab) {
      its_number = a.uniforms[static_cast<size_t>(request) * a.places + tid];
      its_logit = a.logits[static_cast<size_t>(first + tid) * a.vocab + drafted];
      if (a.draft != nullptr) its_draft_logit = a.draft[request * a.draft_request + tid * a.draft_place + drafted];
    }
  }
  for (int i = wave; i < rows + drafts; i += kWaves) {
    const Part part = ahead;
    ahead = part_of(i + kWaves);
    const Row row = gather_row(part, inverse, drawn);
    if (lane == 0) (i < rows ? target[i] : draft[i - rows]) = row;
  }
  __syncthreads();
  if (tid < rows - 1) {                                   // place `tid`'s draft: kept if all before it are
    const Row row = target[tid];
    bool keep = false;
    if (row.fine && t == t && drafted >= 0 && drafted < a.vocab) {
      if (!drawn) {
        keep = row.best == drafted;
      } else {
        const double p = exp_of((static_cast<double>(its_logit) - row.top) * inverse) / row.sum;
        double q = 1.0;
        bool known = true;
        if (a.draft != nullptr) {
          known = draft[tid].fine;
          q = exp_of((static_cast<double>(its_draft_logit) - draft[tid].top) * inverse) / draft[tid].sum;
        }
        keep = known && static_cast<double>(its_number) * q < p;
      }
    }
    fine[tid] = keep ? 1 : its_number != its_number ? 2 : 0;
  }
  __syncthreads();
  int kept = 0;
  while (kept < rows - 1 && fine[kept] == 1) ++kept;
  int* chosen = a.chosen + static_cast<size_t>(request) * a.places;
  if (block == 0)
    for (int i = tid; i < a.places; i += kThreads)
      if (rows == 0 || i != kept) chosen[i] = i < kept ? a.tokens[first + i + 1] : -1;
  if (block == 0 && tid == 0) a.kept[request] = kept;
  if (rows == 0) return;
  const Row row = target[kept];
  const bool rejected = kept < rows - 1;
  const bool from_draft = rejected && a.draft != nullptr;
  const bool no_number = last_number != last_number || (rejected && fine[kept] == 2);
  if (!row.fine || !drawn || (from_draft && !draft[kept].fine) || no_number) {
    if (block == 0 && tid == 0) chosen[kept] = row.fine && !drawn && t == t ? row.best : -1;
    return;
  }
  const int refused = rejected && a.draft == nullptr ? a.tokens[first + kept + 1] : -1;    // (all of q lies on it)
  const float* x = a.logits + static_cast<size_t>(first + kept) * a.vocab;
  const float* y = from_draft ? a.draft + request * a.draft_request + kept * a.draft_place : nullptr;
  // (a logit of `top + t log(sum)` would have a probability of 1: probabilities come without a product)
  double rest, draft_rest = 1.0;
  const float top = static_cast<float>(row.top), draft_top = from_draft ? static_cast<float>(draft[kept].top) : 0.f;
  const Scale of_row = scale_of(t, inverse, top, t * log(row.sum), rest);
  Scale of_draft{};
  if (from_draft) of_draft = scale_of(t, inverse, draft_top, t * log(draft[kept].sum), draft_rest);
  fill_powers(powers, rest);
  if (from_draft) fill_powers(draft_powers, draft_rest);
  __syncthreads();
  // the weight of an id: p's, `plain`, or what q leaves of it (logits of minus infinity count next to nothing)
  auto weight_of = [&](float logit, float draft_logit, int id, bool plain) {
    const double p = just_exp(logit, of_row, powers);
    if (from_draft && !plain) return fmax(difference(p, just_exp(draft_logit, of_draft, draft_powers)), 0.0);
    return !plain && id == refused ? 0.0 : p;
  };
  // the sum of the weights of a part, the same in every thread
  auto sum_part = [&](int of_part, bool plain) {
    float v[kLoads][4], z[kLoads][4];
    fetch_run<kThreads, kPart>(x, a.vocab, of_part * kPart, whole_pieces(a, x), v);
    if (from_draft) fetch_run<kThreads, kPart>(y, a.vocab, of_part * kPart, whole_pieces(a, y), z);
    if (!of_row.near) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) only_largest(v[u], top);
    }
    if (from_draft && !of_draft.near) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) only_largest(z[u], draft_top);
    }
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += weight_of(v[u][j], z[u][j], of_part * kPart + u * kThreads * 4 + 4 * tid + j, plain);
    sum = wave_sum64(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = wave_sum64(lane < kWaves ? sums[lane] : 0.0);
    __syncthreads();
    return sum;
  };
  // Of p alone the parts' weights are known from the first launch, all but the one of the refused draft; what q leaves of it has to
  // be summed, by all of the request's blocks.
  double weight = 0.0;                 // lane i: part i's
  bool plain = !rejected;
  auto weights_of_p = [&]() {
    weight = 0.0;
    if (lane < a.part_count) {
      const Part one = parts[static_cast<size_t>(kept) * a.part_count + lane];
      if (one.top > -INFINITY) weight = one.sum * exp_of((static_cast<double>(one.top) - row.top) * inverse) / row.sum;
    }
  };
  if (from_draft) {
    for (int i = block; i < a.part_count; i += gridDim.x) {
      const double sum = sum_part(i, false);
      if (tid == 0)
        __hip_atomic_store(a.weights + static_cast<size_t>(request) * a.part_count + i, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (tid == 0) is_last = arrive(a.arrivals + request) == gridDim.x - 1 ? 1 : 0;
    __syncthreads();
    if (is_last == 0) return;
    if (lane < a.part_count)
      weight = __hip_atomic_load(a.weights + static_cast<size_t>(request) * a.part_count + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  } else {
    if (block != 0) return;
    weights_of_p();
    if (rejected && refused >= 0 && refused < a.vocab) {
      const double sum = sum_part(refused / kPart, false);
      if (lane == refused / kPart) weight = sum;
    }
  }
  // by the request's last (or only) block: the part that the draw falls into
  double upto = sums_up_to(weight), total = of_lane(upto, kWave - 1);
  if (!(total > kLeast)) {              // nothing is left of p: p itself
    plain = true;
    weights_of_p();
    upto = sums_up_to(weight);
    total = of_lane(upto, kWave - 1);
  }
  // (a number of 1 or more is the end of the line whatever the sums' last bits say)
  const double goal = last_number < 1.f ? static_cast<double>(last_number) * total : INFINITY;
  // the first lane with weight whose sum lies beyond the goal, or the last lane with weight
  auto lane_of = [&](double value, double sum) {
    const unsigned long long some = __ballot(value > kLeast), beyond = __ballot(value > kLeast && sum > goal);
    return beyond != 0ull ? __builtin_ctzll(beyond) : some != 0ull ? kWave - 1 - __builtin_clzll(some) : -1;
  };
  const int at = max(0, lane_of(weight, upto));
  const double before = of_lane(upto, at) - of_lane(weight, at);
  // the part's ids, kLoads * 4 neighbours a thread: which thread, and then which of its ids
  constexpr int kEach = kLoads * 4;
  const int id0 = at * kPart + tid * kEach;
  double w[kEach], own = 0.0;
  {
    float v[kEach], z[kEach];
    auto fetch_own = [&](const float* from, const Scale& scale, float largest, float (&to)[kEach]) {
      if (whole_pieces(a, from)) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
          const float4 four = *reinterpret_cast<const float4*>(from + min(id0 + 4 * u, a.vocab - 4));
          to[4 * u] = four.x; to[4 * u + 1] = four.y; to[4 * u + 2] = four.z; to[4 * u + 3] = four.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < kEach; ++e) to[e] = from[min(id0 + e, a.vocab - 1)];
      }
      if (!scale.near) only_largest(to, largest);
    };
    fetch_own(x, of_row, top, v);
    if (from_draft) fetch_own(y, of_draft, draft_top, z);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      w[e] = id0 + e < a.vocab ? weight_of(v[e], z[e], id0 + e, plain) : 0.0;
      own += w[e];
    }
  }
  double end = sums_up_to(own);
  if (lane == kWave - 1) sums[wave] = end;
  __syncthreads();
  end += before + wave_sum64(lane < wave ? sums[lane] : 0.0);
  const int here = lane_of(own, end);
  const bool beyond = here >= 0 && of_lane(end, max(here, 0)) > goal;
  // the first wave that goes beyond the goal has it, or else the last one with any weight
  if (lane == 0) of_waves[wave] = here < 0 ? 0 : beyond ? 2 : 1;
  __syncthreads();
  const int of_wave = lane < kWaves ? of_waves[lane] : 0;
  const unsigned long long some = __ballot(of_wave == 1), over = __ballot(of_wave == 2);
  const int chosen_wave = over != 0ull ? __builtin_ctzll(over) : some != 0ull ? kWave - 1 - __builtin_clzll(some) : -1;
  if (wave != chosen_wave || lane != here) return;
  double sum = end - own;
  int last = -1;
  bool done = false;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    sum += w[e];
    if (w[e] > kLeast && !done) {
      last = id0 + e;
      done = sum > goal;
    }
  }
  chosen[kept] = last;
}

int part_count_of(int vocab) { return (vocab + kPart - 1) / kPart; }

bool sizes_taken(int requests, int places, int vocab) {
  return requests > 0 && requests <= 65535 && places >= 1 && places <= kMostPlaces && vocab >= 1 && vocab <= kMostParts * kPart;
}

long part_bytes(int requests, int places, int parts) { return static_cast<long>(requests) * (2 * places - 1) * parts * sizeof(Part); }

}  // namespace

extern "C" long akv_verify_workspace(int requests, int places, int vocab) {
  if (!sizes_taken(requests, places, vocab)) return -1;
  const int parts = part_count_of(vocab);
  return part_bytes(requests, places, parts) + static_cast<long>(requests) * (parts * sizeof(double) + sizeof(unsigned));
}

// logits [rows, vocab] and draft_logits (null: none; rows contiguous, its two strides in elements) float32; tokens [rows], the drafts of
// request r behind its first row; uniforms [requests, places], the last for the token that follows; kept [requests], chosen
// [requests, places]: the kept drafts, the token that follows them, -1.  A request without rows gets 0 and -1.
extern "C" int akv_verify_drafts(const float* logits, int rows, int vocab, const int* tokens, const int* q_start,
                                 const float* temperature, const float* uniforms, int requests, int places,
                                 const float* draft_logits, long draft_request_stride, long draft_place_stride, int* kept, int* chosen,
                                 void* workspace, hipStream_t stream) {
  if (!sizes_taken(requests, places, vocab) || rows < 0 || workspace == nullptr) return -2;
  const long last_draft = (requests - 1) * draft_request_stride + (places - 2) * draft_place_stride + vocab;
  const Span spans[] = {{kept, 4L * requests}, {chosen, 4L * requests * places}, {logits, 4L * rows * vocab}, {tokens, 4L * rows},
                        {q_start, 4L * requests + 4}, {temperature, 4L * requests}, {uniforms, 4L * requests * places},
                        {draft_logits, 4 * last_draft}};
  const int shared = shared_spans(spans, 2, 8);
  if (shared != 0) return shared;
  const int parts = part_count_of(vocab);
  char* room = static_cast<char*>(workspace);
  Verify a{};
  a.logits = logits; a.draft = draft_logits; a.tokens = tokens; a.q_start = q_start; a.temperature = temperature; a.uniforms = uniforms;
  a.kept = kept; a.chosen = chosen;
  a.parts = reinterpret_cast<Part*>(room);
  a.weights = reinterpret_cast<double*>(room + part_bytes(requests, places, parts));
  a.arrivals = reinterpret_cast<unsigned*>(a.weights + static_cast<size_t>(requests) * parts);
  a.draft_request = draft_request_stride; a.draft_place = draft_place_stride;
  a.rows = rows; a.vocab = vocab; a.requests = requests; a.places = places; a.part_count = parts;
  const int of_requests = draft_logits != nullptr ? 2 * places - 1 : places;
  parts_kernel<<<dim3((parts + kPerBlock - 1) / kPerBlock, of_requests, requests), kThreads, 0, stream>>>(a);
  const int first = AKV_LAUNCH_STATUS();
  if (first != 0) return first;
  // (as many blocks as the device holds at once, two a unit: every block decides for itself first, which takes it as long as two parts)
  const int blocks = max(1, min(parts, 2 * device_facts().compute_units / requests));
  choose_kernel<<<dim3(blocks, requests), kChooseThreads, 0, stream>>>(a);
  return AKV_LAUNCH_STATUS();
}
