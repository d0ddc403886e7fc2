// Drafted tokens held against the target's probabilities, from given random numbers: how many of a request's drafts are kept, and
// the token that follows them.
//
//   p_i = softmax(logits_i / t), q_i = softmax(draft_logits_i / t), or all of q_i on the drafted token where no draft model is given
//   draft d_i is kept while u_i q_i(d_i) < p_i(d_i); the first that is not ends the walk at i = kept
//   the next token is drawn from max(p - q, 0) at `kept` (from p where that is nothing, or where every draft was kept): the lowest
//   id whose cumulative weight exceeds u_last times the whole, or the last id of any weight
//   t <= 0: a draft is kept where it is the target's largest logit (ties: the lowest id), and the next token is the largest
//
// The rows are read once, a block a part of kPart logits held in registers (`parts_kernel`: the part's largest, and its sum of
// exponentials below that).  A second launch (`choose_kernel`) decides - every block of a request for itself, from the parts' few
// numbers -, sums the weights of its part of the row that is drawn from, and the request's last block finds the part and the id.
// Everything that is compared with a random number is summed in 64 bits: the draw looks for a place among up to 151,936 cumulative
// weights, and sums in 32 bits, off by 1e-7, would choose another id for one draw in thirty; off by 1e-13, for none.  The vector units
// have 64-bit products at the rate of 32-bit ones, and 2^f of a reduced argument is a polynomial of ten of them.

#include "common.h"
#include "api_rounds.h"

using namespace akv;

namespace {

constexpr int kThreads = 256;
constexpr int kLoads = 8;                            // 16-byte pieces a thread
constexpr int kChooseThreads = 512;
constexpr int kPart = kThreads * kLoads * 4;         // logits a block
constexpr int kMostPlaces = 64;                      // rows a request
constexpr int kMostParts = 64;

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

// The same for what is done to whole rows: 2^(z / 32) of z rounded to a whole number k is one of 32 powers (`powers`: in LDS, a bank
// pair each, so that lanes do not wait for each other), shifted; the rest, at most 1/64 of a power, a polynomial of degree 5 (off by
// 2e-15).  Rounding is an addition of 1.5 * 2^52, whose lowest bits are k.  A logit is held above -690 t below the row's largest
// (weights of 1e-299).
constexpr int kPowers = 32;
struct Scale {
  double by, top;      // 32 log2(e) / t; the (possibly none's) logit whose weight is 1
  float lowest;
};
__device__ __forceinline__ Scale scale_of(float t, float top) {
  return Scale{kPowers * 1.4426950408889634074 / static_cast<double>(t), static_cast<double>(top), fmaxf(top - 690.f * t, -3.4e38f)};
}
__device__ __forceinline__ void fill_powers(double* powers) {
  if (threadIdx.x < kPowers) powers[threadIdx.x] = exp2(threadIdx.x * (1.0 / kPowers));
}
// `v` times 2^(a whole power / 32) is e^((x - top) / t)
__device__ __forceinline__ double split_exp(float x, const Scale& s, const double* powers, double& power) {
  constexpr double kMagic = 6755399441055744.0, kStep = 0.69314718055994530942 / kPowers;
  const double d = static_cast<double>(fmaxf(x, s.lowest)) - s.top;
  const double rounded = fma(d, s.by, kMagic);
  const int k = __double2loint(rounded);
  const double f = fma(d, s.by, -(rounded - kMagic));
  double v = kStep * kStep * kStep * kStep * kStep / 120.0;
  v = fma(v, f, kStep * kStep * kStep * kStep / 24.0);
  v = fma(v, f, kStep * kStep * kStep / 6.0);
  v = fma(v, f, kStep * kStep / 2.0);
  v = fma(v, f, kStep);
  power = powers[k & (kPowers - 1)];
  power = __hiloint2double(__double2hiint(power) + ((k >> 5) << 20), __double2loint(power));
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

// Part `part` of a row in a block's registers: piece u of a thread is x[part * kPart + 4 (u * threads + thread) ..], ids beyond the row minus
// infinity.  `whole`: rows of whole 16-byte pieces on 16-byte boundaries.
template <int THREADS>
__device__ __forceinline__ void fetch_part(const float* x, int vocab, int part, bool whole, float (&v)[kPart / 4 / THREADS][4]) {
  constexpr int kLoads = kPart / 4 / THREADS, kThreads = THREADS;
  const int first = part * kPart + 4 * threadIdx.x;
  if (whole) {
    float4 fetched[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) fetched[u] = *reinterpret_cast<const float4*>(x + min(first + u * kThreads * 4, vocab - 4));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const bool inside = first + u * kThreads * 4 < vocab;
      v[u][0] = inside ? fetched[u].x : -INFINITY;
      v[u][1] = inside ? fetched[u].y : -INFINITY;
      v[u][2] = inside ? fetched[u].z : -INFINITY;
      v[u][3] = inside ? fetched[u].w : -INFINITY;
    }
  } else {
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[u][j] = x[min(first + u * kThreads * 4 + j, vocab - 1)];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (first + u * kThreads * 4 + j >= vocab) v[u][j] = -INFINITY;
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

// grid (parts, 2 * places - 1, requests): rows 0 .. places - 1 are the target's, the others the draft's
__global__ __launch_bounds__(kThreads) void parts_kernel(Verify a) {
  const int part = blockIdx.x, request = blockIdx.z;
  const bool target = static_cast<int>(blockIdx.y) < a.places;
  const int place = target ? blockIdx.y : blockIdx.y - a.places;
  if (part == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    __hip_atomic_store(a.arrivals + request, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);     // for the launch behind this one
  int first;
  const int rows = rows_of(a, request, first);
  const float t = a.temperature[request];
  const bool drawn = t > 0.f;
  if (place >= (target ? rows : rows - 1) || (!target && !drawn)) return;
  const float* x = target ? a.logits + static_cast<size_t>(first + place) * a.vocab
                          : a.draft + request * a.draft_request + place * a.draft_place;
  float v[kLoads][4];
  fetch_part<kThreads>(x, a.vocab, part, whole_pieces(a, x), v);
  __shared__ Part of_waves[kThreads / kWave];
  __shared__ double powers[kPowers];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  if (drawn) fill_powers(powers);
  __syncthreads();
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < kLoads; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      nan |= v[u][j] != v[u][j];
      top = fmaxf(top, v[u][j]);
    }
  top = wave_top(top);
  nan = __any(nan);
  int best = 0x7fffffff;
  double sum = 0.0;
  if (!drawn) {
#pragma unroll
    for (int u = kLoads - 1; u >= 0; --u)
#pragma unroll
      for (int j = 3; j >= 0; --j)
        if (v[u][j] == top) best = part * kPart + u * kThreads * 4 + 4 * static_cast<int>(threadIdx.x) + j;
    best = wave_lowest(best);
  } else if (top > -INFINITY && top < INFINITY && !nan) {
    const Scale scale = scale_of(t, top);
    double other = 0.0;                // (two sums: an addition does not wait for the one before it)
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      sum = add_exp(sum, v[u][0], scale, powers);
      other = add_exp(other, v[u][1], scale, powers);
      sum = add_exp(sum, v[u][2], scale, powers);
      other = add_exp(other, v[u][3], scale, powers);
    }
    sum = wave_sum64(sum + other);
  }
  if (lane == 0) of_waves[wave] = Part{sum, top, best, nan ? 1 : 0, 0};
  __syncthreads();
  if (threadIdx.x == 0) {
    Part whole = of_waves[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) {
      const Part one = of_waves[w];
      whole.nan |= one.nan;
      if (one.top > whole.top || (one.top == whole.top && one.best < whole.best)) { whole.top = one.top; whole.best = one.best; }
    }
    whole.sum = 0.0;
    if (drawn && whole.top > -INFINITY && whole.top < INFINITY) {
      const double inverse = 1.0 / static_cast<double>(t), highest = static_cast<double>(whole.top);
#pragma unroll
      for (int w = 0; w < kThreads / kWave; ++w)
        if (of_waves[w].top > -INFINITY)
          whole.sum += of_waves[w].sum * exp_of((static_cast<double>(of_waves[w].top) - highest) * inverse);
    }
    a.parts[(static_cast<size_t>(request) * (2 * a.places - 1) + blockIdx.y) * a.part_count + part] = whole;
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
  __shared__ unsigned char fine[kMostPlaces];
  __shared__ double sums[kWaves], powers[kPowers];
  __shared__ int of_waves[kWaves];
  __shared__ int is_last;
  const int block = blockIdx.x, request = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & (kWave - 1), wave = tid / kWave;
  int first;
  const int rows = rows_of(a, request, first);
  const float t = a.temperature[request];
  const bool drawn = t > 0.f;
  const double inverse = drawn ? 1.0 / static_cast<double>(t) : 1.0;
  const Part* parts = a.parts + static_cast<size_t>(request) * (2 * a.places - 1) * a.part_count;
  const int drafts = a.draft != nullptr && drawn ? rows - 1 : 0;
  if (drawn) fill_powers(powers);
  for (int i = wave; i < rows + drafts; i += kWaves) {
    Part part{0.0, -INFINITY, 0x7fffffff, 0, 0};
    if (lane < a.part_count) part = parts[static_cast<size_t>(i < rows ? i : a.places + i - rows) * a.part_count + lane];
    const Row row = gather_row(part, inverse, drawn);
    if (lane == 0) (i < rows ? target[i] : draft[i - rows]) = row;
  }
  __syncthreads();
  if (tid < rows - 1) {                                   // place `tid`'s draft: kept if all before it are
    const int id = a.tokens[first + tid + 1];
    const Row row = target[tid];
    bool keep = false;
    if (row.fine && id >= 0 && id < a.vocab) {
      if (!drawn) {
        keep = row.best == id;
      } else {
        const double p = exp_of((static_cast<double>(a.logits[static_cast<size_t>(first + tid) * a.vocab + id]) - row.top) * inverse) / row.sum;
        double q = 1.0;
        bool known = true;
        if (a.draft != nullptr) {
          known = draft[tid].fine;
          const float x = a.draft[request * a.draft_request + tid * a.draft_place + id];
          q = exp_of((static_cast<double>(x) - draft[tid].top) * inverse) / draft[tid].sum;
        }
        keep = known && static_cast<double>(a.uniforms[static_cast<size_t>(request) * a.places + tid]) * q < p;
      }
    }
    fine[tid] = keep;
  }
  __syncthreads();
  int kept = 0;
  while (kept < rows - 1 && fine[kept] != 0) ++kept;
  int* chosen = a.chosen + static_cast<size_t>(request) * a.places;
  if (block == 0)
    for (int i = tid; i < a.places; i += kThreads)
      if (rows == 0 || i != kept) chosen[i] = i < kept ? a.tokens[first + i + 1] : -1;
  if (block == 0 && tid == 0) a.kept[request] = kept;
  if (rows == 0) return;
  const Row row = target[kept];
  const bool rejected = kept < rows - 1;
  const bool from_draft = rejected && a.draft != nullptr;
  if (!row.fine || !drawn || (from_draft && !draft[kept].fine)) {
    if (block == 0 && tid == 0) chosen[kept] = row.fine && !drawn ? row.best : -1;
    return;
  }
  const int refused = rejected && a.draft == nullptr ? a.tokens[first + kept + 1] : -1;    // (all of q lies on it)
  const float* x = a.logits + static_cast<size_t>(first + kept) * a.vocab;
  const float* y = from_draft ? a.draft + request * a.draft_request + kept * a.draft_place : nullptr;
  // (a logit of `top + t log(sum)` would have a probability of 1: probabilities come without a product)
  Scale of_row = scale_of(t, static_cast<float>(row.top)), of_draft = of_row;
  of_row.top += static_cast<double>(t) * log(row.sum);
  if (from_draft) {
    of_draft = scale_of(t, static_cast<float>(draft[kept].top));
    of_draft.top += static_cast<double>(t) * log(draft[kept].sum);
  }
  // the weight of an id: p's, `plain`, or what q leaves of it (logits of minus infinity count 1e-299: no more than a rounding)
  auto weight_of = [&](float logit, float draft_logit, int id, bool plain) {
    const double p = just_exp(logit, of_row, powers);
    if (from_draft && !plain) return fmax(difference(p, just_exp(draft_logit, of_draft, powers)), 0.0);
    return !plain && id == refused ? 0.0 : p;
  };
  // the sum of the weights of a part, the same in every thread
  auto sum_part = [&](int of_part, bool plain) {
    float v[kLoads][4], z[kLoads][4];
    fetch_part<kThreads>(x, a.vocab, of_part, whole_pieces(a, x), v);
    if (from_draft) fetch_part<kThreads>(y, a.vocab, of_part, whole_pieces(a, y), z);
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
  if (!(total > 0.0)) {                // nothing is left of p: p itself
    plain = true;
    weights_of_p();
    upto = sums_up_to(weight);
    total = of_lane(upto, kWave - 1);
  }
  // (a number of 1 or more is the end of the line whatever the sums' last bits say)
  const float number = a.uniforms[static_cast<size_t>(request) * a.places + a.places - 1];
  const double goal = number < 1.f ? static_cast<double>(number) * total : INFINITY;
  // the first lane with weight whose sum lies beyond the goal, or the last lane with weight
  auto lane_of = [&](double value, double sum) {
    const unsigned long long some = __ballot(value > 0.0), beyond = __ballot(value > 0.0 && sum > goal);
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
    auto fetch_run = [&](const float* from, float (&to)[kEach]) {
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
    };
    fetch_run(x, v);
    if (from_draft) fetch_run(y, z);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      w[e] = id0 + e < a.vocab && v[e] > -INFINITY ? weight_of(v[e], z[e], id0 + e, plain) : 0.0;
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
    if (w[e] > 0.0 && !done) {
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
  parts_kernel<<<dim3(parts, of_requests, requests), kThreads, 0, stream>>>(a);
  const int first = AKV_LAUNCH_STATUS();
  if (first != 0) return first;
  // (as many blocks as the device holds at once, two a unit: every block decides for itself first, which takes it as long as two parts)
  const int blocks = max(1, min(parts, 2 * device_facts().compute_units / requests));
  choose_kernel<<<dim3(blocks, requests), kChooseThreads, 0, stream>>>(a);
  return AKV_LAUNCH_STATUS();
}
