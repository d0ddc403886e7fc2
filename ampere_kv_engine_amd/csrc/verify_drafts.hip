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
constexpr int kPart = kThreads * kLoads * 4;         // logits a block
constexpr int kMostPlaces = 64;                      // rows a request
constexpr int kMostParts = 64;

// What a part of a row leaves.
struct Part {
  double sum;        // of exp((x - top) / t)
  float top;
  int best;          // the lowest id of the largest logit (a part of minus infinities: none, INT_MAX)
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

// a b - c d with both products rounded: 0 where they are equal, not what the rounding of one leaves of a fused product.
__device__ __forceinline__ double difference(double a, double b, double c, double d) {
#pragma clang fp contract(off)
  const double ab = a * b, cd = c * d;
  return ab - cd;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int offset = kWave / 2; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, kWave);
  return v;
}

// Part `part` of a row in registers: piece u of a thread is x[part * kPart + u * 1024 + 4 * thread ..], ids beyond the row minus
// infinity.  `whole`: rows of whole 16-byte pieces on 16-byte boundaries.
__device__ __forceinline__ void fetch_part(const float* x, int vocab, int part, bool whole, float (&v)[kLoads][4]) {
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
  fetch_part(x, a.vocab, part, whole_pieces(a, x), v);
  float top = -INFINITY;
  int best = 0x7fffffff;
  bool nan = false;
#pragma unroll
  for (int u = 0; u < kLoads; ++u)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      nan |= v[u][j] != v[u][j];
      if (v[u][j] > top) { top = v[u][j]; best = part * kPart + u * kThreads * 4 + 4 * static_cast<int>(threadIdx.x) + j; }
    }
  __shared__ float tops[kThreads / kWave];
  __shared__ int bests[kThreads / kWave];
  __shared__ double sums[kThreads / kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int offset = kWave / 2; offset > 0; offset >>= 1) {
    const float other = __shfl_xor(top, offset, kWave);
    const int other_best = __shfl_xor(best, offset, kWave);
    if (other > top || (other == top && other_best < best)) { top = other; best = other_best; }
  }
  if (lane == 0) { tops[wave] = top; bests[wave] = best; }
  const int any_nan = __syncthreads_or(nan);
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w)
    if (tops[w] > top || (tops[w] == top && bests[w] < best)) { top = tops[w]; best = bests[w]; }
  double sum = 0.0;
  if (drawn && top > -INFINITY && top < INFINITY && any_nan == 0) {
    const double inverse = 1.0 / static_cast<double>(t), highest = static_cast<double>(top);
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += exp_of((static_cast<double>(v[u][j]) - highest) * inverse);
    sum = wave_sum64(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) sum += sums[w];
  }
  if (threadIdx.x == 0)
    a.parts[(static_cast<size_t>(request) * (2 * a.places - 1) + blockIdx.y) * a.part_count + part] = Part{sum, top, best, any_nan, 0};
}

// What a whole row's parts say.
struct Row {
  double sum, top;
  int best;
  bool fine;      // it has a next token: no NaN, something above minus infinity, nothing at plus infinity where it is drawn from
};

__device__ __forceinline__ Row gather_row(const Part* parts, int count, double inverse, bool drawn) {
  Row row{0.0, -INFINITY, 0x7fffffff, true};
  float top = -INFINITY;
  for (int i = 0; i < count; ++i) {
    const Part part = parts[i];
    if (part.nan != 0) row.fine = false;
    if (part.top > top) { top = part.top; row.best = part.best; }
  }
  row.top = top;
  if (top == -INFINITY || (drawn && top == INFINITY)) row.fine = false;
  if (row.fine && drawn)
    for (int i = 0; i < count; ++i)
      if (parts[i].top > -INFINITY) row.sum += parts[i].sum * exp_of((static_cast<double>(parts[i].top) - row.top) * inverse);
  return row;
}

__global__ __launch_bounds__(kThreads) void choose_kernel(Verify a) {
  __shared__ Row target[kMostPlaces], draft[kMostPlaces];
  __shared__ unsigned char fine[kMostPlaces];
  __shared__ double sums[kLoads][kThreads / kWave];
  __shared__ double scan[kMostParts];
  __shared__ int found, is_last, last_id;
  const int part = blockIdx.x, request = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & (kWave - 1), wave = tid / kWave;
  int first;
  const int rows = rows_of(a, request, first);
  const float t = a.temperature[request];
  const bool drawn = t > 0.f;
  const double inverse = drawn ? 1.0 / static_cast<double>(t) : 1.0;
  const Part* parts = a.parts + static_cast<size_t>(request) * (2 * a.places - 1) * a.part_count;
  for (int i = tid; i < 2 * a.places - 1; i += kThreads) {
    const bool of_target = i < a.places;
    const int place = of_target ? i : i - a.places;
    if (of_target && place < rows) target[place] = gather_row(parts + static_cast<size_t>(i) * a.part_count, a.part_count, inverse, drawn);
    if (!of_target && place < rows - 1 && a.draft != nullptr && drawn)
      draft[place] = gather_row(parts + static_cast<size_t>(i) * a.part_count, a.part_count, inverse, drawn);
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
  if (part == 0)
    for (int i = tid; i < a.places; i += kThreads)
      if (rows == 0 || i != kept) chosen[i] = i < kept ? a.tokens[first + i + 1] : -1;
  if (part == 0 && tid == 0) a.kept[request] = kept;
  if (rows == 0) return;
  const Row row = target[kept];
  const bool rejected = kept < rows - 1;
  const bool from_draft = rejected && a.draft != nullptr;
  if (!row.fine || !drawn || (from_draft && !draft[kept].fine)) {
    if (part == 0 && tid == 0) chosen[kept] = row.fine && !drawn ? row.best : -1;
    return;
  }
  const int refused = rejected && a.draft == nullptr ? a.tokens[first + kept + 1] : -1;    // (all of q lies on it)
  const float* x = a.logits + static_cast<size_t>(first + kept) * a.vocab;
  const float* y = from_draft ? a.draft + request * a.draft_request + kept * a.draft_place : nullptr;
  // the weights of a part, of `plain` p or of what q leaves of it
  auto weigh = [&](int of_part, bool plain, double (&w)[kLoads][4]) {
    float v[kLoads][4], z[kLoads][4];
    fetch_part(x, a.vocab, of_part, whole_pieces(a, x), v);
    const bool less = from_draft && !plain;
    if (less) fetch_part(y, a.vocab, of_part, whole_pieces(a, y), z);
    const double scale = 1.0 / row.sum, draft_scale = less ? 1.0 / draft[kept].sum : 0.0, draft_top = less ? draft[kept].top : 0.0;
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        double p = exp_of((static_cast<double>(v[u][j]) - row.top) * inverse);
        p = less ? fmax(difference(p, scale, exp_of((static_cast<double>(z[u][j]) - draft_top) * inverse), draft_scale), 0.0) : p * scale;
        if (!plain && of_part * kPart + u * kThreads * 4 + 4 * tid + j == refused) p = 0.0;
        w[u][j] = p;
      }
  };
  double w[kLoads][4];
  weigh(part, false, w);
  double sum = 0.0;
#pragma unroll
  for (int u = 0; u < kLoads; ++u) sum += (w[u][0] + w[u][1]) + (w[u][2] + w[u][3]);
  sum = wave_sum64(sum);
  if (lane == 0) sums[0][wave] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0;
    for (int i = 0; i < kThreads / kWave; ++i) sum += sums[0][i];
    __hip_atomic_store(a.weights + static_cast<size_t>(request) * a.part_count + part, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    is_last = arrive(a.arrivals + request) == static_cast<unsigned>(a.part_count - 1) ? 1 : 0;
  }
  __syncthreads();
  if (is_last == 0) return;
  // the request's last block: which part the draw falls into, then which id
  if (tid < a.part_count)
    scan[tid] = __hip_atomic_load(a.weights + static_cast<size_t>(request) * a.part_count + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  double total = 0.0;
  for (int i = 0; i < a.part_count; ++i) total += scan[i];
  const bool plain = !(total > 0.0);
  if (plain) {                                             // q leaves nothing of p: p itself, from the parts of the first launch
    __syncthreads();
    if (tid < a.part_count) {
      const Part one = parts[static_cast<size_t>(kept) * a.part_count + tid];
      scan[tid] = one.top > -INFINITY ? one.sum * exp_of((static_cast<double>(one.top) - row.top) * inverse) / row.sum : 0.0;
    }
    __syncthreads();
    total = 0.0;
    for (int i = 0; i < a.part_count; ++i) total += scan[i];
  }
  // (a number of 1 or more is the end of the line whatever the sums' last bits say)
  const float u = a.uniforms[static_cast<size_t>(request) * a.places + a.places - 1];
  const double goal = u < 1.f ? static_cast<double>(u) * total : INFINITY;
  // the first part whose end lies beyond the goal, or the last one of any weight
  int at = -1;
  double before = 0.0, upto = 0.0;
  for (int i = 0; i < a.part_count; ++i) {
    if (scan[i] > 0.0) { at = i; before = upto; }
    upto += scan[i];
    if (at == i && upto > goal) break;
  }
  if (at != part) weigh(at, plain, w);
  else if (plain) weigh(at, true, w);
  if (tid == 0) { found = 0x7fffffff; last_id = -1; }
  double ends[kLoads];       // of a piece's four ids over the lanes up to this one, then over everything before the piece as well
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    double s = (w[u][0] + w[u][1]) + (w[u][2] + w[u][3]);
#pragma unroll
    for (int offset = 1; offset < kWave; offset <<= 1) {
      const double other = __shfl_up(s, offset, kWave);
      if (lane >= offset) s += other;
    }
    ends[u] = s;
    if (lane == kWave - 1) sums[u][wave] = s;
  }
  __syncthreads();
  int mine = 0x7fffffff, last = -1;
  double base = before;
  for (int u = 0; u < kLoads; ++u)
    for (int i = 0; i < kThreads / kWave; ++i) {
      if (i == wave) {
#pragma unroll
        for (int v = 0; v < kLoads; ++v)
          if (v == u) {
            double s = base + ends[v] - ((w[v][0] + w[v][1]) + (w[v][2] + w[v][3]));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              s += w[v][j];
              const int id = at * kPart + v * kThreads * 4 + 4 * tid + j;
              if (w[v][j] > 0.0) {
                last = id;
                if (s > goal && id < mine) mine = id;
              }
            }
          }
      }
      base += sums[u][i];
    }
#pragma unroll
  for (int offset = kWave / 2; offset > 0; offset >>= 1) {
    mine = min(mine, __shfl_xor(mine, offset, kWave));
    last = max(last, __shfl_xor(last, offset, kWave));
  }
  if (lane == 0) { atomicMin(&found, mine); atomicMax(&last_id, last); }
  __syncthreads();
  if (tid == 0) chosen[kept] = found != 0x7fffffff ? found : last_id;
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
  choose_kernel<<<dim3(parts, requests), kThreads, 0, stream>>>(a);
  return AKV_LAUNCH_STATUS();
}
