// Attention of a batch whose requests share a long prefix, over the paged cache.  Compiled once per head size:
// -DAKV_HEAD_DIM=<multiple of 16, at most 256>.
//
// The first `shared` tokens of every request lie in the same pages.  A query's softmax runs over them and over its own request's
// tokens behind them, and sums of exponentials join:  with m the larger of two maxima, l = l1 2^(m1-m) + l2 2^(m2-m), and the same for
// the weighted sums of values.  So the prefix is walked once for the queries of ALL requests - they are the columns of one product,
// and a key is read once for all of them instead of once per request -, a request's own keys for its own queries, both cut into
// segments, each of which leaves (maximum, sum, weighted values); a second launch joins a row's segments.
//
// The columns of a kv head are its (token, query head of the group) pairs, token by token.  Both products are computed transposed:
//     S^T[key][col] = K[key][:] . Q[col][:]       A = 32 keys x 16 dims of a key page    (keys lie [page_size, dim])
//     O^T[dim][col] = V^T[dim][:] . P^T[:][col]   A = 32 dims x 16 keys of a value page  (values lie [dim, page_size])
// on 32 x 32 matrix instructions.  Which of the 32 keys of a step stands in which row of A is free: with row 8a + 4h + b holding key
// 16 (a / 2) + 8h + 4 (a % 2) + b, the scores that a lane gets are those of the keys whose values it multiplies next, in order, so
// that nothing is exchanged between the products.  float32 goes the same way on the float32 instruction (2 dims or keys a turn).

#include <type_traits>

#include "common.h"

#ifndef AKV_HEAD_DIM
#error "compile with -DAKV_HEAD_DIM=<head size>"
#endif

using namespace akv;

namespace {

constexpr int D = AKV_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head sizes are multiples of 16 up to 256");
constexpr int KC = D / 16;             // steps of 16 dims of the score product
constexpr int DT = (D + 31) / 32;      // tiles of 32 dims of the output (the last may be half empty)
constexpr int kThreads = 256, kWaves = 4;
constexpr int kRow = D + 4;            // floats a column takes in LDS: rows then lie 4 banks apart
template <typename T> constexpr size_t narrow_lds(int waves) {      // of `walk`
  return (waves / 2 * 32 * kRow + waves * 32 * 2 + 64) * sizeof(float) + D * 32 * sizeof(T);
}
constexpr float kLog2e = 1.4426950408889634f;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float floatx4;
typedef __attribute__((ext_vector_type(16))) float floatx16;
typedef __attribute__((ext_vector_type(4))) unsigned int uintx4;

struct Args {
  const void* q;              // [tokens, q_heads * D]
  const void* k_pages;        // [pages, kv_heads, page_size, D]
  const void* v_pages;        // [pages, kv_heads, D, page_size]
  void* out;                  // [tokens, q_heads * D]
  float* sums;                // [kv_heads][segments][rows][D] weighted values of a segment, below its maximum
  float* stats;               // [kv_heads][rows][segments][2] a segment's maximum (base 2, scaled) and its sum of weights
  const int* q_start;         // [requests + 1]
  const int* seq_lens;        // [requests] tokens held, the new ones among them
  const int* block_table;     // [.., table_width]
  const int* table_rows;      // null, or [requests]: a request's row of the table
  int table_width, table_count, requests;     // (the table has table_count rows)
  long tokens, rows;          // rows = tokens * group: columns of a kv head
  int q_heads, kv_heads, page_shift, shared, max_own, max_new;
  long num_pages;
  float scale_log2;
  Divider group;
  int prefix_segments, prefix_keys;    // segments of the prefix and keys of one
  int own_segments, own_keys;          // the same of a request's own keys
  int prefix_tiles, own_tiles;         // tiles of columns: of all rows, of the most rows a request brings
  long prefix_blocks;
  const int* prefix_pages;    // the prompt's pages, or null: they are read from the first request's row
};

// What the host could not see of a request: whether its tokens lie within q, its lengths within the bounds and behind the prompt.  The
// walks leave other requests alone, and the join answers their tokens with NaN.
__device__ __forceinline__ bool within_bounds(const Args& a, int begin, int count, int length) {
  return begin >= 0 && count > 0 && count <= a.max_new && static_cast<long>(begin) + count <= a.tokens && length >= count &&
         length - count >= a.shared && length - a.shared <= a.max_own;
}
// A request's row of the table, or null where there is none.
__device__ __forceinline__ const int* table_of(const Args& a, int request) {
  const int row = a.table_rows != nullptr ? a.table_rows[request] : request;
  return row < 0 || row >= a.table_count ? nullptr : a.block_table + static_cast<size_t>(row) * a.table_width;
}

// Eight neighbouring elements of an operand: what a lane holds of 16 dims (or keys).
template <typename T> struct Piece;
template <> struct Piece<bf16_t> { uintx4 v; };
template <> struct Piece<float> { floatx4 low, high; };

template <typename T> __device__ __forceinline__ Piece<T> load_piece(const T* at);
template <> __device__ __forceinline__ Piece<bf16_t> load_piece<bf16_t>(const bf16_t* at) { return {*reinterpret_cast<const uintx4*>(at)}; }
template <> __device__ __forceinline__ Piece<float> load_piece<float>(const float* at) {
  return {*reinterpret_cast<const floatx4*>(at), *reinterpret_cast<const floatx4*>(at + 4)};
}
__device__ __forceinline__ Piece<bf16_t> empty_piece(bf16_t) { return {uintx4{0u, 0u, 0u, 0u}}; }
__device__ __forceinline__ Piece<float> empty_piece(float) { return {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}}; }

// What stays of a piece whose first `count` elements are there.
__device__ __forceinline__ void keep_first(Piece<bf16_t>& p, int count) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (2 * i >= count) p.v[i] = 0u;
    else if (2 * i + 1 >= count) p.v[i] &= 0xffffu;
  }
}
__device__ __forceinline__ void keep_first(Piece<float>& p, int count) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= count) p.low[i] = 0.f;
    if (i + 4 >= count) p.high[i] = 0.f;
  }
}
__device__ __forceinline__ bool all_finite(const Piece<bf16_t>& p) {
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) fine = fine && (p.v[i] & 0x7f80u) != 0x7f80u && (p.v[i] & 0x7f800000u) != 0x7f800000u;
  return fine;
}
__device__ __forceinline__ bool all_finite(const Piece<float>& p) {
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) fine = fine && fabsf(p.low[i]) < INFINITY && fabsf(p.high[i]) < INFINITY;
  return fine;
}

__device__ __forceinline__ void keep_finite(Piece<bf16_t>& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((p.v[i] & 0x7f80u) == 0x7f80u) p.v[i] &= 0xffff0000u;
    if ((p.v[i] & 0x7f800000u) == 0x7f800000u) p.v[i] &= 0xffffu;
  }
}
__device__ __forceinline__ void keep_finite(Piece<float>& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!(fabsf(p.low[i]) < INFINITY)) p.low[i] = 0.f;
    if (!(fabsf(p.high[i]) < INFINITY)) p.high[i] = 0.f;
  }
}

__device__ __forceinline__ floatx16 multiply(const Piece<bf16_t>& a, const Piece<bf16_t>& b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 multiply(const Piece<float>& a, const Piece<float>& b, floatx16 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.low[i], b.low[i], c, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.high[i], b.high[i], c, 0, 0, 0);
  return c;
}

// O += V^T P for 16 keys, `p` a lane's eight weights.  In bfloat16 the weights go in two parts, the rounded one and what the
// rounding left: the sum is then as exact as the 32-bit weights, and here, where reads are what counts, costs nothing.
__device__ __forceinline__ floatx16 weigh(const Piece<bf16_t>& v, const float* p, floatx16 c) {
  Piece<bf16_t> high, low;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    high.v[i] = bf16_pair(p[2 * i], p[2 * i + 1]);
    low.v[i] = bf16_pair(p[2 * i] - __uint_as_float(high.v[i] << 16), p[2 * i + 1] - __uint_as_float(high.v[i] & 0xffff0000u));
  }
  return multiply(v, low, multiply(v, high, c));
}
__device__ __forceinline__ floatx16 weigh(const Piece<float>& v, const float* p, floatx16 c) {
  const Piece<float> w{floatx4{p[0], p[1], p[2], p[3]}, floatx4{p[4], p[5], p[6], p[7]}};
  return multiply(v, w, c);
}

// The same value of the other half's lane joined in: lanes l and l + 32 hold the same column.
__device__ __forceinline__ float max_over_halves(float v) {
  const uint32_t bits = __float_as_uint(v);
  const auto swapped = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
  return fmaxf(__uint_as_float(swapped[0]), __uint_as_float(swapped[1]));
}
__device__ __forceinline__ float sum_over_halves(float v) {
  const uint32_t bits = __float_as_uint(v);
  const auto swapped = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
  return __uint_as_float(swapped[0]) + __uint_as_float(swapped[1]);
}

// One tile of 32 columns over the keys first_key .. end_key - 1, by WAVES waves in turn, 32 keys a step: the block's, or one of its
// TEAMS, which take a tile each (none: `columns` and keys of 0).
// `row0`: the tile's first row of the kv head's, `columns` how many of the 32 are there.  A column sees the keys below `visible`
// (its lane's), `all_see` the least of them over the tile.  `wanted`: a bit for each column whose results are written.
// Reads and their latency are what bounds it where there are few columns, 16 KB a step asked for a step ahead: own keys of 64 requests of
// 328 each, 86 MB, 19 us (4.5 TB/s), of 4 to 2,048 26 us; 8 requests behind 8,192 shared tokens, 42 MB in all, 13.0 us, of which 8 are the
// way to the first keys - launch, page, read - and the results' way back.  A block alone on its unit takes 2.8 us a step of its four
// waves.  With a wave a vector unit and many tiles a step takes 1.4 us: 0.35 of matrix instructions, as much of exponentials, the rest
// waits for operands whose rows' 32-byte pieces are fetched line by line (`walk_wide` has them in LDS).
template <typename T, int WAVES, int TEAMS = 1>
__device__ __forceinline__ void walk(const Args& a, const int* table, int head, long row0, int columns, int first_key, int end_key,
                                     int visible, int all_see, int segment, float* lds, uint32_t wanted = 0xffffffffu) {
  constexpr int kBuffers = WAVES / 2;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave % WAVES, thread = threadIdx.x % (WAVES * kWave);
  if (TEAMS > 1) lds += __builtin_amdgcn_readfirstlane(threadIdx.x / (WAVES * kWave)) * (narrow_lds<T>(WAVES) / sizeof(float));
  const int r = lane & 31, half = lane >> 5;
  const int group = static_cast<int>(a.group.by), segments = a.prefix_segments + a.own_segments;
  const int page_mask = (1 << a.page_shift) - 1;
  // in LDS: half the waves' results, a row a column; every wave's maxima and sums; what a column sees; the queries, as operands
  float* shares = lds + kBuffers * 32 * kRow;         // [waves][32][2]
  // [32], whether a masked value was not finite, a bit for each column without a result (its sum of weights is NaN)
  int* seen = reinterpret_cast<int*>(shares + WAVES * 32 * 2);
  Piece<T>* queries = reinterpret_cast<Piece<T>*>(seen + 64);       // [KC][lane]
  // the key of a step that this lane's row of A holds
  const int key_at = 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3);
  bool bad = false;
  // A step's loads are asked for while the step before is worked on - its keys when those before have been multiplied, its values when
  // those before have -, and what the table says of their pages a step earlier still.
  int key_page = 0, value_pages[2] = {0, 0};
  auto lookup = [&](int base) {
    key_page = table[min(base + key_at, end_key - 1) >> a.page_shift];
#pragma unroll
    for (int c = 0; c < 2; ++c) value_pages[c] = table[min(base + 16 * c + 8 * half, end_key - 1) >> a.page_shift];
  };
  auto place_of = [&](int page) {
    const bool outside = page < 0 || page >= a.num_pages;
    bad |= outside;
    return static_cast<size_t>(outside ? 0 : page) * a.kv_heads + head;
  };
  const int first_base = first_key + 32 * wave;
  if (first_base < end_key) lookup(first_base);
  for (int c = wave; c < KC && (TEAMS == 1 || columns > 0); c += WAVES) {
    const long row = row0 + min(r, columns - 1);
    const long token = group == 1 ? row : row / group;
    const T* q = static_cast<const T*>(a.q) + (token * a.q_heads + static_cast<long>(head) * group + (row - token * group)) * D + 8 * half;
    queries[c * kWave + lane] = load_piece<T>(q + 16 * c);
  }
  if (wave == 0 && half == 0) seen[r] = visible;
  if (thread == 0) seen[32] = 0;
  Piece<T> kf[KC], vf[2][DT];
  auto fetch_keys = [&](int base, int page) {
    const int key = min(base + key_at, end_key - 1);
    const T* k = static_cast<const T*>(a.k_pages) + ((place_of(page) << a.page_shift) + (key & page_mask)) * D + 8 * half;
#pragma unroll
    for (int c = 0; c < KC; ++c) kf[c] = load_piece<T>(k + 16 * c);
  };
  auto fetch_values = [&](int base, const int (&pages)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int octet = min(base + 16 * c + 8 * half, (end_key - 1) & ~7);
      const T* v = static_cast<const T*>(a.v_pages) + ((place_of(pages[c]) * D + r) << a.page_shift) + (octet & page_mask);
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        if (D % 32 == 0 || t + 1 < DT || r < 16) vf[c][t] = load_piece<T>(v + (static_cast<size_t>(32 * t) << a.page_shift));
        else vf[c][t] = empty_piece(T{});
      }
    }
  };
  floatx16 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  float m = -INFINITY, l = 0.f;       // (m is the column's, l what this lane's keys add to its sum)
  bool odd = false;                   // whether a value that some column does not see was not finite
  if (first_base < end_key) {
    fetch_keys(first_base, key_page);
    fetch_values(first_base, value_pages);
    if (first_base + 32 * WAVES < end_key) lookup(first_base + 32 * WAVES);
  }
  __syncthreads();
  for (int base = first_base; base < end_key; base += 32 * WAVES) {
    floatx16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; ++c) s = multiply(kf[c], queries[c * kWave + lane], s);
    const bool more = base + 32 * WAVES < end_key;
    const int next_pages[2] = {value_pages[0], value_pages[1]};
    if (more) {
      fetch_keys(base + 32 * WAVES, key_page);
      if (base + 64 * WAVES < end_key) lookup(base + 64 * WAVES);
    }
    const bool ends = base + 32 > end_key, masked = all_see < end_key && base + 32 > all_see;
    if (ends || masked) {
      const int limit = min(visible, end_key) - base - 8 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (16 * (i >> 3) + (i & 7) >= limit) s[i] = -INFINITY;
    }
    if (ends) {     // what lies behind the last key is not multiplied: it may be anything
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < DT; ++t) keep_first(vf[c][t], end_key - (base + 16 * c + 8 * half));
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
    const float m_new = fmaxf(m, max_over_halves(top) * a.scale_log2);
    const float reference = m_new == -INFINITY ? 0.f : m_new;
    if (__any(m_new > m)) {
      const float by = __builtin_amdgcn_exp2f(m - reference);
      l *= by;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= by;
    }
    m = m_new;
    float p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale_log2, -reference));
      l += p[i];
    }
    if (masked) {
      // A key that some column does not see may have a value that is not finite, and 0 times it would reach that column: such values are
      // left out of the product, and added to the columns that see their key when the results are written.
      bool fine = true;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int t = 0; t < DT; ++t) fine = fine && all_finite(vf[c][t]);
      if (!__all(fine)) {
        odd = true;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int t = 0; t < DT; ++t) keep_finite(vf[c][t]);
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int t = 0; t < DT; ++t) o[t] = weigh(vf[c][t], p + 8 * c, o[t]);
    if (more) fetch_values(base + 32 * WAVES, next_pages);
  }
  l = sum_over_halves(l);
  if (__any(bad)) m = l = NAN;
  // the waves' results, joined through LDS: half of the waves hand theirs to the others, whose sums the block adds up
  if (half == 0) { shares[(wave * 32 + r) * 2] = m; shares[(wave * 32 + r) * 2 + 1] = l; }
  if (odd && lane == 0) seen[32] = 1;          // (every writer stores the same value)
  __syncthreads();
  float top = -INFINITY, whole = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, shares[(w * 32 + r) * 2]);
  const float reference = top == -INFINITY ? 0.f : top;
  if (wave == 0) {      // (which hands on nothing in the first turn below)
#pragma unroll
    for (int w = 0; w < WAVES; ++w) whole += shares[(w * 32 + r) * 2 + 1] * __builtin_amdgcn_exp2f(shares[(w * 32 + r) * 2] - reference);
    const unsigned long long lost = __ballot(whole != whole);
    if (lane == 0) seen[33] = static_cast<int>(lost);
  }
  const float by = __builtin_amdgcn_exp2f(m - reference);
  float* mine = lds + ((wave % kBuffers) * 32 + r) * kRow;
#pragma unroll
  for (int turn = 0; turn < 2; ++turn) {
    if ((wave < kBuffers) == (turn == 1) && r < columns) {
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int dim = 32 * t + 8 * q + 4 * half;
          if (D % 32 == 0 || dim < D) {
            floatx4 four = {o[t][4 * q] * by, o[t][4 * q + 1] * by, o[t][4 * q + 2] * by, o[t][4 * q + 3] * by};
            floatx4* at = reinterpret_cast<floatx4*>(mine + dim);
            *at = turn == 0 ? four : four + *at;
          }
        }
    }
    __syncthreads();
  }
  if (wave == 0 && half == 0 && r < columns && ((wanted >> r) & 1u) != 0u) {
    float* at = a.stats + ((static_cast<size_t>(head) * a.rows + row0 + r) * segments + segment) * 2;
    at[0] = top;
    at[1] = whole;
  }
  float* sums = a.sums + ((static_cast<size_t>(head) * segments + segment) * a.rows + row0) * D;
  const bool any_odd = seen[32] != 0;
  for (int i = thread; i < columns * (D / 4); i += WAVES * kWave) {
    const int column = i / (D / 4), at = i % (D / 4) * 4;
    if (((wanted >> column) & 1u) == 0u) continue;
    floatx4 sum = *reinterpret_cast<const floatx4*>(lds + column * kRow + at);
#pragma unroll
    for (int w = 1; w < kBuffers; ++w) sum += *reinterpret_cast<const floatx4*>(lds + (w * 32 + column) * kRow + at);
    // A value that is not finite makes the sum what it is itself, however small its weight.  The product does not: 0 times it is NaN, where the
    // weight is less than 32 bits hold or its second part is nothing, and so is what a negative second part takes from infinity.  So where a
    // sum is not finite such values are looked for among all keys, and else among those that were left out of the product.
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) finite = finite && fabsf(sum[e]) < INFINITY;
    if ((any_odd || !finite) && ((seen[33] >> column) & 1) == 0) {
      floatx4 odd = {0.f, 0.f, 0.f, 0.f};
      for (int j = finite ? first_key + (max(0, all_see - first_key) & ~31) : first_key; j < min(end_key, seen[column]); ++j) {
        const size_t place = place_of(table[j >> a.page_shift]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = to_float(static_cast<const T*>(a.v_pages)[((place * D + at + e) << a.page_shift) + (j & page_mask)]);
          if (!(fabsf(v) < INFINITY)) odd[e] += v;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (odd[e] != 0.f) sum[e] = odd[e];
    }
    *reinterpret_cast<floatx4*>(sums + static_cast<size_t>(column) * D + at) = sum;
  }
}

// ---- a prompt's keys for many columns ---------------------------------------------------------------------------------------
// bfloat16 heads of 64 and 128 on pages of 16 tokens and more.  A block's eight waves take 32 columns each and share the keys and values
// of 64 tokens, a stage, through LDS, which loads write directly (16 bytes a lane in the lanes' order), in rings of four stages.  In
// LDS a key's row stands where the matrix instruction wants it, its pieces of 16 bytes exchanged by the row's number, and values lie
// [16 keys][32 dims] one operand after the other: every read of an operand is a run of 1 KB or goes over all banks.
// A turn multiplies the scores of step u + 1 (32 keys), turns those of step u into weights and adds the values of step u - 1: the three
// do not wait for each other, and nothing in it depends on what the scores are.  A column's weights are taken below a fixed point,
// the maximum of the segment's first step, and may grow: bfloat16 and float32 reach to 2^127, and a sum that is divided by another of the
// same scale loses nothing.  Where a column's weights pass 2^40, its sums are not finite, or there is no such point (nothing but minus
// infinity, a NaN), the column is done again by `walk`, which keeps a running maximum: what a column gets hangs on nothing beside it.
// (A branch that moves the point in the loop costs it half as much again: the compiler then keeps the sums in two sets of registers.)
// That is dear where it is met - a block does its groups of 32 columns one after the other: 256 columns of 8 heads over 32,768 keys,
// calls, 77 us, and 173 where every head looks at one key 28 nats above its segment's first 32, 222 where each segment has such a
// key; 2,560 over 8,192 131 and 353 (in narrow tiles, the same keys, 100 and 253 us).
// The weights are rounded to bfloat16, once: a second part would cost half the matrix instructions again, and the sum that they are
// divided by is the sum of the rounded ones, so that what is left is the error of an average over the keys.
// What bounds it: the matrix cores while it runs, 1.68 us a stage of 64 keys on all units (1.28 PFLOP/s; a large library product has
// 1.34), and 18 us before and behind: the launch, the way to the first stages (6 us), 128 KB of sums a unit that leave at the end (6).
// 256 columns of 8 heads over 32,768 keys 46 us (0.75 PFLOP/s), 2,560 over 8,192 93 us (0.92).
constexpr bool kWideFits = D == 64 || D == 128;
constexpr int kWideWaves = 8, kWideColumns = 32 * kWideWaves;
constexpr int kStepBytes = (kWideFits ? 32 * D : 32 * 64) * 2, kStageBytes = 2 * kStepBytes;      // of a step's or a stage's keys, and of its values
constexpr int kWideLoads = kStageBytes / 1024 / kWideWaves;               // instructions a wave for a stage's keys, and for its values
constexpr size_t kWideLds = 8 * kStageBytes, kWideNarrowLds = kWideFits ? narrow_lds<bf16_t>(kWideWaves) : 0;
constexpr float kLimit = 0x1p40f;  // what a lane's sixteen weights of a step may sum up to

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// Waits until all but the wave's last `COUNT` loads and all its reads of LDS have arrived, then for the block's other waves.
template <int COUNT> __device__ __forceinline__ void arrived() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(COUNT) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// 16 bytes a lane into LDS at `to` (and on, in the lanes' order).  As text: the compiler would wait for every load before the next
// read of LDS; the turns' counted waits order them.  No register is written.
__device__ __forceinline__ void load_to_lds(const char* from, uint32_t offset, uint32_t to) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(from) : "m0", "memory");
#pragma clang diagnostic pop
}

// Leaves in over[wave] a bit for each of a wave's columns whose weights passed their bounds, and writes the others.
__device__ __forceinline__ void walk_wide(const Args& a, const int* table, int head, long row0, long rows, int first_key, int end_key,
                                          int segment, float* lds, uint32_t* over_of) {
  typedef const __attribute__((address_space(3))) char* lds_chars;
  // (the table is not written while the kernel runs: read as constant memory, by the scalar unit, or each lookup would be a wait for
  // every load on its way)
  typedef const __attribute__((address_space(4))) int* constant_ints;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 31, half = lane >> 5;
  const int group = static_cast<int>(a.group.by);
  const long my_row = row0 + 32 * wave + r;
  const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_chars)(reinterpret_cast<char*>(lds))));
  // what this wave fetches of a stage: half of the rows or operands of one of its four pieces of 16 keys, 1 KB an instruction
  const int chunk = wave >> 1;
  uint32_t key_from[kWideLoads], value_from[kWideLoads];
#pragma unroll
  for (int i = 0; i < kWideLoads; ++i) {
    const int n = wave * kWideLoads + i;
    constexpr int kPieces = D / 8, kRows = 64 / kPieces;         // pieces of a row, rows of an instruction
    const int row = n * kRows + lane / kPieces, slot = lane % kPieces;
    const int piece = slot ^ (D == 128 ? row & 15 : (row >> 1) & 7);
    const int key = 8 * ((row >> 2) & 1) + 4 * ((row >> 3) & 1) + (row & 3);      // (within the 16)
    key_from[i] = static_cast<uint32_t>(key * D * 2 + piece * 16);
    const int dim = n % DT * 32 + r;
    value_from[i] = (static_cast<uint32_t>(dim) << (a.page_shift + 1)) + half * 16u;
  }
  const int steps = (end_key - first_key + 31) / 32, stages = (steps + 1) / 2;
  const int last_chunk = (end_key - 1) & ~15, page_mask = (1 << a.page_shift) - 1;
  const uint32_t page_count = static_cast<uint32_t>(min(a.num_pages, 0x7fffffffL));
  const size_t page_bytes = static_cast<size_t>(D * 2) << a.page_shift, head_bytes = page_bytes * head;
  const size_t block_bytes = page_bytes * a.kv_heads;
  bool bad = false;
  const constant_ints pages = (constant_ints)reinterpret_cast<uintptr_t>(table);
  // (pieces behind the last key are fetched from the last one's page: their scores are masked, their values left out)
  auto key_of = [&](int stage) { return min(first_key + stage * 64 + 16 * chunk, last_chunk); };
  auto lookup = [&](int stage) { return pages[key_of(stage) >> a.page_shift]; };
  auto page_at = [&](int page) {
    const bool outside = static_cast<uint32_t>(page) >= page_count;
    bad |= outside;
    return static_cast<size_t>(outside ? 0 : page) * block_bytes + head_bytes;
  };
  auto fetch_keys = [&](int stage, size_t page) {
    if (stage >= stages) return;
    const char* from = static_cast<const char*>(a.k_pages) + page + static_cast<uint32_t>(key_of(stage) & page_mask) * (D * 2u);
    const uint32_t to = lds_at + (stage & 3) * kStageBytes + wave * kWideLoads * 1024u;
#pragma unroll
    for (int i = 0; i < kWideLoads; ++i) load_to_lds(from, key_from[i], to + i * 1024u);
  };
  auto fetch_values = [&](int stage, size_t page) {
    if (stage >= stages) return;
    const char* from = static_cast<const char*>(a.v_pages) + page + static_cast<uint32_t>(key_of(stage) & page_mask) * 2u;
    const uint32_t to = lds_at + (4 + (stage & 3)) * kStageBytes + wave * kWideLoads * 1024u;
#pragma unroll
    for (int i = 0; i < kWideLoads; ++i) load_to_lds(from, value_from[i], to + i * 1024u);
  };
  Piece<bf16_t> qf[KC];
  {
    const long row = min(my_row, rows - 1), token = group == 1 ? row : row / group;
    const bf16_t* q = static_cast<const bf16_t*>(a.q) + (token * a.q_heads + static_cast<long>(head) * group + (row - token * group)) * D + 8 * half;
#pragma unroll
    for (int c = 0; c < KC; ++c) qf[c] = load_piece<bf16_t>(q + 16 * c);
  }
  // After the middle of stage T's turns nobody reads its keys or the values before it any more: stage T + 4's keys and T + 3's values are
  // asked for there, where stage T + 2's keys and T + 1's values, asked for two stages earlier, have to have arrived (a turn ends with
  // reads for the next one).
  size_t at0 = page_at(lookup(0)), at1 = page_at(lookup(min(1, stages - 1))), at2 = page_at(lookup(min(2, stages - 1)));
  size_t at3 = page_at(lookup(min(3, stages - 1)));
  int pending = lookup(min(4, stages - 1));
  fetch_keys(0, at0);
  fetch_keys(1, at1); fetch_values(0, at0);
  fetch_keys(2, at2); fetch_values(1, at1);
  auto meet = [&](int stage) {
    constexpr int kL = kWideLoads;
    if (stage + 3 < stages) arrived<2 * kL>();
    else if (stage + 2 < stages) arrived<kL>();
    else arrived<0>();
  };
  char* ring = reinterpret_cast<char*>(lds);
  // (the first turn adds the values of a step -1, of no weight: zeros, until the fourth stage's values come)
  for (int i = threadIdx.x; i < kStepBytes / 16; i += kWideWaves * kWave)
    *reinterpret_cast<uintx4*>(ring + 7 * kStageBytes + kStepBytes + i * 16) = uintx4{0u, 0u, 0u, 0u};
  meet(-1);
  fetch_keys(3, at3); fetch_values(2, at2);

  floatx16 o[DT], s[2];                    // (scores and weights of two steps, by the step's parity)
  Piece<bf16_t> weights[2][2];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[t][i] = 0.f;
  weights[1][0] = weights[1][1] = empty_piece(bf16_t{});
  const bf16x2 ones = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
  // Where a step's operands begin, hidden from the compiler, which would otherwise add up each operand's place by itself (beyond 64 KB of
  // LDS places do not fit an instruction).  A key's piece is found by the exchange of the bits above its half, values lie in a row.
  typedef const __attribute__((address_space(3))) uintx4* lds_pieces;
  const uint32_t key_lane = lds_at + r * (D * 2u) + ((half ^ (D == 128 ? r & 15 : (r >> 1) & 7)) << 4);
  const uint32_t value_lane = lds_at + 4 * kStageBytes + lane * 16;
  auto keys_of = [&](int stage, int which) {
    uint32_t at = key_lane + ((stage & 3) * kStageBytes + which * kStepBytes);
    asm volatile("" : "+v"(at));
    return at;
  };
  auto values_of = [&](int stage, int which) {
    uint32_t at = value_lane + ((stage & 3) * kStageBytes + which * kStepBytes);
    asm volatile("" : "+v"(at));
    return at;
  };
  auto key_operand = [&](uint32_t at, int c) { return *(lds_pieces)(at ^ (c << 5)); };
  auto value_operand = [&](uint32_t at, int n) { return *(lds_pieces)(at + n * 1024); };
  uint32_t keys = keys_of(0, 0);
#pragma unroll
  for (int i = 0; i < 16; ++i) s[0][i] = 0.f;
#pragma unroll
  for (int c = 0; c < KC; ++c) s[0] = multiply(Piece<bf16_t>{key_operand(keys, c)}, qf[c], s[0]);
  float below = s[0][0], l = 0.f;
#pragma unroll
  for (int i = 1; i < 16; ++i) below = fmaxf(below, s[0][i]);
  if (end_key - first_key < 32) {      // (one step of 16 keys: the others are no scores)
    below = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) below = fmaxf(below, s[0][i]);
  }
  below = max_over_halves(below) * a.scale_log2;
  bool over = !(fabsf(below) < INFINITY);
  auto pair_of = [&](const floatx16& x, int i) {
    return bf16_pair(__builtin_amdgcn_exp2f(fmaf(x[i], a.scale_log2, -below)), __builtin_amdgcn_exp2f(fmaf(x[i + 1], a.scale_log2, -below)));
  };
  // A turn's order is written down: a matrix instruction, the read of the operand four further on (the next turn's at its end), and as
  // much of the weights as the vector unit does in the meantime.  The scores come first, so that they are there when the next turn
  // begins.  `second`: whether step u is a stage's second, known to the compiler: no scores or weights are moved from one turn to the next.
  constexpr int kSlots = 2 * KC, kAhead = 4;
  Piece<bf16_t> operand[kAhead];
  keys = keys_of(0, 1);
#pragma unroll
  for (int n = 0; n < kAhead; ++n) operand[n].v = key_operand(keys, n);
  auto turn = [&](int stage, auto second) {
    constexpr int B = decltype(second)::value;
    floatx16 &now = s[B], &next = s[1 - B];
    Piece<bf16_t> (&made)[2] = weights[B], (&before)[2] = weights[1 - B];
#pragma unroll
    for (int i = 0; i < 16; ++i) next[i] = 0.f;
    float sum = 0.f;
    const uint32_t values = values_of(stage - 1 + B, 1 - B), further = keys_of(stage + 1, B);
#pragma unroll
    for (int n = 0; n < kSlots; ++n) {
      if (n < KC) next = multiply(operand[n % kAhead], qf[n], next);
      else o[(n - KC) % DT] = multiply(operand[n % kAhead], before[(n - KC) / DT], o[(n - KC) % DT]);
      if (n + kAhead < KC) operand[n % kAhead].v = key_operand(keys, n + kAhead);
      else if (n + kAhead < kSlots) operand[n % kAhead].v = value_operand(values, n + kAhead - KC);
      else operand[n % kAhead].v = key_operand(further, n + kAhead - kSlots);
#pragma unroll
      for (int i = 16 * n / kSlots; i < 16 * (n + 1) / kSlots; ++i)
        if ((i & 1) != 0) {
          const uint32_t pair = pair_of(now, i - 1);
          made[i >> 3].v[(i & 7) >> 1] = pair;
          sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), ones, sum, false);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
    asm volatile("" : "+v"(made[0].v), "+v"(made[1].v), "+v"(sum));     // (made here, beside the products, not where they are used)
    over |= !(sum <= kLimit);
    l += sum;
    keys = further;
  };
  typedef std::integral_constant<int, 0> first;
  typedef std::integral_constant<int, 1> second;
  int stage = 0;
  for (; 2 * stage + 2 < steps; ++stage) {
    turn(stage, first{});
    at2 = at3;
    at3 = page_at(pending);
    pending = lookup(min(stage + 5, stages - 1));
    meet(stage);
    fetch_keys(stage + 4, at3);
    fetch_values(stage + 3, at2);
    turn(stage, second{});
  }
  // the last step: values of the one before it, then its own
  auto add_values = [&](int of_stage, int which, const Piece<bf16_t> (&w)[2], int chunks) {
    const uint32_t values = values_of(of_stage, which);
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (c < chunks)
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = multiply(Piece<bf16_t>{value_operand(values, c * DT + t)}, w[c], o[t]);
  };
  const int there = end_key - first_key - (steps - 1) * 32;     // keys of the last step: 16 or 32
  int second_step = 0;
  if (2 * stage + 1 < steps) {
    turn(stage, first{});
    second_step = 1;
    s[0] = s[1];
    weights[1][0] = weights[0][0];
    weights[1][1] = weights[0][1];
  }
  arrived<0>();
  add_values(stage - 1 + second_step, 1 - second_step, weights[1], 2);
  if (there < 32) {
#pragma unroll
    for (int i = 8; i < 16; ++i) s[0][i] = -INFINITY;
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    const uint32_t pair = pair_of(s[0], i);
    weights[0][i >> 3].v[(i & 7) >> 1] = pair;
    sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), ones, sum, false);
  }
  over |= !(sum <= kLimit);
  l += sum;
  add_values(stage, second_step, weights[0], there < 32 ? 1 : 2);
  // (a column whose sums are not finite is done again too: its weights may be above one, and values may be infinite)
  float nothing = 0.f;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) nothing = fmaf(o[t][i], 0.f, nothing);
  over |= nothing != 0.f;
  l = sum_over_halves(l);
  const unsigned long long passed = __ballot(over && my_row < rows);
  const uint32_t mask = static_cast<uint32_t>(passed) | static_cast<uint32_t>(passed >> 32);
  if (lane == 0) over_of[wave] = mask;
  const bool spoilt = __syncthreads_or(bad);
  if (my_row >= rows || ((mask >> r) & 1u) != 0u) return;
  const int segments = a.prefix_segments + a.own_segments;
  if (half == 0) {
    float* at = a.stats + ((static_cast<size_t>(head) * a.rows + my_row) * segments + segment) * 2;
    at[0] = below;
    at[1] = spoilt ? NAN : l;
  }
  float* sums = a.sums + ((static_cast<size_t>(head) * segments + segment) * a.rows + my_row) * D + 4 * half;
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<floatx4*>(sums + 32 * t + 8 * i) = floatx4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
}

// Blocks go to the XCDs in turn: the tiles of one item, which read the same pages, stand eight apart, on one XCD and in its cache.
__device__ __forceinline__ void tile_of(long block, long items, int tiles, long& item, int& tile) {
  const long run = block / (static_cast<long>(kXcds) * tiles) * kXcds, in_run = block - run * tiles, wide = min(static_cast<long>(kXcds), items - run);
  tile = static_cast<int>(in_run / wide);
  item = run + in_run % wide;
}

// Blocks take (segment and head, tile of 256 columns) of the prefix.
__global__ __launch_bounds__(kWideWaves * kWave, 2) void wide_prefix_kernel(Args a) {
  extern __shared__ __attribute__((aligned(1024))) float aligned_lds[];     // (a row's pieces are exchanged by the low bits of their places)
  float* lds = aligned_lds;
  long item;
  int tile;
  tile_of(blockIdx.x, static_cast<long>(a.prefix_segments) * a.kv_heads, a.prefix_tiles, item, tile);
  const int head = static_cast<int>(item % a.kv_heads), segment = static_cast<int>(item / a.kv_heads);
  const int first = segment * a.prefix_keys, end = min(a.shared, first + a.prefix_keys);
  const int* table = table_of(a, 0);
  // (rows behind the last request's may hold anything, and nobody asks for them)
  const long rows = min(a.rows, static_cast<long>(max(a.q_start[a.requests], 0)) * static_cast<long>(a.group.by));
  const long row0 = static_cast<long>(kWideColumns) * tile;
  __shared__ uint32_t over[kWideWaves];
  if (row0 >= rows || table == nullptr) return;
  walk_wide(a, table, head, row0, rows, first, end, segment, lds, over);
  for (int w = 0; w < kWideWaves; ++w) {
    if (over[w] == 0u) continue;
    __syncthreads();
    const long at = row0 + 32 * w;
    walk<bf16_t, kWideWaves>(a, table, head, at, static_cast<int>(min(32L, rows - at)), first, end, end, end, segment, lds, over[w]);
  }
}

// Sums over the lanes up to each, inside the vector unit: four shifts within rows of 16 lanes, two broadcasts of a row's last lane.
template <int CTRL, int ROWS> __device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int sums_up_to(int v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}

// The `number`-th of the segments that the requests' own keys fill, request by request: the grid has blocks for as many as the longest
// request may fill in each, and those that are not there come last - between the others they would keep the units from work for a
// microsecond each (64 requests of 4 to 2,048 keys in segments of 256: 33 -> 27 us; 27 of up to 2,000: 20 -> 15).  False behind the last.
__device__ __forceinline__ bool own_item(const Args& a, long number, int& request, int& segment, int& begin, int& count, int& length) {
  const int lane = threadIdx.x & (kWave - 1);
  if (a.own_segments == 1) {
    request = static_cast<int>(number);
    segment = 0;
    begin = a.q_start[request];
    count = a.q_start[request + 1] - begin;
    length = a.seq_lens[request];
    return within_bounds(a, begin, count, length);
  }
  for (int r0 = 0; r0 < a.requests; r0 += kWave) {
    const int r = min(r0 + lane, a.requests - 1);
    const int from = a.q_start[r], brings = a.q_start[r + 1] - from, holds = a.seq_lens[r];
    const int filled = r0 + lane < a.requests && within_bounds(a, from, brings, holds) ? (holds - a.shared + a.own_keys - 1) / a.own_keys : 0;
    const int upto = sums_up_to(filled), all = __builtin_amdgcn_readlane(upto, kWave - 1);
    if (number < all) {
      const int at = __builtin_ctzll(__ballot(upto > number));
      request = r0 + at;
      segment = static_cast<int>(number) - __builtin_amdgcn_readlane(upto - filled, at);
      begin = __builtin_amdgcn_readlane(from, at);
      count = __builtin_amdgcn_readlane(brings, at);
      length = __builtin_amdgcn_readlane(holds, at);
      return true;
    }
    number -= all;
  }
  return false;
}

// Blocks 0 .. prefix_blocks - 1 take (segment and head, tile) of the prefix, the others (request, head, two tiles, segment) of the
// requests' own keys.  GIVEN: the prompt's pages are `prefix_pages` (a kernel of its own: the choice costs registers and half a microsecond).
template <typename T, bool GIVEN>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 4 || D > 128 ? 1 : 2)) void shared_prefix_kernel(Args a) {
  extern __shared__ float lds[];
  long block = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1), r = lane & 31;
  int head, segment, request = 0, columns, first, end, visible, all_see, tile;
  long row0, item;
  const bool of_prefix = block < a.prefix_blocks;
  if (of_prefix) {
    tile_of(block, static_cast<long>(a.prefix_segments) * a.kv_heads, a.prefix_tiles, item, tile);
    head = static_cast<int>(item % a.kv_heads);
    segment = static_cast<int>(item / a.kv_heads);
    row0 = 32L * tile;
    columns = static_cast<int>(min(32L, a.rows - row0));
    first = segment * a.prefix_keys;
    visible = all_see = end = min(a.shared, first + a.prefix_keys);
  } else {
    block -= a.prefix_blocks;
    tile_of(block, static_cast<long>(a.requests) * a.kv_heads * a.own_segments, (a.own_tiles + 1) / 2, item, tile);
    head = static_cast<int>(item % a.kv_heads);
    int begin, count, length;
    if (!own_item(a, item / a.kv_heads, request, segment, begin, count, length)) return;
    const int before = length - count;
    const int group = static_cast<int>(a.group.by), left = count * group - 64 * tile;
    if (left <= 0) return;
    // two tiles, where a request brings them, for half of the waves each: what one reads the other finds in the unit's cache (64 requests
    // of 40 rows a head, calls with equal lengths of 517 139 -> 134 us, with lengths up to that 93 -> 89)
    const bool pair = left > 32;
    const int column0 = 64 * tile + (pair ? 32 * __builtin_amdgcn_readfirstlane(threadIdx.x / (kThreads / 2)) : 0);
    columns = min(32, count * group - column0);
    first = a.shared + segment * a.own_keys;
    end = min(before + a.group.quotient(column0 + columns - 1) + 1, first + a.own_keys);       // (what the tile's last token sees)
    if (first >= end) {
      if (!pair) return;
      columns = 0;
    }
    visible = before + a.group.quotient(column0 + min(r, max(columns, 1) - 1)) + 1;
    all_see = before + a.group.quotient(column0) + 1;
    row0 = static_cast<long>(begin) * group + column0;
    segment += a.prefix_segments;
    if (pair) {
      const int* table = table_of(a, request);
      if (table != nullptr) walk<T, kWaves / 2, 2>(a, table, head, row0, columns, first, end, visible, all_see, segment, lds);
      return;
    }
  }
  const int* table = GIVEN && of_prefix ? a.prefix_pages : table_of(a, request);
  if (table == nullptr) return;
  walk<T, kWaves>(a, table, head, row0, columns, first, end, visible, all_see, segment, lds);
}

// A row - (token, query head) - a wave, four of a token a block, or, SHARE, where there are too few rows to fill the device, a block: its
// waves then take the segments in turn.  What a row waits for is a chain of reads - whose the token is, what it sees -, so many
// short waves run beside each other, and the segments that a row is sure to have are on their way meanwhile (20,480 rows of four segments
// 13.9 -> 12.2 us, 43 MB read and 5 written; 2,048 rows of 33 to 38: 8.9 us for 36 MB).
template <typename T, bool SHARE>
__global__ __launch_bounds__(kThreads) void join_kernel(Args a) {
  constexpr int kEach = D <= kWave ? 1 : D <= 2 * kWave ? 2 : 4;    // dims of a lane, kEach in a row (the last lanes may have none)
  static_assert(D % kEach == 0 && D / kEach <= kWave, "a lane's dims lie in its head, all of them or none");   // (three would not: 160, 176)
  constexpr int kStride = SHARE ? kWaves : 1;
  constexpr float kLittle = 0x1p-126f;      // (a segment that is worth less is taken as that: its sum may be infinite, and 0 times it a NaN)
  __shared__ float shares[SHARE ? kWaves : 1][kEach * kWave];
  const int token = blockIdx.x, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int q_head = SHARE ? blockIdx.y : blockIdx.y * kWaves + wave;
  if (q_head >= a.q_heads) return;
  const int group = static_cast<int>(a.group.by), head = a.group.quotient(q_head);
  const int segments = a.prefix_segments + a.own_segments;
  const size_t row = static_cast<size_t>(token) * group + (q_head - head * group);
  const float2* stats = reinterpret_cast<const float2*>(a.stats) + (static_cast<size_t>(head) * a.rows + row) * segments;
  const bool here = kEach * lane < D;
  const float* sums = a.sums + (static_cast<size_t>(head) * segments * a.rows + row) * D + (here ? kEach * lane : 0);
  constexpr int kAhead = SHARE ? 8 : 4;                         // segments whose values are on their way together
  float fetched[kAhead][kEach];
  auto fetch = [&](int from, int end) {                         // (behind the last one, it again)
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const float* at = sums + static_cast<size_t>(min(from + u * kStride, end - 1)) * a.rows * D;
#pragma unroll
      for (int e = 0; e < kEach; ++e) fetched[u][e] = at[e];
    }
  };
  // A row that has a result has all of the prompt's segments and one of its own: they are asked for before it is known whose the row is,
  // into values that are not looked at unless it has.
  const int sure = min(a.prefix_segments + 1, kAhead * kStride), share = SHARE ? wave : 0;
  float2 one = lane < segments ? stats[lane] : float2{-INFINITY, 0.f};
  fetch(share, sure);
  __builtin_amdgcn_sched_barrier(0);
  int before = 0;                                               // requests whose first row is this token's or lies before it
  for (int i0 = 0; i0 < a.requests; i0 += kWave)
    before += __popcll(__ballot(i0 + lane < a.requests && a.q_start[min(i0 + lane, a.requests - 1)] <= token));
  if (before == 0 || token >= a.q_start[a.requests]) return;    // rows behind the last request's are left as they are
  const int request = before - 1;                               // (the last of those: the ones that bring nothing come before it)
  const int begin = a.q_start[request], count = a.q_start[request + 1] - begin, length = a.seq_lens[request];
  const int seen = length - count + token - begin + 1;          // keys of the token
  T* out = static_cast<T*>(a.out) + (static_cast<size_t>(token) * a.q_heads + q_head) * D + kEach * lane;
  float sum[kEach], total = 0.f;
#pragma unroll
  for (int e = 0; e < kEach; ++e) sum[e] = 0.f;
  if (!within_bounds(a, begin, count, length) || token - begin >= count || table_of(a, request) == nullptr ||
      (a.shared > 0 && a.prefix_pages == nullptr && table_of(a, 0) == nullptr)) {
    total = NAN;
  } else {
    const int used = a.prefix_segments + (seen - a.shared + a.own_keys - 1) / a.own_keys;
    float top = -INFINITY;
    for (int i0 = 0; i0 < used; i0 += kWave) {
      if (i0 != 0) one = stats[min(i0 + lane, used - 1)];
      if (i0 + lane >= used) one = float2{-INFINITY, 0.f};
      const float m = fmaxf(top, wave_max(one.x)), reference = m == -INFINITY ? 0.f : m;
      if (i0 != 0) {                                            // (more segments than lanes: what is there already goes along)
        const float by = fmaxf(__builtin_amdgcn_exp2f(top - reference), kLittle);
        total *= by;
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] *= by;
      }
      top = m;
      const float weight = __builtin_amdgcn_exp2f(one.x - reference), worth = fmaxf(weight, kLittle);
      total += wave_sum(weight * one.y);
      const int end = min(i0 + kWave, used);
      auto add = [&](int from, int end) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const float by = __shfl(worth, min(from + u * kStride, end - 1) - i0, kWave);
          if (from + u * kStride < end) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) sum[e] = fmaf(by, fetched[u][e], sum[e]);
          }
        }
      };
      if (i0 == 0) add(share, sure);
      for (int i = share + (i0 == 0 ? sure : i0); i < end; i += kAhead * kStride) {
        fetch(i, end);
        add(i, end);
      }
    }
  }
  if constexpr (SHARE) {
    if (wave != 0) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) shares[wave][e * kWave + lane] = sum[e];
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
#pragma unroll
      for (int e = 0; e < kEach; ++e) sum[e] += shares[w][e * kWave + lane];
  }
  if (here) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) out[e] = from_float<T>(sum[e] / total);
  }
}

template <typename K> int room_for(K kernel, size_t lds) {
  static_assert(kWideLds <= 160 * 1024 && kWideNarrowLds <= 160 * 1024 && 2 * narrow_lds<float>(kWaves / 2) <= 160 * 1024, "LDS of a compute unit");
  if (lds <= 64 * 1024) return 0;
  return static_cast<int>(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds)));
}

// `wide`: the prefix goes to `wide_prefix_kernel`, and the requests' own keys alone to the other one, which holds twice as many blocks a
// unit.
template <typename T> int run(const Args& all, bool wide, hipStream_t stream) {
  Args a = all;
  const size_t lds = a.own_tiles > 1 ? 2 * narrow_lds<T>(kWaves / 2) : narrow_lds<T>(kWaves);       // (the former is the larger)
  int status = 0;
  if constexpr (kWideFits && sizeof(T) == 2)
    if (wide && a.prefix_blocks > 0) {
      constexpr size_t wide_lds = kWideLds > kWideNarrowLds ? kWideLds : kWideNarrowLds;
      if (a.prefix_blocks > 0x7fffffffL) return -2;
      if ((status = room_for(wide_prefix_kernel, wide_lds)) != 0) return status;
      Args of_prompt = a;
      if (a.prefix_pages != nullptr) {      // (a table whose only row they are)
        of_prompt.block_table = a.prefix_pages;
        of_prompt.table_rows = nullptr;
        of_prompt.table_count = 1;
      }
      wide_prefix_kernel<<<static_cast<unsigned>(a.prefix_blocks), kWideWaves * kWave, wide_lds, stream>>>(of_prompt);
      if ((status = AKV_LAUNCH_STATUS()) != 0) return status;
      a.prefix_blocks = 0;
    }
  const long blocks = a.prefix_blocks + static_cast<long>(a.requests) * a.kv_heads * ((a.own_tiles + 1) / 2) * a.own_segments;
  if (blocks > 0x7fffffffL || a.q_heads > 65535) return -2;
  const auto kernel = a.prefix_pages != nullptr && a.prefix_blocks > 0 ? shared_prefix_kernel<T, true> : shared_prefix_kernel<T, false>;
  if ((status = room_for(kernel, lds)) != 0) return status;
  kernel<<<static_cast<unsigned>(blocks), kThreads, lds, stream>>>(a);
  if ((status = AKV_LAUNCH_STATUS()) != 0) return status;
  // (a wave a row where they are 2,048 and more, eight of a unit's thirty-two)
  if (a.tokens * a.q_heads >= 8L * device_facts().compute_units)
    join_kernel<T, false><<<dim3(static_cast<unsigned>(a.tokens), (a.q_heads + kWaves - 1) / kWaves), kThreads, 0, stream>>>(a);
  else
    join_kernel<T, true><<<dim3(static_cast<unsigned>(a.tokens), a.q_heads), kThreads, 0, stream>>>(a);
  return AKV_LAUNCH_STATUS();
}

}  // namespace

#define AKV_NAME_(dim) akv_attention_shared_prefix_d##dim
#define AKV_NAME(dim) AKV_NAME_(dim)

// `sums` and `stats` hold kv_heads * (prefix_segments + own_segments) * tokens * (q_heads / kv_heads) rows of head size and of two
// floats; segments: prefix_segments of prefix_keys (multiples of 32) cover `shared`, own_segments of own_keys `max_own` keys of a
// request behind it, at most 512 together.  `wide`: the prompt's columns go in tiles of 256 (`walk_wide`).  Operands lie on 16-byte boundaries.
extern "C" int AKV_NAME(AKV_HEAD_DIM)(const void* q, const void* k_pages, const void* v_pages, void* out, int dtype, float* sums, float* stats,
                                      const int* q_start, const int* seq_lens, const int* block_table, const int* table_rows, const int* prefix_pages, int table_width,
                                      int table_count, int requests, long tokens, int q_heads, int kv_heads, int page_size, long num_pages, float scale,
                                      int shared, int max_own, int max_new, int prefix_segments, int prefix_keys, int own_segments,
                                      int own_keys, int wide, hipStream_t stream) {
  if (requests <= 0 || tokens <= 0) return 0;
  if (kv_heads <= 0 || q_heads % kv_heads != 0 || page_size < 8 || (page_size & (page_size - 1)) != 0 || shared % page_size != 0 ||
      max_own <= 0 || max_new <= 0 || own_segments < 1 || prefix_segments + own_segments > 512 || prefix_keys % 32 != 0 || own_keys % 32 != 0 ||
      static_cast<long>(prefix_segments) * prefix_keys < shared || static_cast<long>(own_segments) * own_keys < max_own ||
      (static_cast<long>(shared) + max_own + page_size - 1) / page_size > table_width)
    return -2;
  const long size = dtype == kF32 ? 4 : 2, of_q = tokens * q_heads * D * size, of_pages = num_pages * kv_heads * page_size * D * size;
  const Span spans[] = {{out, of_q}, {q, of_q}, {k_pages, of_pages}, {v_pages, of_pages}, {block_table, 4L * table_width * table_count},
                        {q_start, 4L * requests + 4}, {seq_lens, 4L * requests}, {table_rows, 4L * requests}, {prefix_pages, 4L * (shared / page_size)}};
  const int overlap = shared_spans(spans, 1, 9);
  if (overlap != 0) return overlap;
  Args a{};
  const int group = q_heads / kv_heads;
  a.q = q; a.k_pages = k_pages; a.v_pages = v_pages; a.out = out; a.sums = sums; a.stats = stats;
  a.q_start = q_start; a.seq_lens = seq_lens; a.block_table = block_table; a.table_rows = table_rows; a.prefix_pages = prefix_pages;
  a.table_width = table_width; a.table_count = table_count; a.requests = requests; a.tokens = tokens; a.rows = tokens * group;
  a.q_heads = q_heads; a.kv_heads = kv_heads; a.shared = shared; a.max_own = max_own; a.max_new = max_new;
  a.num_pages = num_pages; a.scale_log2 = scale * kLog2e; a.group = Divider::of(group);
  while ((1 << a.page_shift) < page_size) ++a.page_shift;
  a.prefix_segments = prefix_segments; a.prefix_keys = prefix_keys; a.own_segments = own_segments; a.own_keys = own_keys;
  if (wide != 0 && (!kWideFits || dtype != kBF16 || page_size < 16)) return -2;
  a.prefix_tiles = static_cast<int>(wide != 0 ? (a.rows + kWideColumns - 1) / kWideColumns : (a.rows + 31) / 32);
  a.own_tiles = static_cast<int>((static_cast<long>(max_new) * group + 31) / 32);
  a.prefix_blocks = static_cast<long>(prefix_segments) * kv_heads * a.prefix_tiles;
  if (dtype == kF32) return run<float>(a, false, stream);
  if (dtype == kBF16) return run<bf16_t>(a, wide != 0, stream);
  return -1;
}
