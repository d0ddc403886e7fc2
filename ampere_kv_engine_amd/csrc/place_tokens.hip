// A step's layout from the requests' lengths, all of it on the device: how many pages each request takes from the pool, its
// block-table entries, and the position, request and cache slot of every token it brings.
//
//   after_r = length_r + count_r                    had_r = held_r, or the prompt's pages for a request that holds none yet
//   has_r   = max(had_r, ceil(after_r / page))      its new pages: free[cursor + (new pages of requests before r) + 0, 1, ...]
//   token j of request r: position length_r + j, slot = page of that position * page size + position within the page
//
// One launch.  Every block runs the prefix sums over the requests for itself (a few hundred requests: cheaper than a launch of its
// own or a wait between blocks), keeps what it has read of them in LDS, and then takes its share of the tokens and of the table's
// entries.  A token's page is computed, not read back from the table entries that another block may be writing: an entry below `had` was
// there before the call (or is the prompt's), one from `had` on follows from the free list.  So no block reads what another writes.
// Nothing but `status` is written where the step cannot be laid out - or, `clear_rest`, a layout in which nobody brings anything: every
// block finds that out before it writes.
// What bounds it is latency: a launch (2.8 us), the lengths' reads, the scan's barriers, one dependent read (free list or table) a token:
// 8 requests 4.7 us, 500 of up to 5 tokens 6.6, 64 prompts of 115,000 tokens together 6.4; a call takes the host 9.

#include "common.h"
#include "api_rounds.h"

using namespace akv;

namespace {

constexpr int kMost = 4096;       // requests: five ints each in LDS, and two of the hash
constexpr int kThreads = 1024;

struct Place {
  const int *lengths, *counts, *held, *free_pages, *cursor, *rows, *prefix_pages;
  int *table, *q_start, *seq_lens, *held_after, *cursor_after, *positions, *seq_of_token, *slot_map, *status;
  long free_count;
  int table_rows, table_width, page_size, prefix_count, requests, tokens;
  int clear_rest;                 // whether slots behind the last token, and what a step that cannot be laid out leaves, are written too
  int hash_places;                // a power of two, at least twice the requests
  Divider page;
};

// Sums over the lanes up to each, inside the vector unit: four shifts within rows of 16 lanes, two broadcasts of a row's last lane.
template <int CTRL, int ROWS> __device__ __forceinline__ long moved(long v) {
  const int low = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
  const int high = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
  return (static_cast<long>(high) << 32) | static_cast<uint32_t>(low);
}
__device__ __forceinline__ long sums_up_to(long v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}

__global__ __launch_bounds__(kThreads) void place_kernel(Place p) {
  constexpr int kWaves = kThreads / kWave;
  extern __shared__ int lds[];
  __shared__ long of_waves[2][kWaves];
  __shared__ int wrong;
  const int n = p.requests;
  int* first_token = lds;               // [n + 1] tokens before a request's
  int* first_page = first_token + n + 1;    // [n + 1] pages taken before a request's
  int* had_of = first_page + n + 1;     // [n] pages before the call; of a request that starts on the prompt's, -1 - their number
  int* length_of = had_of + n;          // [n]
  int* row_of = length_of + n;          // [n]
  int* rows_seen = row_of + n;          // a hash of the table's rows that requests name, by open addressing
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int cursor = p.cursor[0];
  if (tid == 0) wrong = 0;
  if (p.rows != nullptr)
    for (int i = tid; i < p.hash_places; i += kThreads) rows_seen[i] = -1;
  __syncthreads();
  // Whether a request brings places of the prompt's own pages.  That is how a prompt is written - by requests of a batch none of which
  // has it yet, a place by one of them at most; beside a request that has pages or starts behind the prompt (8) it would be written over.
  const long prompt_end = static_cast<long>(p.prefix_count) * p.page_size;
  auto writes_prompt = [&](bool fresh, int length, int brings) { return fresh && brings > 0 && length < prompt_end; };
  long tokens_before = 0, pages_before = 0;
  for (int r0 = 0; r0 < n; r0 += kThreads) {
    const int r = r0 + tid;
    long count = 0, taken = 0;
    // 1 a length or count that cannot be, 2 a table row that is too narrow, not there or named twice; 4 and 8: see `writes_prompt`
    int fault = 0;
    if (r < n) {
      const int length = p.lengths[r], held = p.held[r], brings = p.counts[r];
      const int row = p.rows != nullptr ? p.rows[r] : r;
      const long after = static_cast<long>(length) + brings;
      const int had = held == 0 ? p.prefix_count : held;
      if (length < 0 || brings < 0 || held < 0 || after > 0x7fffffffL) {
        fault = 1;
      } else {
        const int whole = p.page.quotient(static_cast<int>(after)), old = p.page.quotient(length);
        const int need = whole + (p.page.rest(static_cast<int>(after), whole) != 0 ? 1 : 0);
        // (what a request held before has to lie on pages that it has: the entries of those are read)
        if (had < old + (p.page.rest(length, old) != 0 ? 1 : 0)) fault = 1;
        count = brings;
        taken = max(0, need - had);
        if (writes_prompt(held == 0, length, brings)) fault |= 4;
        else if (prompt_end > 0 && (held != 0 || brings != 0)) fault |= 8;
        if (row < 0 || row >= p.table_rows || had + taken > p.table_width) {
          fault |= 2;
        } else if (p.rows != nullptr) {
          // (as many rows as requests at most in twice as many places: the walk ends at a free place or at the row's own)
          for (int at = (row * 0x9E3779B1u >> 8) & (p.hash_places - 1);; at = (at + 1) & (p.hash_places - 1)) {
            const int there = atomicCAS(&rows_seen[at], -1, row);
            if (there == row) fault |= 2;
            if (there == row || there == -1) break;
          }
        }
      }
      had_of[r] = held == 0 && p.prefix_count > 0 ? -1 - had : had;
      length_of[r] = length;
      row_of[r] = row;
    }
    // (one of a wave says so for all: every request of a batch with a prompt has one, and a thousand of them on one word take 2 us)
    int faults = 0;
#pragma unroll
    for (int bit = 1; bit <= 8; bit *= 2)
      if (__any((fault & bit) != 0)) faults |= bit;
    if (lane == 0 && faults != 0) atomicOr(&wrong, faults);
    const long token_end = sums_up_to(count), page_end = sums_up_to(taken);      // (64 bits hold any sum of 4,096 requests')
    if (lane == kWave - 1) { of_waves[0][wave] = token_end; of_waves[1][wave] = page_end; }
    __syncthreads();
    long tokens_here = tokens_before + token_end - count, pages_here = pages_before + page_end - taken;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const long a = of_waves[0][w], b = of_waves[1][w];
      if (w < wave) { tokens_here += a; pages_here += b; }
      tokens_before += a;
      pages_before += b;
    }
    // (sums beyond 31 bits are refused below, by their totals)
    if (r < n) { first_token[r] = static_cast<int>(tokens_here); first_page[r] = static_cast<int>(pages_here); }
    __syncthreads();
  }
  int verdict = pages_before > 0x7fffffffL ? -1 : static_cast<int>(pages_before);
  const int faults = wrong;
  bool meet = (faults & 12) == 12;
  if ((faults & 13) == 4 && tokens_before <= p.tokens) {     // (a request's tokens lie in LDS as a difference)
    if (tid == 0) first_token[n] = static_cast<int>(tokens_before);
    __syncthreads();
    for (int r = tid; r < n && !meet; r += kThreads) {
      const int brings = first_token[r + 1] - first_token[r], from = length_of[r];
      if (!writes_prompt(had_of[r] < 0, from, brings)) continue;
      for (int other = 0; other < r && !meet; ++other) {
        const int its = first_token[other + 1] - first_token[other], at = length_of[other];
        meet = writes_prompt(had_of[other] < 0, at, its) && max(from, at) < min(prompt_end, min(from + static_cast<long>(brings), at + static_cast<long>(its)));
      }
    }
    meet = __syncthreads_or(meet);
  }
  if ((faults & 1) != 0 || meet) verdict = -4;
  else if (tokens_before > p.tokens) verdict = -3;
  else if ((faults & 2) != 0) verdict = -2;
  else if (cursor < 0 || cursor + pages_before > p.free_count) verdict = -1;
  if (blockIdx.x == 0 && tid == 0) {
    p.status[0] = verdict;
    if (verdict >= 0) p.cursor_after[0] = cursor + verdict;
  }
  const int begin = blockIdx.x * kThreads + tid, stride = gridDim.x * kThreads;
  if (verdict < 0) {
    if (p.clear_rest == 0) return;
    for (int i = begin; i < p.tokens; i += stride) p.slot_map[i] = -1;
    for (int r = begin; r < n; r += stride) {
      p.q_start[r] = 0;
      p.seq_lens[r] = p.lengths[r];
      p.held_after[r] = p.held[r];
    }
    if (begin == 0) {
      p.q_start[n] = 0;
      p.cursor_after[0] = cursor;
    }
    return;
  }
  const int tokens = static_cast<int>(tokens_before), pages = static_cast<int>(pages_before);
  if (tid == 0) { first_token[n] = tokens; first_page[n] = pages; }
  __syncthreads();
  auto pages_had = [&](int r) { return had_of[r] < 0 ? -1 - had_of[r] : had_of[r]; };
  // the last request whose first number is <= i (requests that bring nothing are stepped over)
  auto owner = [&](const int* first, int i) {
    int low = 0, high = n;       // first[low] <= i < first[high]
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (first[middle] <= i) low = middle; else high = middle;
    }
    return low;
  };
  for (int i = begin; i < tokens; i += stride) {
    const int r = owner(first_token, i);
    const int position = length_of[r] + i - first_token[r], had = pages_had(r);
    const int at = p.page.quotient(position), inside = p.page.rest(position, at);
    const int id = at >= had ? p.free_pages[cursor + first_page[r] + at - had]
                   : had_of[r] < 0 ? p.prefix_pages[at] : p.table[static_cast<size_t>(row_of[r]) * p.table_width + at];
    p.positions[i] = position;
    p.seq_of_token[i] = r;
    const long slot = static_cast<long>(id) * p.page_size + inside;      // (beyond 31 bits it would be another page's)
    p.slot_map[i] = id < 0 || slot > 0x7fffffffL ? -1 : static_cast<int>(slot);
  }
  if (p.clear_rest != 0)
    for (int i = tokens + begin; i < p.tokens; i += stride) p.slot_map[i] = -1;
  for (int i = begin; i < pages; i += stride) {
    const int r = owner(first_page, i);
    p.table[static_cast<size_t>(row_of[r]) * p.table_width + pages_had(r) + i - first_page[r]] = p.free_pages[cursor + i];
  }
  for (int r = begin; r < n; r += stride) {
    p.q_start[r] = first_token[r];
    p.seq_lens[r] = length_of[r] + first_token[r + 1] - first_token[r];
    p.held_after[r] = pages_had(r) + first_page[r + 1] - first_page[r];
  }
  if (begin == 0) p.q_start[n] = tokens;
  if (p.prefix_count > 0)                 // requests that hold nothing yet start on the prompt's pages: a wave each
    for (int r = begin / kWave; r < n; r += stride / kWave)
      if (had_of[r] < 0)
        for (int i = lane; i < p.prefix_count; i += kWave) p.table[static_cast<size_t>(row_of[r]) * p.table_width + i] = p.prefix_pages[i];
}

}  // namespace

extern "C" int akv_shared_spans(const void* const* begins, const long* bytes, int written, int count) {
  Span spans[64];
  if (count < 0 || count > 64) return -2;
  for (int i = 0; i < count; ++i) spans[i] = Span{begins[i], bytes[i]};
  return shared_spans(spans, written, count);
}

extern "C" int akv_place_most_requests() { return kMost; }

// `status` [1]: the pages taken, or why nothing but `status` was written: -1 too few free pages, -2 a request's row is not in the
// table, too narrow for its pages or another request's too, -3 more tokens than the maps have room for, -4 a negative length, count or
// number of pages, a request that holds fewer pages than its length fills, or one that would write into a prompt that another one of the batch has
// or writes as well.  `clear_rest` not 0: slot_map is -1 behind the last token, and where the step cannot be laid out everywhere, with q_start
// all 0 and the lengths, pages and cursor as before.  No output may lie in an input but `table`, whose entries below a request's
// pages are read and never written.
extern "C" int akv_place_tokens(const int* lengths, const int* counts, const int* held, const int* free_pages, long free_count,
                                const int* cursor, int* table, const int* rows, int table_rows, int table_width, int page_size,
                                const int* prefix_pages, int prefix_count, int requests, int tokens, int* q_start, int* seq_lens,
                                int* held_after, int* cursor_after, int* positions, int* seq_of_token, int* slot_map, int* status,
                                int clear_rest, hipStream_t stream) {
  if (requests < 0 || requests > kMost || tokens < 0 || page_size <= 0 || table_width < 0 || table_rows < 0 || prefix_count < 0) return -2;
  const long of_requests = 4L * requests, of_tokens = 4L * tokens;
  const Span spans[] = {{q_start, of_requests + 4}, {seq_lens, of_requests}, {held_after, of_requests}, {cursor_after, 4}, {positions, of_tokens},
                        {seq_of_token, of_tokens}, {slot_map, of_tokens}, {status, 4}, {table, 4L * table_rows * table_width},
                        {lengths, of_requests}, {counts, of_requests}, {held, of_requests}, {cursor, 4}, {free_pages, 4 * free_count},
                        {rows, of_requests}, {prefix_pages, 4L * prefix_count}};
  const int shared = shared_spans(spans, 9, 16);
  if (shared != 0) return shared;
  int places = kWave;
  while (places < 2 * requests) places *= 2;
  const Place p{lengths, counts, held, free_pages, cursor, rows, prefix_pages, table, q_start, seq_lens, held_after, cursor_after,
                positions, seq_of_token, slot_map, status, free_count, table_rows, table_width, page_size, prefix_count, requests,
                tokens, clear_rest, places, Divider::of(page_size)};
  // (a wave takes a forked request's entries, some hundred reads and writes of the prompt's pages: with blocks enough for all of them)
  const long entries = max(static_cast<long>(max(tokens, requests)), static_cast<long>(requests) * min(prefix_count, kWave));
  const int blocks = static_cast<int>(max(1L, min(256L, (entries + kThreads - 1) / kThreads)));
  const size_t lds = (5 * static_cast<size_t>(requests) + 2 + (rows != nullptr ? places : 0)) * sizeof(int);
  if (lds > 60 * 1024) {
    const hipError_t status = hipFuncSetAttribute(reinterpret_cast<const void*>(place_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                  static_cast<int>(lds));
    if (status != hipSuccess) return static_cast<int>(status);
  }
  place_kernel<<<blocks, kThreads, lds, stream>>>(p);
  return AKV_LAUNCH_STATUS();
}
