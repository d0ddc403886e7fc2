// A step's layout from the requests' lengths, all of it on the device: how many pages each request takes from the pool, its
// block-table entries, and the position, request and cache slot of every token it brings.
//
//   after_r = length_r + count_r                    had_r = held_r, or the prompt's pages for a request that holds none yet
//   has_r   = max(had_r, ceil(after_r / page))      its new pages: free[cursor + (new pages of requests before r) + 0, 1, ...]
//   token j of request r: position length_r + j, slot = page of that position * page size + position within the page
//
// One launch.  Every block runs the prefix sums over the requests for itself, in LDS (a few hundred requests: cheaper than a
// launch of its own or a wait between blocks), and then takes its share of the tokens and of the table's entries.  A token's page
// is computed, not read back from the table entries that another block may be writing: an entry below `had` was there
// before the call (or is the prompt's), one from `had` on follows from the free list.  So no block reads what another writes.
// Nothing but `status` is written where the step cannot be laid out: every block finds that out before it writes.
// What bounds it is latency: a launch, the lengths' reads, the scan's barriers, one dependent read (free list or table) a token.

#include "common.h"
#include "api_rounds.h"

using namespace akv;

namespace {

constexpr int kMost = 4096;       // requests: three ints each in LDS
constexpr int kThreads = 256;

struct Place {
  const int *lengths, *counts, *held, *free_pages, *cursor, *rows, *prefix_pages;
  int *table, *q_start, *seq_lens, *held_after, *cursor_after, *positions, *seq_of_token, *slot_map, *status;
  long free_count;
  int table_rows, table_width, page_size, prefix_count, requests, tokens;
  Divider page;
};

// Inclusive sums over the block's threads of two counts at once (64 bits hold any sum of a request's 31-bit counts).
__device__ __forceinline__ void scan_pair(long& a, long& b, long (*scratch)[2]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int offset = 1; offset < kWave; offset <<= 1) {
    const long x = __shfl_up(a, offset, kWave), y = __shfl_up(b, offset, kWave);
    if (lane >= offset) { a += x; b += y; }
  }
  __syncthreads();
  if (lane == kWave - 1) { scratch[wave][0] = a; scratch[wave][1] = b; }
  __syncthreads();
  for (int w = 0; w < wave; ++w) { a += scratch[w][0]; b += scratch[w][1]; }
}

__global__ __launch_bounds__(kThreads) void place_kernel(Place p) {
  __shared__ int first_token[kMost + 1];     // tokens before a request's
  __shared__ int first_page[kMost + 1];      // pages taken before a request's
  __shared__ int had_of[kMost];
  __shared__ long scratch[kThreads / kWave][2];
  __shared__ int rows_seen[2 * kMost];       // a hash of the table's rows that requests name, by open addressing
  const int tid = threadIdx.x;
  long tokens_before = 0, pages_before = 0;
  int wrong = 0;           // 1 a length or count that cannot be, 2 a table row that is too narrow, not there or named twice
  int places = kThreads;   // of the hash: a power of two, at least twice the requests
  while (places < 2 * p.requests) places *= 2;
  if (p.rows != nullptr) {
    for (int i = tid; i < places; i += kThreads) rows_seen[i] = -1;
    __syncthreads();
  }
  for (int r0 = 0; r0 < p.requests; r0 += kThreads) {
    const int r = r0 + tid;
    long count = 0, taken = 0;
    if (r < p.requests) {
      const int length = p.lengths[r], held = p.held[r], brings = p.counts[r];
      const int row = p.rows != nullptr ? p.rows[r] : r;
      const long after = static_cast<long>(length) + brings;
      int had = held;
      if (length < 0 || brings < 0 || held < 0 || after > 0x7fffffffL) {
        wrong |= 1;
      } else {
        if (held == 0) had = p.prefix_count;
        const int quotient = p.page.quotient(static_cast<int>(after));
        const int need = quotient + (p.page.rest(static_cast<int>(after), quotient) != 0 ? 1 : 0);
        // (what a request held before has to lie on pages that it has: the entries of those are read)
        const int old = p.page.quotient(length) + (p.page.rest(length, p.page.quotient(length)) != 0 ? 1 : 0);
        if (had < old) wrong |= 1;
        count = brings;
        taken = max(0, need - had);
        if (row < 0 || row >= p.table_rows || had + taken > p.table_width) {
          wrong |= 2;
        } else if (p.rows != nullptr) {
          // (as many rows as requests at most in twice as many places: the walk ends at a free place or at the row's own)
          for (int at = (row * 0x9E3779B1u >> 8) & (places - 1);; at = (at + 1) & (places - 1)) {
            const int there = atomicCAS(&rows_seen[at], -1, row);
            if (there == row) wrong |= 2;
            if (there == row || there == -1) break;
          }
        }
      }
      had_of[r] = had;
    }
    long token_end = count, page_end = taken;
    scan_pair(token_end, page_end, scratch);
    if (r < p.requests) {
      // (sums beyond 31 bits are refused below, by their totals)
      first_token[r] = static_cast<int>(tokens_before + token_end - count);
      first_page[r] = static_cast<int>(pages_before + page_end - taken);
    }
    __syncthreads();
    if (tid == kThreads - 1) { scratch[0][0] = token_end; scratch[0][1] = page_end; }    // the last thread's sums are the totals
    __syncthreads();
    tokens_before += scratch[0][0];
    pages_before += scratch[0][1];
    __syncthreads();
  }
  const bool bad_numbers = __syncthreads_or(wrong & 1), bad_rows = __syncthreads_or(wrong & 2);
  const int cursor = p.cursor[0];
  int verdict = pages_before > 0x7fffffffL ? -1 : static_cast<int>(pages_before);
  if (bad_numbers) verdict = -4;
  else if (tokens_before > p.tokens) verdict = -3;
  else if (bad_rows) verdict = -2;
  else if (cursor < 0 || cursor + pages_before > p.free_count) verdict = -1;
  if (blockIdx.x == 0 && tid == 0) {
    p.status[0] = verdict;
    if (verdict >= 0) p.cursor_after[0] = cursor + verdict;
  }
  if (verdict < 0) return;
  const int tokens = static_cast<int>(tokens_before), pages = static_cast<int>(pages_before);
  if (tid == 0) { first_token[p.requests] = tokens; first_page[p.requests] = pages; }
  __syncthreads();
  const int begin = blockIdx.x * kThreads + tid, stride = gridDim.x * kThreads;
  for (int r = begin; r < p.requests; r += stride) {
    p.q_start[r] = first_token[r];
    p.seq_lens[r] = p.lengths[r] + first_token[r + 1] - first_token[r];
    p.held_after[r] = had_of[r] + first_page[r + 1] - first_page[r];
  }
  if (begin == 0) p.q_start[p.requests] = tokens;
  // the last request whose first number is <= n (requests that bring nothing are stepped over)
  auto owner = [&](const int* first, int n) {
    int low = 0, high = p.requests;       // first[low] <= n < first[high]
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (first[middle] <= n) low = middle; else high = middle;
    }
    return low;
  };
  for (int n = begin; n < pages; n += stride) {
    const int r = owner(first_page, n);
    const int row = p.rows != nullptr ? p.rows[r] : r;
    p.table[static_cast<size_t>(row) * p.table_width + had_of[r] + n - first_page[r]] = p.free_pages[cursor + n];
  }
  if (p.prefix_count > 0) {               // requests that hold nothing yet start on the prompt's pages: a wave each
    const int lane = tid & (kWave - 1), wave = begin / kWave, waves = stride / kWave;
    for (int r = wave; r < p.requests; r += waves) {
      if (p.held[r] != 0) continue;
      const int row = p.rows != nullptr ? p.rows[r] : r;
      for (int i = lane; i < p.prefix_count; i += kWave) p.table[static_cast<size_t>(row) * p.table_width + i] = p.prefix_pages[i];
    }
  }
  for (int n = begin; n < tokens; n += stride) {
    const int r = owner(first_token, n);
    const int position = p.lengths[r] + n - first_token[r];
    const int at = p.page.quotient(position), inside = p.page.rest(position, at);
    int id;
    if (at >= had_of[r]) {
      id = p.free_pages[cursor + first_page[r] + at - had_of[r]];
    } else if (p.held[r] == 0) {
      id = p.prefix_pages[at];
    } else {
      const int row = p.rows != nullptr ? p.rows[r] : r;
      id = p.table[static_cast<size_t>(row) * p.table_width + at];
    }
    p.positions[n] = position;
    p.seq_of_token[n] = r;
    p.slot_map[n] = id < 0 ? -1 : id * p.page_size + inside;
  }
}

}  // namespace

extern "C" int akv_place_most_requests() { return kMost; }

// `status` [1]: the pages taken, or why nothing but `status` was written: -1 too few free pages, -2 a request's row is not in the
// table, too narrow for its pages or another request's too, -3 more tokens than the maps have room for, -4 a negative length, count or number of pages, or a
// request that holds fewer pages than its length fills.  No output may lie in an input but `table`, whose entries below a request's
// pages are read and never written.
extern "C" int akv_place_tokens(const int* lengths, const int* counts, const int* held, const int* free_pages, long free_count,
                                const int* cursor, int* table, const int* rows, int table_rows, int table_width, int page_size,
                                const int* prefix_pages, int prefix_count, int requests, int tokens, int* q_start, int* seq_lens,
                                int* held_after, int* cursor_after, int* positions, int* seq_of_token, int* slot_map, int* status,
                                hipStream_t stream) {
  if (requests < 0 || requests > kMost || tokens < 0 || page_size <= 0 || table_width < 0 || table_rows < 0 || prefix_count < 0) return -2;
  const Place p{lengths, counts, held, free_pages, cursor, rows, prefix_pages, table, q_start, seq_lens, held_after, cursor_after,
                positions, seq_of_token, slot_map, status, free_count, table_rows, table_width, page_size, prefix_count, requests,
                tokens, Divider::of(page_size)};
  const int blocks = max(1, min(256, (max(tokens, requests) + kThreads - 1) / kThreads));
  place_kernel<<<blocks, kThreads, 0, stream>>>(p);
  return AKV_LAUNCH_STATUS();
}
