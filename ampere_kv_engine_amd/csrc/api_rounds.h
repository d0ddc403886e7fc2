// C entry points of the library for rounds of drafted tokens: a step's tables and maps from lengths that lie on the device, and the
// drafted tokens held against the target's probabilities.  As in api.h every function enqueues on `stream` and returns 0, a
// hipError_t of the launch, or -2 for sizes the kernel does not take; pointers are device pointers, shapes are checked by the
// caller.
#pragma once

#include <hip/hip_runtime.h>

extern "C" {

// -(1000 + 64 i + j): spans i and j overlap, of which i is written (see `shared_spans` in common.h); the spans' order stands at each entry.
// (For checks: the same for any spans.)
int akv_shared_spans(const void* const* begins, const long* bytes, int written, int count);

// The most requests `akv_place_tokens` takes.
int akv_place_most_requests();
int akv_place_tokens(const int* lengths, const int* counts, const int* held, const int* free_pages, long free_count,
                     const int* cursor, int* table, const int* rows, int table_rows, int table_width, int page_size,
                     const int* prefix_pages, int prefix_count, int requests, int tokens, int* q_start, int* seq_lens,
                     int* held_after, int* cursor_after, int* positions, int* seq_of_token, int* slot_map, int* status,
                     int clear_rest, hipStream_t stream);

// Bytes of `workspace` (on a 16-byte boundary) for `requests` requests of up to `places` rows; -1 for sizes not taken.
long akv_verify_workspace(int requests, int places, int vocab);
int akv_verify_drafts(const float* logits, int rows, int vocab, const int* tokens, const int* q_start, const float* temperature,
                      const float* uniforms, int requests, int places, const float* draft_logits, long draft_request_stride,
                      long draft_place_stride, int* kept, int* chosen, void* workspace, hipStream_t stream);
}
