// Argument blocks and launchers of the paged cache's tables on the GPU (paged_plan.cu).
#pragma once

#include <stdint.h>

#include <cuda_runtime.h>

namespace omni {

constexpr int kPlanMaxRequests = 8192;

// What the sequences hold: length [seqs], the page numbers of a sequence's positions in a row of table, and a stack of
// free pages (the first *count of free [pages]).
struct PageState {
  int64_t* length;
  int64_t seqs;
  int32_t* table;
  int64_t table_stride;
  int table_width;
  int32_t* free;
  int64_t* count;
  int64_t pages;
  int page;
};

struct PlanArgs {
  PageState s;
  const int64_t* rows;  // [requests] sequence of each request
  const int64_t* want;  // [requests] new tokens (plan), positions kept (trim)
  int requests;
  int tokens;             // entries of pos and slots
  int last;               // refused requests' tokens get positions up to this
  int64_t* pos;           // [tokens]
  int64_t* slots;         // [tokens]
  int32_t* batch_table;   // [requests, batch_width]
  int batch_width;
  int64_t* lengths;    // [requests]
  int64_t* q_offsets;  // [requests + 1]
  int64_t* k_offsets;  // [requests + 1]
  uint8_t* taken;      // [requests]
  unsigned* arrivals;  // zero on entry, left zero
  int* status;
};
cudaError_t launch_paged_plan(const PlanArgs& a, cudaStream_t stream);
cudaError_t launch_paged_trim(const PlanArgs& a, cudaStream_t stream);

}  // namespace omni
