// extern "C" entry points of the gradients' norm (cascmm_gradients_kernel.h): argument checks, chunks and launches.
#include "cascmm_gradients_kernel.h"

#include <cmath>
#include <cstring>

#include <algorithm>
#include <new>
#include <vector>

namespace cascmm {

static int64_t grad_size(int dtype) { return dtype == CASCMM_DT_F32 ? 4 : 2; }
static bool grad_dtype(int dtype) { return dtype == CASCMM_DT_F32 || dtype == CASCMM_DT_F16 || dtype == CASCMM_DT_BF16; }

// Elements of a chunk: about 2048 chunks of what there is, 4096 elements at least; of more than 2^26 elements 8192 chunks, which balance better over several launches
struct GradPlan { int64_t chunk, parts; };
static int grad_plan(int count, const cascmm_gradient* list, GradPlan& plan) {
  if (count < 0) return CASCMM_ERR_BAD_SHAPE;
  if (count > 0 && !list) return CASCMM_ERR_NULL_POINTER;
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    if (list[i].elements < 0) return CASCMM_ERR_BAD_SHAPE;
    if (__builtin_add_overflow(total, list[i].elements, &total) || total > (int64_t)1 << 48) return CASCMM_ERR_TOO_LARGE;
  }
  const int64_t most = total > ((int64_t)1 << 26) ? 8192 : 2048;
  plan.chunk = std::max<int64_t>(kGradChunk, ((total + most - 1) / most + 255) / 256 * 256);
  plan.parts = 0;
  for (int i = 0; i < count; ++i) plan.parts += (list[i].elements + plan.chunk - 1) / plan.chunk;
  return plan.parts > (1 << 24) ? CASCMM_ERR_TOO_LARGE : CASCMM_OK;   // (a launch has fewer than 2^32 threads)
}

// Whether a result shares memory with another result, or with a gradient that is not its own (its own: the same elements in place)
static bool grad_overlap(int count, const cascmm_gradient* list) {
  struct Span { uintptr_t from, to; bool written; };
  std::vector<Span> spans;
  spans.reserve((size_t)count * 2);
  for (int i = 0; i < count; ++i) {
    const cascmm_gradient& g = list[i];
    if (g.elements == 0) continue;
    const uintptr_t from = (uintptr_t)g.data, out = (uintptr_t)g.out;
    spans.push_back({out, out + (uintptr_t)(g.elements * grad_size(g.out_dtype)), true});
    if (g.data != g.out || g.dtype != g.out_dtype) spans.push_back({from, from + (uintptr_t)(g.elements * grad_size(g.dtype)), false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& p, const Span& q) { return p.from < q.from; });
  uintptr_t read = 0, written = 0;   // ends of what came before
  for (const Span& s : spans) {
    if (s.from < written || (s.written && s.from < read)) return true;
    (s.written ? written : read) = std::max(s.written ? written : read, s.to);
  }
  return false;
}

// one pass over all tensors, as many at a time as a launch's arguments hold
template <typename Kernel>
static hipError_t grad_pass(Kernel kernel, GradBatch& b, int count, const cascmm_gradient* list, hipStream_t s) {
  hipError_t err = hipSuccess;
  unsigned part = 0;
  int at = 0;
  while (at < count) {
    unsigned chunks = 0;
    b.count = 0;
    b.part0 = part;
    for (; at < count && b.count < kGradTensors; ++at) {
      const cascmm_gradient& g = list[at];
      if (g.elements == 0) continue;
      const int k = b.count++;
      b.g[k] = g.data; b.out[k] = g.out; b.n[k] = g.elements; b.first[k] = chunks;
      b.dtype[k] = (unsigned char)g.dtype; b.out_dtype[k] = (unsigned char)g.out_dtype;
      chunks += (unsigned)((g.elements + b.chunk - 1) / b.chunk);
    }
    if (chunks) CASCMM_LAUNCH(err, kernel, dim3(chunks), dim3(256), 0, s, b);
    part += chunks;
  }
  return err;
}

}  // namespace cascmm

using namespace cascmm;

extern "C" {

size_t cascmm_gradients_workspace_bytes(int count, const cascmm_gradient* gradients) {
  GradPlan plan;
  if (grad_plan(count, gradients, plan) != CASCMM_OK) return 0;
  return 16 + (size_t)plan.parts * sizeof(double);
}

int cascmm_clip_gradients(int count, const cascmm_gradient* gradients, int norm_type, double max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  GradPlan plan;
  const int st = grad_plan(count, gradients, plan);
  if (st != CASCMM_OK) return st;
  if (norm_type < 0 || norm_type > 2) return CASCMM_ERR_BAD_FORMAT;
  if (!(max_norm >= 0)) return CASCMM_ERR_BAD_SHAPE;
  if (!norm) return CASCMM_ERR_NULL_POINTER;
  if ((uintptr_t)norm % 4) return CASCMM_ERR_ALIGNMENT;
  int results = 0, filled = 0;
  for (int i = 0; i < count; ++i) {
    const cascmm_gradient& g = gradients[i];
    if (!grad_dtype(g.dtype) || (g.out && g.out_dtype != g.dtype && g.out_dtype != CASCMM_DT_F32)) return CASCMM_ERR_BAD_DTYPE;
    if (g.elements == 0) continue;
    if (!g.data) return CASCMM_ERR_NULL_POINTER;
    if ((uintptr_t)g.data % grad_size(g.dtype) || (g.out && (uintptr_t)g.out % grad_size(g.out_dtype))) return CASCMM_ERR_ALIGNMENT;
    ++filled;
    results += g.out != nullptr;
  }
  if (results != 0 && results != filled) return CASCMM_ERR_NULL_POINTER;
  if (!workspace || workspace_bytes < 16 + (size_t)plan.parts * sizeof(double)) return CASCMM_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 16) return CASCMM_ERR_ALIGNMENT;
  try {
    if (results && grad_overlap(count, gradients)) return CASCMM_ERR_OVERLAP;
  } catch (const std::bad_alloc&) {
    return CASCMM_ERR_TOO_LARGE;
  }
  GradBatch b;
  memset(&b, 0, sizeof(b));
  b.chunk = plan.chunk;
  b.parts = (double*)((char*)workspace + 16);
  b.head = (double*)workspace;
  b.max_norm = max_norm;
  b.norm = norm;
  b.type = norm_type;
  b.all_parts = (unsigned)plan.parts;
  // (few partial sums are added by every workgroup of the second pass: a launch less)
  b.merged = results && plan.parts > 0 && plan.parts <= kGradMerged;
  const hipStream_t s = (hipStream_t)stream;
  hipError_t err = grad_pass(cascmm_gradient_parts_kernel<0>, b, count, gradients, s);
  if (!b.merged && err == hipSuccess)
    CASCMM_LAUNCH(err, cascmm_gradient_norm_kernel<0>, dim3(1), dim3(1024), 0, s, (const double*)b.parts, b.all_parts, norm_type, max_norm, norm, b.head);
  if (results && err == hipSuccess) err = grad_pass(cascmm_gradient_scale_kernel<0>, b, count, gradients, s);
  return err == hipSuccess ? CASCMM_OK : CASCMM_ERR_LAUNCH;
}

}  // extern "C"
