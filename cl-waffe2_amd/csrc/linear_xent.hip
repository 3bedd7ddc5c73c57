// linear_xent.hip -- softmax cross entropy over a vocabulary, straight from the hidden states and the
// token table, and its gradients.
//
//   s[n, v] = x[n] . w[v]          lse[n] = log sum_v exp s[n, v]          loss[n] = lse[n] - s[n, label[n]]
//   ds[n, v] = g[n] (exp(s[n, v] - lse[n]) - [v = label[n]])     dx = ds w     dw = ds^T x
//
// What the reference composes from !matmul, !softmax and cross-entropy-loss on one-hot labels
// (source/nn/criterion.lisp:82-196, the lm-head of examples/gpt-2/model.lisp:137-196) holds the (rows, vocab)
// logits, the softmax, the one-hot labels and their gradients.  Here the vocabulary is walked in pieces:
// a piece's logits live in a workspace, every row keeps a running maximum and sum, and the gradient forms
// a piece's logits anew.
#include <utility>

#include "wf2_rows.h"

namespace wf2 {

constexpr float kLog2eF = 1.44269504088896340736f;
constexpr float kLn2F = 0.693147180559945309417f;

// A row's running state over the pieces: maximum, sum of exp(s - maximum), the label's logit.
struct XentRow {
  float top, sum, at;
};

// One workgroup per row of a piece: fold the piece's maximum and sum into the row's state.
__global__ __launch_bounds__(kBlock) void xent_fold_piece(const float* __restrict__ s, long cols, long first,
                                                          const int32_t* __restrict__ labels,
                                                          XentRow* __restrict__ state) {
  __shared__ float part[kWavesPerBlock];
  const int64_t row = blockIdx.x;
  const float* r = s + row * cols;
  float top = -INFINITY;
  bool bad = false;
  for (long c = threadIdx.x; c < cols; c += kBlock) {
    top = fmaxf(top, r[c]);
    bad |= r[c] != r[c];
  }
  if (bad) top = NAN;
  // a maximum that lets a NaN through, as the sums below do
  const int w = threadIdx.x / kWave;
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) {
    const float other = __shfl_xor(top, o);
    top = (top != top || other != other) ? NAN : fmaxf(top, other);
  }
  if ((threadIdx.x & (kWave - 1)) == 0) part[w] = top;
  __syncthreads();
  const XentRow old = state[row];
  top = first ? old.top : -INFINITY;
#pragma unroll
  for (int i = 0; i < kWavesPerBlock; i++) top = (top != top || part[i] != part[i]) ? NAN : fmaxf(top, part[i]);
  __syncthreads();
  const float base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (long c = threadIdx.x; c < cols; c += kBlock) sum += __builtin_amdgcn_exp2f((r[c] - base) * kLog2eF);
  sum = wave_sum32(sum);
  if ((threadIdx.x & (kWave - 1)) == 0) part[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    float total = first ? old.sum * __builtin_amdgcn_exp2f((old.top - base) * kLog2eF) : 0.0f;
    for (int i = 0; i < kWavesPerBlock; i++) total += part[i];
    const long label = labels[row];
    float at = first ? old.at : NAN;   // a label behind the vocabulary finds no logit: its loss is NaN
    if (label >= first && label < first + cols) at = r[label - first];
    state[row] = XentRow{top, total, at};
  }
}

// loss and row statistic from the rows' states
__global__ __launch_bounds__(kBlock) void xent_rows(long rows, const XentRow* __restrict__ state,
                                                    const int32_t* __restrict__ labels, float* __restrict__ loss,
                                                    float* __restrict__ lse) {
  const long row = (long)blockIdx.x * kBlock + threadIdx.x;
  if (row >= rows) return;
  const XentRow r = state[row];
  const float l = r.top + logf(r.sum);
  lse[row] = l;
  loss[row] = labels[row] < 0 ? 0.0f : l - r.at;
}

// out[0] = sum of the losses (over the number of rows with a label)
__global__ __launch_bounds__(kBlock) void xent_reduce(long rows, const float* __restrict__ loss,
                                                      const int32_t* __restrict__ labels, bool mean,
                                                      float* __restrict__ out) {
  __shared__ double part[kWavesPerBlock];
  double sum = 0.0, count = 0.0;
  for (long i = threadIdx.x; i < rows; i += kBlock) {
    sum += loss[i];
    count += labels[i] >= 0;
  }
  sum = block_sum(sum, part);
  __syncthreads();
  count = block_sum(count, part);
  if (threadIdx.x == 0) out[0] = (float)(mean ? sum / count : sum);
}

// 1 / the number of rows with a label
__global__ __launch_bounds__(kBlock) void xent_weight(long rows, const int32_t* __restrict__ labels, float* __restrict__ out) {
  __shared__ double part[kWavesPerBlock];
  double count = 0.0;
  for (long i = threadIdx.x; i < rows; i += kBlock) count += labels[i] >= 0;
  count = block_sum(count, part);
  if (threadIdx.x == 0) out[0] = (float)(1.0 / count);
}

// s <- g (exp(s - lse) - [label]); rows without a label are zero whatever they hold
__global__ __launch_bounds__(kBlock) void xent_gradient(float* __restrict__ s, long cols, long first,
                                                        const int32_t* __restrict__ labels, const float* __restrict__ lse,
                                                        const float* __restrict__ weight, const float* __restrict__ dloss,
                                                        bool per_row, float scale, long vocab) {
  const int64_t row = blockIdx.x;
  float* r = s + row * cols;
  const long label = labels[row];
  float g = scale;
  if (weight) g *= weight[0];
  if (dloss) g *= dloss[per_row ? row : 0];
  if (label >= vocab) g = NAN;
  const float l = lse[row];
  for (long c = threadIdx.x; c < cols; c += kBlock) {
    const float p = __builtin_amdgcn_exp2f((r[c] - l) * kLog2eF) - (c + first == label ? 1.0f : 0.0f);
    r[c] = label < 0 ? 0.0f : g * p;
  }
}

// rows of x without a label contribute nothing to dw, also where they hold no numbers
__global__ __launch_bounds__(kBlock) void xent_clean_rows(const float* __restrict__ x, const int32_t* __restrict__ labels,
                                                          long dim, float* __restrict__ out) {
  const int64_t row = blockIdx.x;
  const bool held = labels[row] >= 0;
  for (long c = threadIdx.x; c < dim; c += kBlock) out[row * dim + c] = held ? x[row * dim + c] : 0.0f;
}

static bool meets(const void* a, int64_t na, const void* b, int64_t nb) {
  const char *p = (const char*)a, *q = (const char*)b;
  return p && q && p < q + nb * 4 && q < p + na * 4;
}

static int xent_check(const char* name, long rows, long dim, long vocab, const void* x, const void* w, const void* labels,
                      const void* lse, int reduction) {
  if (rows < 0 || dim < 0 || vocab < 0) return fail(WF2HIP_EINVAL, "%s: negative extent", name);
  if (reduction < WF2HIP_REDUCE_NONE || reduction > WF2HIP_REDUCE_MEAN)
    return fail(WF2HIP_EINVAL, "%s: unknown reduction %d", name, reduction);
  if (dim < 1 || vocab < 1) return fail(WF2HIP_EINVAL, "%s: needs a vocabulary and hidden states of at least one element", name);
  if (rows > INT32_MAX || dim > INT32_MAX || vocab > INT32_MAX)
    return fail(WF2HIP_EUNSUPPORTED, "%s: an extent beyond 2^31 - 1", name);
  if (!w || (rows && (!x || !labels || !lse))) return fail(WF2HIP_EINVAL, "%s: null pointer", name);
  return 0;
}

// columns of the vocabulary that a workspace of at most 256 MiB of logits takes
static long xent_piece(long rows, long vocab) {
  const int64_t fit = ((int64_t)64 << 20) / (rows > 0 ? rows : 1);
  const int64_t cols = fit < 256 ? 256 : fit / 256 * 256;
  return (long)(cols < vocab ? cols : vocab);
}

}  // namespace wf2

using namespace wf2;

WF2_API int wf2hip_linear_cross_entropy_f32(long rows, long dim, long vocab, const float* x, const float* w,
                                            const int32_t* labels, int reduction, float* loss, float* lse) {
  const char* name = "linear cross entropy";
  WF2_TRY(require_init());
  WF2_TRY(xent_check(name, rows, dim, vocab, x, w, labels, lse, reduction));
  const int64_t losses = reduction == WF2HIP_REDUCE_NONE ? rows : 1;
  if (losses && !loss) return fail(WF2HIP_EINVAL, "%s: null pointer", name);
  for (auto [out, n] : {std::pair<const float*, int64_t>(loss, losses), std::pair<const float*, int64_t>(lse, rows)})
    if (meets(out, n, x, (int64_t)rows * dim) || meets(out, n, w, (int64_t)vocab * dim) || meets(out, n, labels, rows))
      return fail(WF2HIP_EOVERLAP, "%s: an output overlaps an input", name);
  if (meets(loss, losses, lse, rows)) return fail(WF2HIP_EOVERLAP, "%s: the loss overlaps the row statistics", name);
  hipStream_t st = rt().stream;
  const long piece = xent_piece(rows, vocab);
  void *s = nullptr, *state = nullptr, *each = nullptr;
  int rc = 0;
  if (rows) {
    if ((rc = wf2hip_malloc_uninitialized(&s, (size_t)rows * piece * 4)) == 0 &&
        (rc = wf2hip_malloc_uninitialized(&state, (size_t)rows * sizeof(XentRow))) == 0 &&
        reduction != WF2HIP_REDUCE_NONE)
      rc = wf2hip_malloc_uninitialized(&each, (size_t)rows * 4);
    for (long c = 0; rc == 0 && c < vocab; c += piece) {
      const long cols = piece < vocab - c ? piece : vocab - c;
      rc = wf2hip_sgemm('T', 'N', cols, rows, dim, 1.0f, w + (int64_t)c * dim, dim, x, dim, 0.0f, (float*)s, cols);
      if (rc == 0) {
        xent_fold_piece<<<(uint32_t)rows, kBlock, 0, st>>>((const float*)s, cols, c, labels, (XentRow*)state);
        rc = after_launch("xent_fold_piece");
      }
    }
    if (rc == 0) {
      xent_rows<<<(uint32_t)ceil_div(rows, kBlock), kBlock, 0, st>>>(rows, (const XentRow*)state, labels,
                                                                    each ? (float*)each : loss, lse);
      rc = after_launch("xent_rows");
    }
  }
  if (rc == 0 && reduction != WF2HIP_REDUCE_NONE) {
    xent_reduce<<<1, kBlock, 0, st>>>(rows, (const float*)each, labels, reduction == WF2HIP_REDUCE_MEAN, loss);
    rc = after_launch("xent_reduce");
  }
  for (void* block : {s, state, each})
    if (block) (void)wf2hip_free(block);
  return rc;
}

WF2_API int wf2hip_linear_cross_entropy_backward_f32(long rows, long dim, long vocab, const float* x, const float* w,
                                                     const int32_t* labels, const float* lse, int reduction,
                                                     const float* dloss, float scale, float* dx, float* dw) {
  const char* name = "linear cross entropy backward";
  WF2_TRY(require_init());
  WF2_TRY(xent_check(name, rows, dim, vocab, x, w, labels, lse, reduction));
  if (!dw || (rows && !dx)) return fail(WF2HIP_EINVAL, "%s: null pointer", name);
  const int64_t nx = (int64_t)rows * dim, nw = (int64_t)vocab * dim, ng = reduction == WF2HIP_REDUCE_NONE ? rows : 1;
  for (auto [out, n] : {std::pair<const float*, int64_t>(dx, nx), std::pair<const float*, int64_t>(dw, nw)})
    if (meets(out, n, x, nx) || meets(out, n, w, nw) || meets(out, n, labels, rows) || meets(out, n, lse, rows) ||
        meets(out, n, dloss, ng))
      return fail(WF2HIP_EOVERLAP, "%s: a gradient overlaps an input", name);
  if (meets(dx, nx, dw, nw)) return fail(WF2HIP_EOVERLAP, "%s: the gradients overlap", name);
  if (rows == 0) return wf2hip_fill_f32(dw, (size_t)nw, 0.0f);
  hipStream_t st = rt().stream;
  const long piece = xent_piece(rows, vocab);
  void *s = nullptr, *clean = nullptr, *weight = nullptr;
  int rc = wf2hip_malloc_uninitialized(&s, (size_t)rows * piece * 4);
  if (rc == 0) rc = wf2hip_malloc_uninitialized(&clean, (size_t)nx * 4);
  if (rc == 0 && reduction == WF2HIP_REDUCE_MEAN) {
    rc = wf2hip_malloc_uninitialized(&weight, 4);
    if (rc == 0) {
      xent_weight<<<1, kBlock, 0, st>>>(rows, labels, (float*)weight);
      rc = after_launch("xent_weight");
    }
  }
  if (rc == 0) {
    xent_clean_rows<<<(uint32_t)rows, kBlock, 0, st>>>(x, labels, dim, (float*)clean);
    rc = after_launch("xent_clean_rows");
  }
  for (long c = 0; rc == 0 && c < vocab; c += piece) {
    const long cols = piece < vocab - c ? piece : vocab - c;
    const float* wc = w + (int64_t)c * dim;
    rc = wf2hip_sgemm('T', 'N', cols, rows, dim, 1.0f, wc, dim, (const float*)clean, dim, 0.0f, (float*)s, cols);
    if (rc == 0) {
      xent_gradient<<<(uint32_t)rows, kBlock, 0, st>>>((float*)s, cols, c, labels, lse, (const float*)weight, dloss,
                                                      reduction == WF2HIP_REDUCE_NONE, scale, vocab);
      rc = after_launch("xent_gradient");
    }
    if (rc == 0)
      rc = wf2hip_sgemm('N', 'N', dim, rows, cols, 1.0f, wc, dim, (const float*)s, cols, c ? 1.0f : 0.0f, dx, dim);
    if (rc == 0)
      rc = wf2hip_sgemm('N', 'T', dim, cols, rows, 1.0f, (const float*)clean, dim, (const float*)s, cols, 0.0f,
                        dw + (int64_t)c * dim, dim);
  }
  for (void* block : {s, clean, weight})
    if (block) (void)wf2hip_free(block);
  return rc;
}
