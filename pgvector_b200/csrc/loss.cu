// loss.cu - softmax loss of queries over all of a shard's rows, and its
// gradients (AnnB200SoftmaxLoss, AnnB200SoftmaxLossGrad).
//
// The rows are walked in pieces. Forward: a piece's logits, then each query's
// running maximum m and sum s = sum exp(l - m). Gradient: a piece's logits
// again, G = grad * (exp(l - lse) - onehot) over them in place, dqueries +=
// G rows, drows = G^T queries.
#include <algorithm>
#include <cmath>

#include "ops.cuh"

namespace annb200 {
namespace {

constexpr uint64_t kPieceBytes = 64ull << 20;  // a piece's logits

struct Plan {
  uint64_t piece;   // rows a piece
  uint64_t logits, m, s, t, dq, total;
};

uint64_t up256(uint64_t x) { return (x + 255) & ~255ull; }

Plan plan_of(const AnnB200LossJob &j) {
  Plan p;
  const uint64_t nq = std::max(1u, j.nq);
  p.piece = std::min<uint64_t>(j.nrows, std::max<uint64_t>(64, std::min<uint64_t>(1u << 20, kPieceBytes / (4 * nq))));
  p.logits = 0;
  p.m = up256(nq * p.piece * 4);
  p.s = p.m + up256(nq * 4);
  p.t = p.s + up256(nq * 4);
  p.dq = p.t + up256(nq * 4);
  p.total = p.dq + up256(nq * j.dims * 4);
  return p;
}

// One block a query: the running maximum, sum and target logit over a piece.
__global__ void __launch_bounds__(256) piece_stats(const float *logits, uint64_t n, uint64_t first, bool start,
                                                   const int64_t *targets, float *m, float *s, float *t) {
  const uint32_t q = blockIdx.x;
  const float *l = logits + q * n;
  __shared__ float red[256];
  float mx = -INFINITY;
  for (uint64_t i = threadIdx.x; i < n; i += 256) mx = fmaxf(mx, l[i]);
  red[threadIdx.x] = mx;
  __syncthreads();
  for (int h = 128; h; h >>= 1) {
    if (threadIdx.x < h) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + h]);
    __syncthreads();
  }
  const float old = start ? -INFINITY : m[q];
  mx = fmaxf(red[0], old);
  const float base = mx == -INFINITY ? 0.0f : mx;
  __syncthreads();
  float sum = 0.0f;
  for (uint64_t i = threadIdx.x; i < n; i += 256) sum += expf(l[i] - base);
  red[threadIdx.x] = sum;
  __syncthreads();
  for (int h = 128; h; h >>= 1) {
    if (threadIdx.x < h) red[threadIdx.x] += red[threadIdx.x + h];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    s[q] = red[0] + (start ? 0.0f : s[q] * expf(old - base));
    m[q] = mx;
    const int64_t at = targets[q] - (int64_t)first;
    if (at >= 0 && at < (int64_t)n) t[q] = l[at];
  }
}

__global__ void finish(uint32_t nq, uint64_t nrows, const int64_t *targets, const float *m, const float *s,
                       const float *t, float *loss, float *lse, int32_t *status) {
  const uint32_t q = blockIdx.x * blockDim.x + threadIdx.x;
  if (q >= nq) return;
  const bool bad = targets[q] >= (int64_t)nrows;
  const float ls = logf(s[q]);
  if (lse) lse[q] = m[q] + ls;
  if (loss) loss[q] = targets[q] < 0 ? 0.0f : (bad ? NAN : (m[q] - t[q]) + ls);
  if (status) status[q] = bad ? OP_INVALID : OP_OK;
}

__global__ void piece_grad(float *logits, uint64_t n, uint64_t first, uint64_t nrows, const int64_t *targets,
                           const float *lse, const float *grad) {
  const uint32_t q = blockIdx.x;
  const int64_t t = targets[q];
  const float g = t < 0 || t >= (int64_t)nrows ? 0.0f : (grad ? grad[q] : 1.0f);
  const bool kept = t >= 0 && t < (int64_t)nrows;
  const float z = lse[q];
  for (uint64_t i = threadIdx.x; i < n; i += 256) {
    const float p = expf(logits[q * n + i] - z) - ((int64_t)(first + i) == t ? 1.0f : 0.0f);
    logits[q * n + i] = kept ? g * p : 0.0f;
  }
}

template <typename T>
__global__ void store_queries(const float *sum, uint64_t n, T *out) {
  const uint64_t i = blockIdx.x * 256ull + threadIdx.x;
  if (i < n) out[i] = from_float<T>(sum[i]);
}

template <typename T>
int run_loss(const AnnB200LossJob &j, bool grad, cudaStream_t st) {
  const Plan p = plan_of(j);
  uint8_t *ws = static_cast<uint8_t *>(j.workspace);
  float *logits = reinterpret_cast<float *>(ws + p.logits), *m = reinterpret_cast<float *>(ws + p.m);
  float *s = reinterpret_cast<float *>(ws + p.s), *t = reinterpret_cast<float *>(ws + p.t);
  float *dq = reinterpret_cast<float *>(ws + p.dq);
  const T *x = static_cast<const T *>(j.queries), *w = static_cast<const T *>(j.rows);
  const uint64_t xs = j.query_stride, ws_ = j.row_stride;
  const float scale = j.scale;
  const int64_t *targets = j.targets;
  const uint64_t nrows = j.nrows;
  T *drows = static_cast<T *>(j.drows);
  unsigned long long launches = 0;
  for (uint64_t first = 0; first < nrows; first += p.piece) {
    const uint64_t n = std::min(p.piece, nrows - first);
    launch_simt_gemm([=] __device__(int64_t i, int64_t k) { return to_float(x[i * xs + k]); },
                     [=] __device__(int64_t r, int64_t k) { return to_float(w[(first + r) * ws_ + k]); }, j.nq, n,
                     j.dims, [=] __device__(int64_t i, int64_t r, float v) { logits[i * n + r] = v * scale; }, st);
    launches++;
    if (!grad) {
      piece_stats<<<j.nq, 256, 0, st>>>(logits, n, first, first == 0, targets, m, s, t);
      launches++;
      continue;
    }
    piece_grad<<<j.nq, 256, 0, st>>>(logits, n, first, nrows, targets, j.lse, j.grad);
    launches++;
    if (j.dqueries) {
      const bool start = first == 0;
      launch_simt_gemm([=] __device__(int64_t i, int64_t r) { return logits[i * n + r]; },
                       [=] __device__(int64_t d, int64_t r) { return to_float(w[(first + r) * ws_ + d]); }, j.nq,
                       j.dims, n,
                       [=, dims = j.dims] __device__(int64_t i, int64_t d, float v) {
                         float *o = dq + i * dims + d;
                         const bool kept = targets[i] >= 0 && targets[i] < (int64_t)nrows;
                         *o = kept ? (start ? 0.0f : *o) + v * scale : 0.0f;
                       },
                       st);
      launches++;
    }
    if (drows) {
      launch_simt_gemm([=] __device__(int64_t r, int64_t i) { return logits[i * n + r]; },
                       [=] __device__(int64_t d, int64_t i) {
                         // a query without a target adds nothing, whatever it holds
                         return targets[i] >= 0 && targets[i] < (int64_t)nrows ? to_float(x[i * xs + d]) : 0.0f;
                       },
                       n, j.dims, j.nq,
                       [=, dims = j.dims] __device__(int64_t r, int64_t d, float v) {
                         drows[(first + r) * dims + d] = from_float<T>(v * scale);
                       },
                       st);
      launches++;
    }
  }
  if (!grad) {
    finish<<<(j.nq + 127) / 128, 128, 0, st>>>(j.nq, nrows, targets, m, s, t, j.loss, j.lse, j.status);
    launches++;
  } else if (j.dqueries) {
    const uint64_t n = (uint64_t)j.nq * j.dims;
    store_queries<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(dq, n, static_cast<T *>(j.dqueries));
    launches++;
  }
  return op_launched(grad ? "softmax loss gradient" : "softmax loss", launches);
}

int check_job(const AnnB200LossJob *j) {
  if (!j) return report_error(OP_INVALID, "NULL job");
  if (!op_dtype(j->dtype)) return report_error(OP_INVALID, "type %u", j->dtype);
  if (j->dims == 0 || j->dims > 65536) return report_error(OP_INVALID, "%u dimensions", j->dims);
  if (j->nq > (1u << 22)) return report_error(OP_INVALID, "more than 2^22 queries");
  if (j->nrows == 0 || j->nrows > 0x7fffffffull) return report_error(OP_INVALID, "no rows, or 2^31 and more");
  if (j->query_stride < j->dims || j->row_stride < j->dims) return report_error(OP_INVALID, "rows overlap");
  if (!std::isfinite(j->scale)) return report_error(OP_INVALID, "scale is not finite");
  return OP_OK;
}

int run_job(const AnnB200LossJob *j, bool grad, void *stream) {
  int r = check_job(j);
  if (r != OP_OK || j->nq == 0) return r;
  if (!j->queries || !j->rows || !j->targets) return report_error(OP_INVALID, "NULL pointer");
  if (grad && !j->lse) return report_error(OP_INVALID, "the gradient needs lse");
  if (grad && !j->dqueries && !j->drows) return OP_OK;
  if (!j->workspace || (reinterpret_cast<uintptr_t>(j->workspace) & 255) || j->workspace_bytes < plan_of(*j).total)
    return report_error(OP_INVALID, "workspace too small or not 256-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (j->dtype) {
    case ANNB200_F32: return run_loss<float>(*j, grad, st);
    case ANNB200_F16: return run_loss<__half>(*j, grad, st);
    default: return run_loss<__nv_bfloat16>(*j, grad, st);
  }
}

}  // namespace
}  // namespace annb200

using namespace annb200;

extern "C" int AnnB200SoftmaxLossWorkspace(const AnnB200LossJob *job, uint64_t *loss_bytes, uint64_t *grad_bytes) {
  int r = check_job(job);
  if (r != OP_OK) return r;
  if (loss_bytes) *loss_bytes = plan_of(*job).total;
  if (grad_bytes) *grad_bytes = plan_of(*job).total;
  return OP_OK;
}
extern "C" int AnnB200SoftmaxLoss(const AnnB200LossJob *job, void *stream) { return run_job(job, false, stream); }
extern "C" int AnnB200SoftmaxLossGrad(const AnnB200LossJob *job, void *stream) { return run_job(job, true, stream); }
