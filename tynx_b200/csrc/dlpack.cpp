// Zero-copy exchange of device tensors with other libraries in one process
// (the DLPack in-memory structure), ordered on the streams of both sides.
//
// A lent block stays out of the allocator's free lists until its owner and
// every borrower are done with it.  A loan may end on any thread (whichever
// drops the borrowed tensor): that records an event on the borrower's stream
// and notes it; the context's own thread collects the note on its next
// allocation, makes the compute stream wait for the event, and frees the block
// in stream order.  The borrower's stream is not used after the loan has ended:
// it may be gone by then.  The legacy default stream never is: its loans share
// one event, recorded when they are collected (0.3 us a loan less).  So do those
// of threads' default streams, which the legacy one waits for: their handle
// means another stream on another thread.
#include <new>

#include "common.h"

namespace {

// The structure's layout is the protocol's (version without a header).
struct DlDevice {
  int32_t type, id;
};
struct DlType {
  uint8_t code, bits;
  uint16_t lanes;
};
struct DlTensor {
  void *data;
  DlDevice device;
  int32_t ndim;
  DlType dtype;
  int64_t *shape, *strides;
  uint64_t byte_offset;
};
struct DlManaged {
  DlTensor t;
  void *owner;
  void (*deleter)(DlManaged *);
};

struct Loan {
  DlManaged managed;
  int64_t shape[TX_MAX_DIMS];
  tx_ctx *ctx;
  void *block;
  cudaStream_t borrower;
  cudaEvent_t passed;  // null where the borrower's stream cannot go away
};

// Whether work issued to the stream runs, rather than becoming part of a graph.
cudaError_t runs(cudaStream_t stream, bool &yes) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(stream, &status);
  if (e != cudaSuccess) cudaGetLastError();  // not the borrower's next call's
  yes = e == cudaSuccess && status == cudaStreamCaptureStatusNone;
  return e == cudaErrorStreamCaptureImplicit ? cudaSuccess : e;
}

// Where the event cannot be recorded the block stays lent: on a stream that is being captured it would become
// part of the borrower's graph, which may reference the block (and a wait for it would draw the compute stream
// into that capture).
void end_loan(DlManaged *m) {
  Loan *loan = static_cast<Loan *>(m->owner);
  tx_ctx *ctx = loan->ctx;
  bool ok = true;
  if (loan->passed) {
    DeviceScope device(ctx);
    runs(loan->borrower, ok);
    if (ok && cudaEventRecord(loan->passed, loan->borrower) != cudaSuccess) {
      cudaGetLastError();
      ok = false;
    }
    if (!ok) cudaEventDestroy(loan->passed);
  }
  try {
    std::lock_guard<std::mutex> hold(ctx->alloc.lock);
    if (ok) ctx->alloc.ended.push_back({loan->block, loan->passed, loan->borrower});
  } catch (...) {  // no host memory for the note: the block stays lent
  }
  delete loan;
}

int join(tx_ctx *ctx, cudaStream_t first, cudaStream_t then) {
  if (!ctx->order) TX_CUDA(ctx, cudaEventCreateWithFlags(&ctx->order, cudaEventDisableTiming));
  TX_CUDA(ctx, cudaEventRecord(ctx->order, first));
  TX_CUDA(ctx, cudaStreamWaitEvent(then, ctx->order, 0));
  return TX_OK;
}

}  // namespace

void tx_collect_loans(tx_ctx *ctx) {
  if (ctx->capturing) return;  // a capture cannot wait for work outside it
  std::vector<tx_allocator::Ended> ended;
  {
    std::lock_guard<std::mutex> hold(ctx->alloc.lock);
    if (ctx->alloc.ended.empty()) return;
    ended.swap(ctx->alloc.ended);
  }
  DeviceScope device(ctx);
  enum { kUnknown, kJoined, kLater } legacy = kUnknown;
  for (const auto &loan : ended) {
    if (loan.passed) {
      if (cudaStreamWaitEvent(ctx->stream, loan.passed, 0) != cudaSuccess) {
        cudaGetLastError();
        cudaEventDestroy(loan.passed);
        continue;  // no order with the borrower: the block stays lent
      }
      ctx->alloc.spare_events.push_back(loan.passed);
    } else if (loan.stream != ctx->stream) {
      if (legacy == kUnknown) {  // while a stream that synchronises with it is captured, it takes no work
        bool yes;
        runs(cudaStreamLegacy, yes);
        legacy = yes && join(ctx, cudaStreamLegacy, ctx->stream) == TX_OK ? kJoined : kLater;
      }
      if (legacy == kLater) {
        std::lock_guard<std::mutex> hold(ctx->alloc.lock);
        ctx->alloc.ended.push_back(loan);
        continue;
      }
    }
    tx_free_raw(ctx, loan.block);
  }
}

extern "C" int tx_dlpack_export(tx_ctx *ctx, void *d_block, void *d_data, int dtype, const int64_t *shape, int ndim,
                                void *stream, void **out) {
  if (!ctx || !out) return TX_ERR_INVALID;
  *out = nullptr;
  if (ctx->capturing) return tx_fail(ctx, TX_ERR_CAPTURE, "a tensor cannot be exported during a capture");
  if (dtype < TX_DL_F32 || dtype > TX_DL_BOOL || ndim < 0 || ndim > TX_MAX_DIMS || (ndim && !shape))
    return tx_fail(ctx, TX_ERR_INVALID, "dlpack export: dtype or rank");
  {
    std::lock_guard<std::mutex> hold(ctx->alloc.blocks);
    if (!ctx->alloc.live.count(d_block))
      return tx_fail(ctx, TX_ERR_INVALID, "only a tensor that owns its memory can be exported; clone() it first");
  }
  DeviceScope device(ctx);
  cudaStream_t borrower = stream ? static_cast<cudaStream_t>(stream) : cudaStreamLegacy;
  cudaEvent_t passed = nullptr;
  if (borrower != ctx->stream) {
    bool yes;
    TX_CUDA(ctx, runs(borrower, yes));
    if (!yes) return tx_fail(ctx, TX_ERR_CAPTURE, "a tensor cannot be exported to a stream that is being captured");
    TX_TRY(join(ctx, ctx->stream, borrower));
    std::vector<cudaEvent_t> &spare = ctx->alloc.spare_events;
    if (borrower == cudaStreamPerThread) borrower = cudaStreamLegacy;
    if (borrower != cudaStreamLegacy && spare.empty()) {
      TX_CUDA(ctx, cudaEventCreateWithFlags(&passed, cudaEventDisableTiming));
    } else if (borrower != cudaStreamLegacy) {
      passed = spare.back();
      spare.pop_back();
    }
  }
  Loan *loan = new (std::nothrow) Loan();
  try {
    std::lock_guard<std::mutex> hold(ctx->alloc.blocks);
    if (loan) ++ctx->alloc.lent[d_block].others;
  } catch (...) {
    delete loan;
    loan = nullptr;
  }
  if (!loan) {
    if (passed) cudaEventDestroy(passed);
    return tx_fail(ctx, TX_ERR_OOM, "dlpack export");
  }
  static const DlType types[3] = {{2, 32, 1}, {0, 64, 1}, {6, 8, 1}};
  for (int i = 0; i < ndim; ++i) loan->shape[i] = shape[i];
  loan->managed.t = DlTensor{d_data, {2 /* CUDA */, ctx->device}, ndim, types[dtype], loan->shape, nullptr, 0};
  loan->managed.owner = loan;
  loan->managed.deleter = end_loan;
  loan->ctx = ctx;
  loan->block = d_block;
  loan->borrower = borrower;
  loan->passed = passed;
  *out = &loan->managed;
  return TX_OK;
}

extern "C" int tx_dlpack_release(void *managed) {
  DlManaged *m = static_cast<DlManaged *>(managed);
  if (m && m->deleter) m->deleter(m);
  return TX_OK;
}

extern "C" int tx_dlpack_give_back(tx_ctx *ctx, void *managed) {
  if (!ctx) return TX_ERR_INVALID;
  {
    std::lock_guard<std::mutex> hold(ctx->capture_lock);
    if (ctx->capturing) {  // the graph may reference the memory: it stays as long as the graph
      try {
        ctx->alloc.arena->borrowed.push_back(managed);
      } catch (...) {  // no host memory for the note: it stays for good
      }
      return TX_OK;
    }
    // a stream that failed no longer uses the memory either
    cudaStreamSynchronize(ctx->stream);
    cudaStreamSynchronize(ctx->comm);
  }
  return tx_dlpack_release(managed);  // calls into the other library: not under the lock
}
