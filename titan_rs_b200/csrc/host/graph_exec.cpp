// CUDA graphs over a session stream: the device work enqueued on a stream between
// tb_capture_begin and tb_capture_end (operators, device-to-device copies, memsets,
// event records) becomes one graph that tb_graph_exec_launch replays with a single
// launch. No counterpart in the reference, whose runtime launches every kernel from
// the host (titan-backend-cuda/src/lib.rs:1413-1507); here it serves launch-bound
// sequences of small operators.
//
// Capture is per thread (CU_STREAM_CAPTURE_MODE_THREAD_LOCAL): other host threads keep
// using the session meanwhile. Work that is not stream-ordered device work invalidates
// the capture and tb_capture_end reports it: host-staged uploads and downloads (their
// host side runs at enqueue time), waits on the host, and an operator's first use of
// per-stream scratch memory (it allocates), so such an operator runs once before capture.
// The attention operators' workspace is the graph's own (stream_workspace): allocated at
// capture, freed with the graph, shared with no other graph and no eager call. Graphs and
// workspaces released while a stream is being captured are freed when the last capture ends.
// A replay reads and writes the same device buffers the captured work named.
#include "ops_common.hpp"

namespace tb {

struct GraphExec : RefCounted {
  Session* session = nullptr;
  CUgraphExec exec = nullptr;
  std::vector<CUdeviceptr> work;  // workspace of its operators (stream_workspace)
  CUevent done = nullptr;  // of its last launch, where it has workspace
  std::mutex launch;       // keeps `done` in the launches' order
};

}  // namespace tb

using namespace tb;

extern "C" {

tb_status tb_capture_begin(tb_session* session, tb_stream* stream) try {
  Session* s = reinterpret_cast<Session*>(session);
  if (!s) return set_error(TB_ERR_INVALID, "capture", "null session");
  Stream* st = nullptr;
  tb_status rc = check_stream(s, stream, &st);
  if (rc) return rc;
  rc = activate(s);
  if (rc) return rc;
  TB_CU("cuStreamBeginCapture", driver()->cuStreamBeginCapture_v2(st->raw, CU_STREAM_CAPTURE_MODE_THREAD_LOCAL));
  st->capture = capture_id(st);
  if (st->capture) capture_began(s);
  return TB_OK;
} catch (const std::exception& e) {
  return tb::caught(e);
}

tb_status tb_capture_end(tb_session* session, tb_stream* stream, tb_graph_exec** out) try {
  Session* s = reinterpret_cast<Session*>(session);
  if (!s || !out) return set_error(TB_ERR_INVALID, "capture", "null argument");
  *out = nullptr;
  Stream* st = nullptr;
  tb_status rc = check_stream(s, stream, &st);
  if (rc) return rc;
  rc = activate(s);
  if (rc) return rc;
  const DriverApi* d = driver();
  CUgraph graph = nullptr;
  // What needs host memory comes before the capture's end, so that it can still be ended without.
  const unsigned long long id = st->capture;  // (an invalidated capture has lost its id in the driver)
  auto g = std::make_unique<GraphExec>();
  std::vector<CUdeviceptr> work = id ? take_captured_work(s, id) : std::vector<CUdeviceptr>();
  st->capture = 0;
  const auto drop_work = [&] {
    retire_work(s, {nullptr, work, nullptr});
  };
  // Ends the capture in every case; an invalidated capture (a call that cannot be
  // captured ran meanwhile) reports the driver's error and yields no graph.
  const CUresult ended = d->cuStreamEndCapture(st->raw, &graph);
  if (id) capture_ended(s);
  if (ended != CUDA_SUCCESS || !graph) drop_work();
  if (ended != CUDA_SUCCESS) return cu_error("cuStreamEndCapture", ended);
  if (!graph) return set_error(TB_ERR_INVALID, "capture", "nothing was captured");
  CUgraphExec exec = nullptr;
  const CUresult r = d->cuGraphInstantiateWithFlags(&exec, graph, 0);
  d->cuGraphDestroy(graph);
  if (r != CUDA_SUCCESS) {
    drop_work();
    return cu_error("cuGraphInstantiate", r);
  }
  CUevent done = nullptr;
  if (!work.empty()) {
    const CUresult e = d->cuEventCreate(&done, CU_EVENT_DISABLE_TIMING);
    if (e != CUDA_SUCCESS) {
      d->cuGraphExecDestroy(exec);
      drop_work();
      return cu_error("cuEventCreate", e);
    }
  }
  g->session = s;
  g->done = done;
  g->exec = exec;
  g->work = std::move(work);
  s->refs.fetch_add(1);
  *out = reinterpret_cast<tb_graph_exec*>(g.release());
  return TB_OK;
} catch (const std::exception& e) {
  return tb::caught(e);
}

tb_status tb_graph_exec_launch(tb_session* session, tb_graph_exec* graph, tb_stream* stream) try {
  Session* s = reinterpret_cast<Session*>(session);
  GraphExec* g = reinterpret_cast<GraphExec*>(graph);
  if (!s || !g) return set_error(TB_ERR_INVALID, "launch", "null argument");
  if (g->session != s) return set_error(TB_ERR_INVALID, "launch", "graph belongs to another session");
  Stream* st = nullptr;
  tb_status rc = check_stream(s, stream, &st);
  if (rc) return rc;
  rc = activate(s);
  if (rc) return rc;
  const DriverApi* d = driver();
  if (g->work.empty()) {
    TB_CU("cuGraphLaunch", d->cuGraphLaunch(g->exec, st->raw));
    return TB_OK;
  }
  // (A graph that took this one in would outlive its workspace.)
  if (stream_capturing(st))
    return set_error(TB_ERR_INVALID, "launch", "a graph with operators' workspace cannot be launched into a capture");
  std::lock_guard<std::mutex> lock(g->launch);
  TB_CU("cuGraphLaunch", d->cuGraphLaunch(g->exec, st->raw));
  TB_CU("cuEventRecord", d->cuEventRecord(g->done, st->raw));
  return TB_OK;
} catch (const std::exception& e) {
  return tb::caught(e);
}

void tb_graph_exec_release(tb_graph_exec* graph) {
  GraphExec* g = reinterpret_cast<GraphExec*>(graph);
  if (!g || g->refs.fetch_sub(1) != 1) return;
  Session* s = g->session;
  const DriverApi* d = driver();
  if (d && g->exec) {
    d->cuCtxSetCurrent(s->context);
    retire_work(s, {g->exec, std::move(g->work), g->done});
  }
  delete g;
  tb_session_release(reinterpret_cast<tb_session*>(s));
}

}  // extern "C"
