// A request kept for repeated launches (tb_request_*): the operator, its tensors and
// attributes as one handle, enqueued with one argument. A serving loop that runs the same
// operators on the same buffers every step pays for the request's assembly once; the checks and
// the kernel choice still run at every enqueue. No counterpart in the reference, whose
// Runtime::execute takes an OpRequest by value (titan-runtime/src/lib.rs:1171).
#include "ops_common.hpp"

namespace tb {

struct Request {
  tb_session* session = nullptr;
  tb_stream* stream = nullptr;
  std::string op;
  std::vector<tb_tensor> inputs, outputs;
  std::vector<tb_attr> attrs;
  std::vector<std::string> texts;  // keys and string values that `attrs` points to
};

namespace {

void drop(Request* r) {
  for (const auto* list : {&r->inputs, &r->outputs})
    for (const tb_tensor& t : *list) tb_buffer_release(t.buffer);
  tb_stream_release(r->stream);
  tb_session_release(r->session);
  delete r;
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" {

tb_status tb_request_create(tb_session* session, tb_stream* stream, const char* op, const tb_tensor* inputs,
                            uint32_t num_inputs, const tb_tensor* outputs, uint32_t num_outputs, const tb_attr* attrs,
                            uint32_t num_attrs, tb_request** out) try {
  Session* s = reinterpret_cast<Session*>(session);
  if (!out || !op || (num_inputs && !inputs) || (num_outputs && !outputs) || (num_attrs && !attrs))
    return contract("a request needs an operator name, its tensors and a place for the handle");
  if (!s) return set_error(TB_ERR_INVALID, "contract", "null session");
  if (num_inputs > 64 || num_outputs > 64 || num_attrs > 64)
    return contract("a request takes up to 64 inputs, outputs and attributes each");
  Stream* st = nullptr;
  tb_status rc = check_stream(s, stream, &st);
  if (rc) return rc;
  for (uint32_t i = 0; i < num_inputs + num_outputs; ++i) {
    const tb_tensor& t = i < num_inputs ? inputs[i] : outputs[i - num_inputs];
    Buffer* b = nullptr;
    if ((rc = check_buffer(s, t.buffer, &b))) return rc;
  }
  auto r = std::make_unique<Request>();
  r->op = op;
  r->inputs.assign(inputs, inputs + num_inputs);
  r->outputs.assign(outputs, outputs + num_outputs);
  r->texts.reserve(2 * (size_t)num_attrs);  // never grows: the attributes point into it
  for (uint32_t i = 0; i < num_attrs; ++i) {
    tb_attr a = attrs[i];
    if (a.key) a.key = r->texts.emplace_back(a.key).c_str();
    if (a.str) a.str = r->texts.emplace_back(a.str).c_str();
    r->attrs.push_back(a);
  }
  r->session = session;
  r->stream = stream;
  tb_session_retain(session);
  st->refs.fetch_add(1);
  for (const auto* list : {&r->inputs, &r->outputs})
    for (const tb_tensor& t : *list) tb_buffer_retain(t.buffer);
  *out = reinterpret_cast<tb_request*>(r.release());
  return TB_OK;
} catch (const std::exception& e) {
  return tb::caught(e);
}

tb_status tb_request_enqueue(const tb_request* request, tb_event** out) try {
  const Request* r = reinterpret_cast<const Request*>(request);
  if (!r) return contract("null request");
  return tb_execute_outputs(r->session, r->stream, r->op.c_str(), r->inputs.data(), (uint32_t)r->inputs.size(),
                            r->outputs.data(), (uint32_t)r->outputs.size(), r->attrs.data(), (uint32_t)r->attrs.size(),
                            out);
} catch (const std::exception& e) {
  return tb::caught(e);
}

void tb_request_release(tb_request* request) {
  if (request) drop(reinterpret_cast<Request*>(request));
}

}  // extern "C"
