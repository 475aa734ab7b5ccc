"""The XLA handlers of the distillation operators and of the sandwich norm compare the buffers that they are given with each other before
they hand their addresses to a kernel.  The handlers are compiled with g++ against buffers that have dimensions and no memory, with the C entries
replaced by ones that count their calls."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

MAIN = r"""
#include <cstdio>
#include <functional>
#include "xla_ffi.cc"

static int calls = 0;
extern "C" {
int tg_sandwich_norm_fwd(const void*, const void*, const void*, const void*, const void*, int, float, float, void*, void*, void*, float*, int64_t, int64_t, void*) { ++calls; return TG_OK; }
int64_t tg_sandwich_norm_bwd_scratch_bytes(int64_t rows, int64_t cols) { return rows * cols; }
int tg_sandwich_norm_bwd(const void*, const void*, const void*, const void*, const void*, int, float, float, const void*, const void*, void*, void*, void*, void*, void*, void*, int64_t, int64_t, void*) { ++calls; return TG_OK; }
int tg_top_logits(const void*, float, float, int32_t*, float*, float*, int64_t, int64_t, int64_t, int, void*) { ++calls; return TG_OK; }
int tg_softcap_distill(const tg_distill_args*, void*) { ++calls; return TG_OK; }
const char* tg_last_cuda_error(void) { return ""; }
}

using D = std::vector<int64_t>;
// each buffer in its turn with dimensions of another size: {name, right, wrong}
struct Arg { const char* name; D right, wrong; };
static void each(const char* handler, const std::vector<Arg>& args, const std::function<ffi::Error(const std::vector<D>&)>& call) {
  for (int which = -1; which < int(args.size()); ++which) {
    std::vector<D> d;
    for (int i = 0; i < int(args.size()); ++i) d.push_back(i == which ? args[size_t(i)].wrong : args[size_t(i)].right);
    calls = 0;
    const ffi::Error e = call(d);
    std::printf("%s %s %s %d\n", handler, which < 0 ? "-" : args[size_t(which)].name, e.code == ffi::ErrorCode::kOk ? "ok" : "invalid", calls);
  }
}

int main() {
  const D x = {2, 3, 256}, one = {256}, less = {2, 2, 256}, row = {2, 3}, rows = {2, 3, 1};
  for (int kind : {TG_GATE_NONE, TG_GATE_CHANNEL, TG_GATE_TOKEN}) {
    const D gate = kind == TG_GATE_CHANNEL ? one : kind == TG_GATE_TOKEN ? rows : D{};
    const D other = kind == TG_GATE_CHANNEL ? rows : one;      // a gate of the other kind
    std::vector<Arg> fwd = {{"branch", x, less}, {"post", one, {128}}, {"pre", one, {128}}, {"gate", gate, kind == TG_GATE_NONE ? gate : other},
                            {"x_new", x, less}, {"h", x, less}};
    std::vector<Arg> bwd = {{"branch", x, less}, {"post", one, {128}}, {"pre", one, {128}}, {"gate", gate, kind == TG_GATE_NONE ? gate : other}, {"g_new", x, less},
                            {"g_h", x, less}, {"dx", x, less}, {"dbranch", x, less}, {"dpost", one, {128}}, {"dpre", one, {128}},
                            {"dgate", gate, kind == TG_GATE_NONE ? gate : other}, {"scratch", {6 * 256}, {6 * 256 - 1}}};
    if (kind == TG_GATE_NONE) {                                 // (a gate that is not read may be any buffer)
      fwd.erase(fwd.begin() + 3);
      bwd.erase(bwd.begin() + 10);
      bwd.erase(bwd.begin() + 3);
      each("fwd0", fwd, [&](const std::vector<D>& d) { return SandwichNormFwd(nullptr, x, d[0], d[1], d[2], one, d[3], d[4], kind, 1.f, 1e-5f); });
      each("bwd0", bwd, [&](const std::vector<D>& d) { return SandwichNormBwd(nullptr, x, d[0], d[1], d[2], rows, d[3], d[4], d[5], d[6], d[7], d[8], rows, d[9], kind, 1.f, 1e-5f); });
      continue;
    }
    each(kind == TG_GATE_CHANNEL ? "fwd1" : "fwd2", fwd, [&](const std::vector<D>& d) { return SandwichNormFwd(nullptr, x, d[0], d[1], d[2], d[3], d[4], d[5], kind, 1.f, 1e-5f); });
    each(kind == TG_GATE_CHANNEL ? "bwd1" : "bwd2", bwd, [&](const std::vector<D>& d) {
      return SandwichNormBwd(nullptr, x, d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7], d[8], d[9], d[10], d[11], kind, 1.f, 1e-5f);
    });
    std::vector<Arg> quant = fwd;
    quant.push_back({"q", x, less});
    quant.push_back({"scales", {2, 3, 2}, {2, 3, 1}});
    each(kind == TG_GATE_CHANNEL ? "quant1" : "quant2", quant, [&](const std::vector<D>& d) {
      return SandwichNormQuantFwd(nullptr, x, d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7], kind, 1.f, 1e-5f);
    });
  }
  each("top", {{"ids", {2, 3, 8}, {2, 2, 8}}, {"logp", {2, 3, 8}, {2, 3, 7}}, {"log_rest", row, {2, 2}}},
       [&](const std::vector<D>& d) { return TopLogits(nullptr, x, d[0], d[1], d[2], 15.f, 1.f); });
  each("distill", {{"ids", {2, 3, 8}, {2, 2, 8}}, {"logp", {2, 3, 8}, {2, 3, 7}}, {"log_rest", row, {2, 2}}, {"targets", row, {2, 2}}, {"row_loss", row, {1}}, {"dlogits", x, less}},
       [&](const std::vector<D>& d) { return SoftcapDistill(nullptr, x, d[0], d[1], d[2], d[3], d[4], d[5], 15.f, 1.f, 0.5f); });
  return 0;
}
"""


@pytest.fixture(scope="module")
def results(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    where = tmp_path_factory.mktemp("ffi")
    (where / "main.cc").write_text(MAIN)
    inc = [os.path.join(ROOT, *p) for p in (("tests", "ffi_run"), ("tests", "ffi_stub"), ("include",), ("train_gpt_b200", "xla_ffi"))]
    # (the handlers of the other operators are compiled too, and never called)
    r = subprocess.run(["g++", "-std=c++17", "-w", *[f"-I{i}" for i in inc], str(where / "main.cc"), "-o", str(where / "main"), "-Wl,--unresolved-symbols=ignore-all"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([str(where / "main")], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    return [line.split() for line in r.stdout.splitlines()]


def test_buffers_that_fit_reach_the_kernel(results):
    right = [r for r in results if r[1] == "-"]
    assert len(right) == 10 and all(r[2:] == ["ok", "1"] for r in right), right


def test_a_buffer_of_another_size_is_refused(results):
    wrong = [r for r in results if r[1] != "-"]
    assert len(wrong) == 5 + 10 + 2 * (6 + 12 + 8) + 3 + 6
    assert not [r for r in wrong if r[2:] != ["invalid", "0"]]
