"""Host side of the block-scaled e4m3 path, without a GPU: the numpy oracle
against torch's e4m3 type, the refusals of the C entries and of the Python
calls, and the sizes and strides that the calls hand to the C entries."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8 as O

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def L():
    from nanopointllm_b200 import _lib
    return _lib


@pytest.fixture
def F(monkeypatch):
    """nanopointllm_b200.fp8 on CPU tensors: the device check is off and the
    C call is written down instead of made."""
    from nanopointllm_b200 import fp8
    calls = []
    monkeypatch.setattr(fp8, "_same_device", lambda *a: None)
    monkeypatch.setattr(fp8, "_call", lambda fn, device, *args: calls.append((fn.__name__, args)))
    fp8_calls = calls
    return fp8, fp8_calls


def test_oracle_rounds_as_the_type():
    table = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(E4M3).float().numpy()
    fin = table[np.isfinite(table)]
    np.testing.assert_array_equal(O.round_e4m3(fin), fin)
    g = np.random.default_rng(0)
    x = np.concatenate([g.normal(size=4000) * s for s in (1e-3, 0.05, 1.0, 60.0)]).astype(np.float32)
    pos = np.sort(fin[fin >= 0]).astype(np.float32)
    x = np.clip(np.concatenate([x, (pos[1:] + pos[:-1]) / 2]), -448, 448)  # ties among them
    np.testing.assert_array_equal(O.round_e4m3(x), torch.from_numpy(x).to(E4M3).float().numpy())
    assert (np.abs(O.round_e4m3(x) - x) <= O.half_step_e4m3(x)).all()


def _buf(n=1 << 16):
    b = ctypes.create_string_buffer(n + 16)
    at = ctypes.addressof(b)
    return b, at + (-at) % 16


def test_c_entries_refuse_bad_arguments(L):
    keep, p = _buf()
    arg, bad = L.NPL_ERR_ARG, []
    q = L.lib.npl_fp8_quant_rows
    bad += [q(p, 7, 4, 256, 256, p, 256, p, 2, None),       # element type
            q(p, 1, -1, 256, 256, p, 256, p, 2, None),      # rows
            q(p, 1, 4, 0, 256, p, 256, p, 2, None),         # columns
            q(p, 1, 4, 256, 255, p, 256, p, 2, None),       # rows that overlap
            q(p, 1, 4, 256, 256, p, 255, p, 2, None),       # code stride
            q(p, 1, 4, 256, 256, p, 256, p, 1, None),       # scale stride
            q(None, 1, 4, 256, 256, p, 256, p, 2, None), q(p, 1, 4, 256, 256, None, 256, p, 2, None),
            q(p, 1, 4, 256, 256, p, 256, None, 2, None),
            q(p + 1, 1, 4, 256, 256, p, 256, p, 2, None),   # alignment of the elements
            q(p, 1, 4, 256, 256, p, 256, p + 2, 2, None),
            q(p, 1, 1 << 40, 256, 256, p, 256, p, 2, None), q(p, 1, 4, 1 << 40, 1 << 40, p, 1 << 40, p, 1 << 33, None)]
    w = L.lib.npl_fp8_quant_weight
    bad += [w(p, 9, 4, 256, 256, p, 256, p, 2, None), w(p, 1, 4, 256, 200, p, 256, p, 2, None)]
    r = L.lib.npl_fp8_rmsnorm_quant
    ok = dict(x=p, ldx=256, res=p, ldr=256, w=p, dt=1, eps=1e-6, rows=4, cols=256, so=p, lds=256, q=p, ldq=256, s=p,
              ldsc=2, st=None)
    for change in (dict(dt=0), dict(res=None), dict(so=None), dict(w=None), dict(ldr=255), dict(lds=1), dict(ldx=2)):
        bad.append(r(*{**ok, **change}.values()))
    s = L.lib.npl_fp8_silu_mul_quant
    bad += [s(p, 256, p, 256, 0, 4, 256, p, 256, p, 2, None), s(p, 100, p, 256, 1, 4, 256, p, 256, p, 2, None),
            s(p, 256, None, 256, 1, 4, 256, p, 256, p, 2, None)]
    lin = L.lib.npl_fp8_linear
    ok = dict(qa=p, lda=256, sa=p, ldsa=2, qw=p, ldw=256, sw=p, ldsw=2, bias=None, M=4, N=8, K=256, res=None, ldr=0,
              out=p, ldo=8, dt=1, st=None)
    for change in (dict(M=-1), dict(N=0), dict(K=0), dict(K=1 << 40), dict(qa=p + 8), dict(qw=p + 1), dict(lda=264),
                   dict(ldw=250), dict(lda=240), dict(ldsa=1), dict(ldsw=1), dict(dt=0), dict(ldo=7),
                   dict(res=p, ldr=7), dict(out=p + 1), dict(bias=p + 2), dict(out=None), dict(sw=None)):
        bad.append(lin(*{**ok, **change}.values()))
    assert bad == [arg] * len(bad), bad
    assert b"npl_fp8_linear" in L.lib.npl_last_error_string()
    # no rows: nothing to launch, no device needed
    assert lin(*{**ok, "M": 0, "qa": None, "sa": None, "out": None}.values()) == L.NPL_OK
    assert q(None, 1, 0, 256, 256, None, 256, None, 2, None) == L.NPL_OK


def test_cpu_tensors_are_refused():
    from nanopointllm_b200 import fp8
    with pytest.raises(ValueError, match="CUDA"):
        fp8.quantize_token_blocks(torch.zeros(2, 128, dtype=torch.float16))


def test_quantiser_layouts(F):
    f, calls = F
    x = torch.zeros(6, 301, dtype=torch.float16)
    q, s = f.quantize_token_blocks(x[:, 1:301])  # strided rows go as they are
    name, a = calls.pop()
    assert name == "npl_fp8_quant_rows" and a[1:5] == (f.L.NPL_F16, 6, 300, 301) and a[6] == 304 and a[8] == 3
    assert q.shape == (6, 300) and q.stride(0) == 304 and s.shape == (6, 3)
    q, s = f.quantize_token_blocks(torch.zeros(2, 3, 256).transpose(0, 1))
    assert q.shape == (3, 2, 256) and s.shape == (3, 2, 2)
    assert calls.pop()[1][1:5] == (f.L.NPL_F32, 6, 256, 256)
    q, s = f.quantize_token_blocks(torch.zeros(1, 256, dtype=torch.bfloat16).expand(4, 256))  # broadcast rows
    assert calls.pop()[1][4] == 256
    q, s = f.quantize_token_blocks(torch.zeros(0, 200, dtype=torch.float16))
    assert not calls and q.shape == (0, 200) and s.shape == (0, 2)
    q, s = f.quantize_token_blocks(torch.zeros(0, 3, 200, dtype=torch.float16))
    assert not calls and q.shape == (0, 3, 200) and s.shape == (0, 3, 2)
    q, s = f.quantize_token_blocks(torch.zeros(7, 1, dtype=torch.float16))
    assert q.shape == (7, 1) and s.shape == (7, 1) and calls.pop()[1][2:4] == (7, 1)
    y = torch.zeros(5, 400, dtype=torch.float16)
    f.silu_mul_quant_blocks(y[:, :200], y[:, 200:])
    a = calls.pop()[1]
    assert a[1] == a[3] == 400 and a[2] - a[0] == 400 and a[5:7] == (5, 200)


def test_c_entries_refuse_rows_past_int_columns(L):
    """The kernels' column counters are 32-bit and go one step past the row."""
    keep, p = _buf()
    for cols in ((1 << 31) - 129, (1 << 31) - 1000, (1 << 31) - 8192):
        ld, kb = 1 << 31, 1 << 24
        rc = [L.lib.npl_fp8_quant_rows(p, 1, 1, cols, ld, p, ld, p, kb, None),
              L.lib.npl_fp8_quant_weight(p, 1, 1, cols, ld, p, ld, p, kb, None),
              L.lib.npl_fp8_rmsnorm_quant(p, ld, None, 0, p, 1, 1e-6, 1, cols, None, 0, p, ld, p, kb, None),
              L.lib.npl_fp8_silu_mul_quant(p, ld, p, ld, 1, 1, cols, p, ld, p, kb, None)]
        assert rc == [L.NPL_ERR_ARG] * 4, (cols, rc)


def test_outputs_that_are_an_input_by_another_name(F):
    """A view of the same rows is the input itself; an output that is one input
    must not overlap the other."""
    f, calls = F
    h = torch.float16
    flat, w, other = torch.zeros(4096, dtype=h), torch.ones(256, dtype=h), torch.zeros(4, 256, dtype=h)
    x, shifted = flat[:1024].view(4, 256), flat[256:1280].view(4, 256)
    for call in (lambda: f.rmsnorm_quant_blocks(x, w, 1e-6, shifted, sum_out=x),
                 lambda: f.rmsnorm_quant_blocks(shifted, w, 1e-6, x, sum_out=x),
                 lambda: f.rmsnorm_quant_blocks(other, flat[:256], 1e-6, shifted, sum_out=x)):
        with pytest.raises(ValueError):
            call()
    assert not calls
    f.rmsnorm_quant_blocks(x, w, 1e-6, other, sum_out=flat[:1024].view(4, 256))
    f.rmsnorm_quant_blocks(other, w, 1e-6, x, sum_out=flat[:1024].view(4, 256))
    f.rmsnorm_quant_blocks(x, w, 1e-6, x, sum_out=x)
    qa, qw = torch.zeros(4, 256).to(E4M3), torch.zeros(256, 256).to(E4M3)
    f.linear_blocks(qa, torch.ones(4, 2), qw, torch.ones(2, 2), residual=x, out=flat[:1024].view(4, 256))
    assert len(calls) == 4


def test_refusals_of_the_python_calls(F):
    f, calls = F
    h = torch.float16
    x, w = torch.zeros(4, 256, dtype=h), torch.ones(256, dtype=h)
    qa, sa = torch.zeros(4, 256).to(E4M3), torch.ones(4, 2)
    qw, sw = torch.zeros(100, 256).to(E4M3), torch.ones(1, 2)
    flat = torch.zeros(4096, dtype=h)
    bad = [
        lambda: f.quantize_token_blocks(torch.zeros(4, 0)),
        lambda: f.quantize_token_blocks(torch.zeros(4, 8, dtype=torch.int8)),
        lambda: f.quantize_token_blocks(torch.zeros(())),
        lambda: f.quantize_weight_blocks(torch.zeros(256)),
        lambda: f.quantize_weight_blocks(torch.zeros(0, 256)),
        lambda: f.rmsnorm_quant_blocks(x.float(), w, 1e-6),
        lambda: f.rmsnorm_quant_blocks(x, w[:128], 1e-6),
        lambda: f.rmsnorm_quant_blocks(x, w.bfloat16(), 1e-6),
        lambda: f.rmsnorm_quant_blocks(x, w, 1e-6, x[:3]),
        lambda: f.rmsnorm_quant_blocks(x, w, 1e-6, sum_out=x),
        lambda: f.rmsnorm_quant_blocks(x, w, 1e-6, x, sum_out=torch.zeros(256, 4, dtype=h).t()),
        # a sum that overlaps its inputs without being one of them
        lambda: f.rmsnorm_quant_blocks(flat[:1024].view(4, 256), w, 1e-6, x, sum_out=flat[8:1032].view(4, 256)),
        lambda: f.silu_mul_quant_blocks(x, x[:, :128]),
        lambda: f.silu_mul_quant_blocks(x.float(), x.float()),
        lambda: f.linear_blocks(qa.float(), sa, qw, sw),
        lambda: f.linear_blocks(qa, sa, qw[:, :128], sw),
        lambda: f.linear_blocks(qa, sa[:, :1], qw, sw),
        lambda: f.linear_blocks(qa, sa.double(), qw, sw),
        lambda: f.linear_blocks(qa, sa, qw, sw, out_dtype=torch.float32),
        lambda: f.linear_blocks(qa, sa, qw, sw, bias=torch.zeros(100, dtype=h)),
        lambda: f.linear_blocks(qa, sa, qw, sw, bias=torch.zeros(99)),
        lambda: f.linear_blocks(qa, sa, qw, sw, residual=torch.zeros(4, 99, dtype=h)),
        lambda: f.linear_blocks(qa, sa, qw, sw, residual=torch.zeros(4, 100, dtype=h), out_dtype=torch.bfloat16),
        lambda: f.linear_blocks(qa, sa, qw, sw, out=torch.zeros(100, 4, dtype=h).t()),
        lambda: f.linear_blocks(torch.zeros(4, 264).to(E4M3)[:, 8:], sa, qw, sw),       # rows off 16 bytes
        lambda: f.linear_blocks(torch.zeros(4, 260).to(E4M3)[:, :256], sa, qw, sw),     # stride off 16 bytes
        lambda: f.linear_blocks(qa, sa, qw, sw, residual=flat[:400].view(4, 100), out=flat[8:408].view(4, 100)),
        lambda: f.Fp8BlockLinear(qw, torch.ones(2, 2)),
        lambda: f.Fp8BlockLinear(qw.float(), sw),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert not calls
    # what is allowed: the residual in place, an output with a row stride, an odd K
    res = torch.zeros(4, 100, dtype=h)
    assert f.linear_blocks(qa, sa, qw, sw, residual=res, out=res) is res
    wide = torch.zeros(4, 128, dtype=torch.bfloat16)
    assert f.linear_blocks(qa, sa, qw, sw, out=wide[:, :100]).dtype == torch.bfloat16
    assert calls[-1][1][-2] == 128
    halves = torch.zeros(4, 200, dtype=h)  # two columns of one buffer's rows do not overlap
    assert f.linear_blocks(qa, sa, qw, sw, residual=halves[:, 100:], out=halves[:, :100]).shape == (4, 100)
    pair = torch.zeros(4, 512, dtype=h)
    assert f.rmsnorm_quant_blocks(pair[:, :256], w, 1e-6, x, sum_out=pair[:, 256:])[2].shape == (4, 256)
    odd = f._new_codes(1, 77, torch.device("cpu"))
    f.linear_blocks(odd, torch.ones(1, 1), f._new_codes(9, 77, torch.device("cpu")), torch.ones(1, 1))
    assert calls[-1][1][1] == 80 and calls[-1][1][5] == 80 and calls[-1][1][9:12] == (1, 9, 77)


def test_block_linear_lays_out_checkpoint_rows():
    from nanopointllm_b200 import fp8
    codes = torch.randn(10, 77).to(E4M3)
    lin = fp8.Fp8BlockLinear(codes, torch.ones(1, 1))
    assert lin.qweight.stride(0) == 80 and torch.equal(lin.qweight.float(), codes.float())
    assert (lin.in_features, lin.out_features) == (77, 10)



def test_torch_without_the_raw_queries(monkeypatch):
    """A torch build that lacks the private queries falls back to the public
    ones, also while the module is loaded."""
    import importlib.util
    import types
    from nanopointllm_b200 import fp8
    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda i: types.SimpleNamespace(cuda_stream=100 + i))
    spec = importlib.util.spec_from_file_location("nanopointllm_b200.fp8_without_raw", fp8.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    seen = []
    again._call(lambda *args: seen.append(args) or 0, torch.device("cuda", 3), 7)
    assert seen == [(7, 103)]



def test_a_single_row_by_another_stride_is_the_input_itself(F):
    """One row of a wide buffer, seen with the buffer's row stride or its own."""
    f, calls = F
    h = torch.float16
    wide, w, other = torch.zeros(3, 512, dtype=h), torch.ones(256, dtype=h), torch.zeros(1, 256, dtype=h)
    x, same = wide[:1, :256], wide[0, :256].unsqueeze(0)
    assert x.stride() != same.stride()
    assert f.rmsnorm_quant_blocks(x, w, 1e-6, other, sum_out=same)[2] is same
    assert f.rmsnorm_quant_blocks(other, w, 1e-6, same, sum_out=x)[2] is x
    qa, qw = torch.zeros(1, 256).to(E4M3), torch.zeros(256, 256).to(E4M3)
    assert f.linear_blocks(qa, torch.ones(1, 2), qw, torch.ones(2, 2), residual=x, out=same) is same
    column = torch.zeros(4, 8, dtype=h)[:, :1]
    f.linear_blocks(torch.zeros(4, 256).to(E4M3), torch.ones(4, 2), torch.zeros(1, 256).to(E4M3), torch.ones(1, 2),
                    residual=column.as_strided((4, 1), (8, 5)), out=column)
    assert len(calls) == 4
    with pytest.raises(ValueError):  # one element on, and two rows that only start alike
        f.rmsnorm_quant_blocks(x, w, 1e-6, other, sum_out=wide[0, 1:257].unsqueeze(0))
    flat = torch.zeros(1024, dtype=h)
    with pytest.raises(ValueError):
        f.rmsnorm_quant_blocks(flat[:512].view(2, 256), w, 1e-6, torch.zeros(2, 256, dtype=h),
                               sum_out=flat.as_strided((2, 256), (512, 1)))
    assert len(calls) == 4



def linear_path(m, n, k, sms=148, clusters_of_4=33):
    """Which tiles npl_fp8_linear takes on a B200: its host code's rules once
    more (launch, launch_prefill and decode_split of csrc/fp8_linear.cu)."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    kb, n_tiles, pairs, m_tiles = up(k, 128), up(n, 128), sms // 2, up(m, 256)

    def split(tiles):
        s = min(8, 7 * sms // (4 * tiles), kb // 2)
        return 1 if s <= 2 else s

    if m <= 64 or (m <= 128 and kb >= 20 and split(2 * n_tiles) >= 3):
        tokens = 16 if m <= 16 else 32 if m <= 32 else 64
        s = split(up(m, tokens) * n_tiles)
        return "decode", tokens, s, up(kb, s), 1
    wide, narrow = m_tiles * up(n, 256), m_tiles * up(n, 192)
    if 2 * wide <= pairs and kb >= 24 and wide <= clusters_of_4:
        return "prefill", 256, 2, up(kb, 2), 1
    rows, tiles = (192, narrow) if up(narrow, pairs) <= up(wide, pairs) else (256, wide)
    return "prefill", rows, 1, kb, up(tiles, pairs)


def test_cases_reach_the_paths_that_they_name():
    from test_fp8_gpu import LINEAR_PATHS
    for shape, path in LINEAR_PATHS.items():
        assert linear_path(*shape) == path, (shape, linear_path(*shape))
    # a 7B layer's own sizes go by paths that have a case above
    named = {path[:3] for path in LINEAR_PATHS.values()}
    for m, n, k in ((8, 12288, 4096), (8, 22016, 4096), (64, 32003, 4096), (560, 4096, 11008), (560, 12288, 4096),
                    (16000, 22016, 4096), (16000, 4096, 11008)):
        assert linear_path(m, n, k)[:3] in named, (m, n, k)


_EPILOGUE = r"""
// Threads as lanes or warps on the loops of fp8_epilogue.cuh; a meeting that one of them
// misses is seen after a second and ends the program.
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <mutex>
#include <thread>
#include <vector>
#include "fp8_epilogue.cuh"

struct Meeting {  // n threads; and of what they bring
  std::mutex m;
  std::condition_variable cv;
  int n, here = 0, turn = 0;
  bool all = true, result[2];
  explicit Meeting(int k) : n(k) {}
  void leave() {
    std::unique_lock<std::mutex> l(m);
    if (here == --n && n > 0) done();
  }
  void done() {
    result[turn & 1] = all, all = true, here = 0, ++turn;
    cv.notify_all();
  }
  bool meet(bool v, const char* what) {
    std::unique_lock<std::mutex> l(m);
    const int t = turn;
    all = all && v;
    if (++here == n) {
      done();
    } else if (!cv.wait_for(l, std::chrono::seconds(1), [&] { return turn != t; })) {
      std::printf("left alone in %s\n", what);
      std::fflush(stdout);
      std::_Exit(1);
    }
    return result[t & 1];
  }
};

void run(int n, const std::function<void(int)>& f) {
  std::vector<std::thread> ts;
  for (int i = 0; i < n; ++i) ts.emplace_back(f, i);
  for (auto& t : ts) t.join();
}

void expect(bool v, const char* what) {
  if (v) return;
  std::printf("%s\n", what);
  std::fflush(stdout);
  std::_Exit(1);
}

int main() {
  // one warp gives up at a unit, or none does (fail = -1)
  for (int fail : {-1, 0, 7, 8, 9, 35, 36}) {
    Meeting m(4);
    std::vector<int> units(4, 0), chunks(4, 0);
    run(4, [&](int w) {
      npl::decode_epilogue(3, 76, 32, 2, [&](int kc) { ++chunks[w], m.meet(true, "the scales"); },
                           [&](int i, int kc, int k, int kn) {
                             expect(i == units[w] && i == (kc - 3 + k) / 2 && kn == (kc == 67 ? 9 : 32), "wrong unit");
                             if (w == 2 && i == fail) return false;
                             ++units[w];
                             return true;
                           });
      expect(chunks[w] == 3 && units[w] == (w == 2 && fail >= 0 ? fail : 37), "wrong count");
    });
  }
  // one warp has no sums of a tile: none writes it or goes on
  for (int fail : {-1, 0, 2, 4}) {
    Meeting m(4);
    std::vector<int> wrote(4, 0);
    run(4, [&](int w) {
      npl::prefill_epilogue(5, 3, 19, [&](int t) { return !(w == 1 && t == 5 + 3 * fail); },
                            [&](bool ok) { return m.meet(ok, "the agreement"); },
                            [&](int t) {
                              expect(t == 5 + 3 * wrote[w], "wrong tile");
                              for (int box = 0; box < 4; ++box) m.meet(true, "the boxes");
                              ++wrote[w];
                            });
      expect(wrote[w] == (fail < 0 ? 5 : fail), "wrote a tile that a warp has no sums of");
    });
  }
  // One lane's deadline passes after three tries, all others' never. The phase is complete for lanes 6
  // and 7 in try arrival / 2, for the others one try later where the arrival is odd.
  for (int arrival : {0, 3, 5, 6, 7, 8, 9, 1000})
    for (bool voting : {false, true}) {
      Meeting vote(8), after(8);
      std::vector<int> got(8, -1);
      run(8, [&](int lane) {
        int tries = 0;
        auto try_once = [&] { return 2 * tries++ + (lane > 5) >= arrival; };
        auto late = [&] { return lane == 3; };
        got[lane] = voting ? npl::wait_voting(3, try_once, [&](bool x) { return vote.meet(x, "a vote"); }, late)
                           : npl::wait_as_one(3, try_once, [&](bool x) { return !vote.meet(!x, "the vote"); }, late);
        vote.leave();
        after.meet(true, "a warp-wide instruction");
      });
      for (int lane = 0; lane < 8; ++lane) expect(got[lane] == (arrival < (voting ? 5 : 8)), "lanes differ");
    }
  std::printf("ok\n");
}
"""


def test_epilogue_meets_in_full_when_a_wait_runs_out(tmp_path):
    """The epilogue's own loops, compiled for the host: whichever warp (or lane)
    gives up a wait, all of them meet as often as each other."""
    import pathlib
    import shutil
    import subprocess
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    src = tmp_path / "epilogue.cpp"
    src.write_text(_EPILOGUE)
    csrc = pathlib.Path(__file__).resolve().parent.parent / "nano-pointllm_b200" / "csrc"
    subprocess.run([cxx, "-std=c++17", "-O1", "-pthread", f"-I{csrc}", str(src), "-o", str(tmp_path / "epilogue")],
                   check=True)
    out = subprocess.run([str(tmp_path / "epilogue")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout == "ok\n", out.stdout
    # the kernels run these loops, and meet at a named barrier nowhere else
    kernel = (csrc / "fp8_linear.cu").read_text()
    for loop in ("wait_as_one(", "wait_voting(", "decode_epilogue(kb0", "prefill_epilogue(cluster"):
        assert kernel.count(loop) == 1, loop
    assert kernel.count("bar.sync") == 3 and kernel.count("barrier.cta") == 1
