"""Class / vocabulary operators (ser_amd.vocabulary) against plain 64-bit implementations (oracle/class_ops.py).

Tolerances come from the arithmetic, not from a run: a rounding to type t is off by at most eps(t)/2 of the value, an
f32 sum of n terms by n * 2^-24 of the sum of their magnitudes, the hardware's 2^x by one unit in the last place
(2^-23), and an exponent a = (x - m) / T * log2(e) that went through two f32 roundings moves 2^a by |a| * 2^-23 of
itself (ln 2 * 2 * 2^-24 < 2^-23).  Whole numbers are equal or wrong.
"""

import ctypes
import math
import subprocess
import threading
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import class_ops as plain

ROOT = Path(__file__).resolve().parent.parent
gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
LOWEST = {t: torch.finfo(t).min for t in TYPES}


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _scores(n, v, dtype, seed, spread=3.0):
    return (torch.randn((n, v), generator=_gen(seed)) * spread).to(dtype)


def _np(t):
    return t.detach().cpu().double().numpy()


# ------------------------------------------------------------------------------------------------ CPU
def _c_calls(lib):
    """(name, argument list that would be accepted, positions by name) of every entry point, with host memory in the
    place of device memory: the calls below are refused before anything is launched."""
    room = ctypes.create_string_buffer(4096)
    base = (ctypes.addressof(room) + 255) // 256 * 256
    ctx = base
    head = {"ctx": ctx, "logits": base, "dtype": 0, "n_rows": 4, "n_classes": 8, "stride": 8, "index": base, "i64": 1,
            "teacher": base, "t_dtype": 0, "k": 2, "T": 1.0}
    calls = {
        "serhip_sample": {"ctx": ctx, "logits": base, "dtype": 0, "n_rows": 4, "n_classes": 8, "stride": 8, "uniform": base,
                          "T": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "a": None, "b": None, "c": None, "d": None,
                          "token": base, "logprob": base, "stream": None},
        "serhip_distill_loss": {**head, "loss": base, "stats": base, "ws": base, "ws_bytes": 1 << 20, "stream": None},
        "serhip_distill_gradient": {**head, "stats": base, "weight": None, "grad": base + 64, "g_stride": 8, "stream": None},
        "serhip_distill_step": {**head, "weight": None, "loss": base, "grad": base + 64, "g_stride": 8, "ws": base,
                                "ws_bytes": 1 << 20, "stream": None},
        "serhip_embed": {"ctx": ctx, "tokens": base, "i64": 1, "n_tokens": 4, "table": base, "dtype": 0, "stride": 8,
                         "n_classes": 8, "width": 8, "scale": 1.0, "out": base, "o_stride": 8, "stream": None},
        "serhip_embed_gradient": {"ctx": ctx, "grad": base, "dtype": 1, "stride": 8, "tokens": base, "i64": 1, "n_tokens": 4,
                                  "n_classes": 8, "width": 8, "scale": 1.0, "acc": 0, "out": base, "o_dtype": 1,
                                  "o_stride": 8, "ws": base, "ws_bytes": 1 << 20, "stream": None},
    }
    return calls, room


REFUSALS = [
    ("serhip_sample", {"ctx": None}, "ctx"), ("serhip_sample", {"dtype": 3}, "element type"),
    ("serhip_sample", {"n_rows": -1}, "n_rows"), ("serhip_sample", {"n_classes": 0}, "n_classes"),
    ("serhip_sample", {"n_classes": (1 << 24) + 1}, "n_classes"), ("serhip_sample", {"stride": -8}, "stride"),
    ("serhip_sample", {"uniform": None}, "NULL"), ("serhip_sample", {"logits": None}, "NULL"),
    ("serhip_sample", {"token": None}, "NULL"), ("serhip_sample", {"n_rows": 1 << 31}, "too many"),
    ("serhip_sample", {"n_rows": 1 << 22, "n_classes": 65, "stride": 65}, "too many"),   # of 1 024 threads: 2^32
    ("serhip_embed", {"n_tokens": 1 << 31}, "too many"), ("serhip_embed_gradient", {"n_classes": (1 << 31) - 2}, "too many"),
    ("serhip_embed", {"ctx": None}, "ctx"), ("serhip_embed", {"dtype": -1}, "element type"),
    ("serhip_embed", {"n_tokens": -1}, "n_tokens"), ("serhip_embed", {"width": 0}, "width"),
    ("serhip_embed", {"o_stride": 7}, "stride"), ("serhip_embed", {"table": None}, "NULL"),
    ("serhip_embed", {"n_tokens": 1 << 41}, "too many"),
    ("serhip_embed_gradient", {"o_dtype": 2}, "f32"), ("serhip_embed_gradient", {"n_tokens": 1 << 31}, "MAX_TOKENS"),
    ("serhip_embed_gradient", {"ws_bytes": 8}, "too small"), ("serhip_embed_gradient", {"o_stride": 7}, "stride"),
    ("serhip_embed_gradient", {"out": None}, "NULL"), ("serhip_embed_gradient", {"tokens": None}, "NULL"),
    ("serhip_embed_gradient", {"n_classes": 1 << 31}, "n_classes"),
] + [(name, change, word) for name in ("serhip_distill_loss", "serhip_distill_gradient", "serhip_distill_step")
     for change, word in (({"ctx": None}, "ctx"), ({"t_dtype": 9}, "element type"), ({"k": 0}, "n_teacher"),
                          ({"k": 2049}, "2048"), ({"T": 0.0}, "temperature"), ({"T": float("nan")}, "temperature"),
                          ({"T": 1e4}, "temperature"), ({"n_rows": -1}, "n_rows"), ({"n_rows": 1 << 26}, "too many"),
                          ({"n_rows": 1 << 22, "n_classes": 65}, "too many"), ({"n_classes": 0}, "n_classes"),
                          ({"stride": -1}, "stride"), ({"index": None}, "NULL"), ({"logits": None}, "NULL"))] + [
    ("serhip_distill_loss", {"ws_bytes": 1}, "too small"), ("serhip_distill_loss", {"stats": None}, "NULL"),
    ("serhip_distill_step", {"ws_bytes": 1}, "too small"), ("serhip_distill_step", {"g_stride": 7}, "overlap"),
    ("serhip_distill_gradient", {"g_stride": 4}, "overlap"), ("serhip_distill_gradient", {"grad": None}, "NULL"),
]


@pytest.mark.parametrize("name,change,word", REFUSALS)
def test_entry_points_refuse(native_lib, name, change, word):
    from ser_amd import _native

    calls, room = _c_calls(native_lib)
    arguments = {**calls[name], **change}
    with pytest.raises(_native.SerhipError, match=word):
        _native.check(getattr(native_lib, name)(*arguments.values()))
    del room


def test_entry_points_refuse_misaligned_pointers(native_lib):
    from ser_amd import _native

    for name, key in (("serhip_sample", "logits"), ("serhip_distill_loss", "index"), ("serhip_distill_loss", "ws"),
                      ("serhip_distill_step", "grad"), ("serhip_embed", "table"), ("serhip_embed_gradient", "ws"),
                      ("serhip_embed_gradient", "tokens")):
        calls, room = _c_calls(native_lib)
        arguments = dict(calls[name])
        arguments[key] += 1
        with pytest.raises(_native.SerhipError, match="aligned"):
            _native.check(getattr(native_lib, name)(*arguments.values()))
    calls, room = _c_calls(native_lib)   # a gradient in place of the logits, but with other rows
    arguments = {**calls["serhip_distill_step"], "stride": 16, "g_stride": 8}
    arguments["grad"] = arguments["logits"]
    with pytest.raises(_native.SerhipError, match="in place"):
        _native.check(native_lib.serhip_distill_step(*arguments.values()))


@pytest.mark.parametrize("name", ["serhip_distill_loss", "serhip_distill_gradient", "serhip_distill_step"])
def test_more_threads_than_a_launch_has_are_refused(native_lib, name):
    """33 to 64 classes with a list that a wave has no room for: a workgroup of 256 for each row (a lane for each of up to 32
    classes, and a wave up to 256 entries, take as many rows again)."""
    from ser_amd import _native

    for v, k, rows in ((40, 300, 1 << 25), (64, 257, (1 << 24) + 1), (33, 2048, 1 << 24)):
        calls, room = _c_calls(native_lib)
        arguments = {**calls[name], "n_rows": rows, "n_classes": v, "stride": v, "k": k, "ws_bytes": 0}
        if "g_stride" in arguments:
            arguments["g_stride"] = v
        with pytest.raises(_native.SerhipError, match="too many"):
            _native.check(getattr(native_lib, name)(*arguments.values()))
        # what is refused next (nothing is launched): fewer rows are no longer "too many"
        arguments.update(n_rows=1 << 23, **({"ws": None} if "ws" in arguments else {"stats": None}))
        with pytest.raises(_native.SerhipError, match="NULL"):
            _native.check(getattr(native_lib, name)(*arguments.values()))
        del room


def test_empty_calls_touch_nothing(native_lib):
    calls, room = _c_calls(native_lib)
    for name, key in (("serhip_sample", "n_rows"), ("serhip_distill_loss", "n_rows"), ("serhip_distill_gradient", "n_rows"),
                      ("serhip_distill_step", "n_rows"), ("serhip_embed", "n_tokens")):
        assert getattr(native_lib, name)(*{**calls[name], key: 0}.values()) == 0, name


def test_workspace_sizes(native_lib):
    assert native_lib.serhip_distill_workspace(0, 8, 0) >= 0
    assert native_lib.serhip_distill_workspace(1000, 50001, 1) >= 2 * 8 * 1000
    assert native_lib.serhip_distill_workspace(-1, 8, 0) < 0 and native_lib.serhip_distill_workspace(1, 8, 5) < 0
    few, many = (native_lib.serhip_embed_gradient_workspace(n, 50001, 1024) for n in (1, 100000))
    assert 0 < few < many and many >= 16 * 100000
    assert native_lib.serhip_embed_gradient_workspace(-1, 8, 8) < 0
    assert native_lib.serhip_embed_gradient_workspace((1 << 31) - 1, 8, 8) < 0


def test_python_refusals():
    """Everything that is checked before the tensors' device: the same message with and without a GPU."""
    import ser_amd

    x, u = torch.zeros(3, 8), torch.zeros(3)
    idx, top = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    for call, word in (
        (lambda: ser_amd.sample_tokens([1.0], u), "torch tensor"),
        (lambda: ser_amd.sample_tokens(x.double(), u), "dtype"),
        (lambda: ser_amd.sample_tokens(x, u.double()), "dtype"),
        (lambda: ser_amd.sample_tokens(x, torch.zeros(4)), "shape"),
        (lambda: ser_amd.sample_tokens(x[:, :0], u), "classes"),
        (lambda: ser_amd.sample_tokens(x, u, temperature=-1.0), "temperature"),
        (lambda: ser_amd.sample_tokens(x, u, temperature=math.nan), "temperature"),
        (lambda: ser_amd.sample_tokens(x, u, temperature=math.inf), "temperature"),
        (lambda: ser_amd.sample_tokens(x, u, top_k=-1), "top_k"),
        (lambda: ser_amd.sample_tokens(x, u, top_k=1.5), "top_k"),
        (lambda: ser_amd.sample_tokens(x, u, top_k=torch.zeros(3)), "whole"),
        (lambda: ser_amd.sample_tokens(x, u, top_k=torch.zeros(2, dtype=torch.int32)), "shape"),
        (lambda: ser_amd.sample_tokens(x, u, top_p=1.5), "top_p"),
        (lambda: ser_amd.sample_tokens(x, u, top_p=torch.zeros(3, dtype=torch.int32)), "floating"),
        (lambda: ser_amd.sample_tokens(x, u, min_p=-0.1), "min_p"),
        (lambda: ser_amd.sample_tokens(x, u), "on the GPU"),
        (lambda: ser_amd.distillation_loss(x, idx, top[:, :1]), "teacher_logits"),
        (lambda: ser_amd.distillation_loss(x, idx[:2], top), "teacher_index"),
        (lambda: ser_amd.distillation_loss(x, idx.float(), top), "dtype"),
        (lambda: ser_amd.distillation_loss(x, idx[:, :0], top[:, :0]), "teacher_index"),
        (lambda: ser_amd.distillation_loss(x, idx.expand(3, 2).repeat(1, 1025), top.repeat(1, 1025)), "2048"),
        (lambda: ser_amd.distillation_loss(x, idx, top, temperature=0.0), "temperature"),
        (lambda: ser_amd.distillation_loss(x, idx, top.clone().requires_grad_()), "teacher"),
        (lambda: ser_amd.distillation_loss(x.clone().requires_grad_(), idx, top, temperature=-1.0), "temperature"),
        (lambda: ser_amd.distillation_loss(x, idx, top), "on the GPU"),
        (lambda: ser_amd.distillation_step(x, idx, top), "on the GPU"),
        (lambda: ser_amd.embed_tokens(idx, x[0]), "table"),
        (lambda: ser_amd.embed_tokens(idx.to(torch.int16), x), "dtype"),
        (lambda: ser_amd.embed_tokens(idx, x.clone().requires_grad_(), out=torch.zeros(3, 2, 8)), "gradient"),
        (lambda: ser_amd.embed_tokens(idx, x, out=torch.zeros(3, 8)), "shape"),
        (lambda: ser_amd.embed_tokens(idx, x), "on the GPU"),
        (lambda: ser_amd.embedding_gradient(x, idx, 4), "grad"),
        (lambda: ser_amd.embedding_gradient(x, idx[:, 0], 0), "classes"),
        (lambda: ser_amd.embedding_gradient(x, idx[:, 0], 4, accumulate=True), "out="),
        (lambda: ser_amd.embedding_gradient(x, idx[:, 0], 4, dtype=torch.bfloat16), "float32"),
        (lambda: ser_amd.embedding_gradient(x, idx[:, 0], 4, out=torch.zeros(5, 8)), "shape"),
        (lambda: ser_amd.embedding_gradient(x, idx[:, 0], 4, out=torch.zeros(8, 4).t()), "contiguous"),
        (lambda: ser_amd.embedding_gradient(x, idx[:, 0], 4), "on the GPU"),
    ):
        with pytest.raises(ValueError, match=word):
            call()


@pytest.fixture
def no_launch(monkeypatch, native_lib):
    """The Python side of the calls on CPU tensors, with nothing behind it: results are what their memory happens to hold."""
    from types import SimpleNamespace

    from ser_amd import vocabulary

    monkeypatch.setattr(vocabulary, "_engine_of", lambda t, name: SimpleNamespace(_lib=native_lib))
    monkeypatch.setattr(vocabulary, "_call", lambda engine, function, *args: None)
    return vocabulary


def test_out_raises_its_version(no_launch):
    """What a call wrote through a pointer is known to autograd: a saved tensor that was written to is an error in backward."""
    x, idx, top = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    base = torch.zeros(3, 9)
    for out in (torch.zeros(3, 8), x, base[:, :8]):
        before = out._version
        no_launch.distillation_step(x, idx, top, out=out)
        assert out._version > before
    assert base._version > 0
    out = torch.zeros(3, 2, 8)
    no_launch.embed_tokens(idx, x, out=out)
    assert out._version == 1
    out = torch.zeros(4, 8)
    no_launch.embedding_gradient(x, idx[:, 0], 4, out=out)
    no_launch.embedding_gradient(x, idx[:, 0], 4, out=out, accumulate=True)
    assert out._version == 2
    with torch.inference_mode():
        out = torch.zeros(3, 8)
        no_launch.distillation_step(x, idx, top, out=out)
    leaf = torch.zeros(3, 8, requires_grad=True)
    logits = leaf * 2
    loss = no_launch.distillation_loss(logits, idx, top)
    no_launch.distillation_step(logits.detach(), idx, top, out=logits.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


def test_out_must_not_require_a_gradient(no_launch):
    """As torch's own out=: refused while gradients are enabled, whatever the operator does inside."""
    x, idx, top = torch.zeros(3, 8), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    leaf = torch.zeros(3, 8, requires_grad=True)
    for out in (leaf, leaf * 2):
        for call in (lambda: no_launch.distillation_step(x, idx, top, out=out), lambda: no_launch.distillation_step(out, idx, top, out=out),
                     lambda: no_launch.embed_tokens(idx[:, 0], x, out=out), lambda: no_launch.embedding_gradient(x, idx[:, 0], 3, out=out)):
            with pytest.raises(ValueError, match="must not require a gradient"):
                call()
            with torch.no_grad():
                call()
        no_launch.distillation_step(out.detach(), idx, top, out=out.detach())


def test_a_teacher_that_requires_a_gradient_is_refused(no_launch):
    """Also, and above all, where the student is trained: no gradient would reach the teacher."""
    idx, top = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2, requires_grad=True)
    for student in (torch.zeros(3, 8), torch.zeros(3, 8, requires_grad=True), torch.zeros(3, 8, requires_grad=True) * 2):
        with pytest.raises(ValueError, match="teacher"):
            no_launch.distillation_loss(student, idx, top)
        no_launch.distillation_loss(student, idx, top.detach())
        with torch.no_grad():
            no_launch.distillation_loss(student, idx, top)


def test_what_backward_needs_is_kept_by_autograd_alone(no_launch):
    """Scores and teacher are freed after a backward pass though the loss lives on, and go through saved-tensor hooks."""
    import gc
    import weakref

    def step(strided):
        leaf = torch.zeros(4, 6, 8, requires_grad=True)
        logits = (leaf * 2).transpose(0, 1) if strided else leaf * 2
        index, top = torch.zeros(*logits.shape[:-1], 2, dtype=torch.int64), torch.zeros(*logits.shape[:-1], 2)
        return [weakref.ref(t) for t in (logits, index, top)], no_launch.distillation_loss(logits, index, top)

    for strided in (False, True):
        held, loss = step(strided)
        loss.sum().backward()
        gc.collect()
        assert all(t() is None for t in held)

        packed = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(tuple(t.shape)) or len(packed) - 1,
                                                      lambda i: torch.zeros(packed[i], dtype=torch.int64 if i % 4 == 1 else torch.float32)):
            held, loss = step(strided)
            gc.collect()
        # nothing but the hooks holds them now
        assert len(packed) >= 4 and all(t() is None for t in held)
        loss.sum().backward()


def test_tangents_are_refused(no_launch):
    """Forward-mode derivatives: an error, where the tangent was dropped without a word."""
    from torch.autograd import forward_ad

    idx, top = torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(3, 8), torch.ones(3, 8))
        dual_top = forward_ad.make_dual(top, torch.ones(3, 2))
        for call in (lambda: no_launch.distillation_loss(dual, idx, top), lambda: no_launch.distillation_loss(torch.zeros(3, 8), idx, dual_top),
                     lambda: no_launch.embed_tokens(idx, dual)):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        no_launch.distillation_loss(torch.zeros(3, 8), idx, top)


def test_out_may_lie_beside_the_inputs(no_launch):
    """One buffer may hold both, where they do not overlap; where they do, other storages do not hide it."""
    n, v = 3, 8
    idx, top = torch.zeros(n, 2, dtype=torch.int64), torch.zeros(n, 2)
    flat = torch.zeros(2 * n * v)
    x, out = flat[: n * v].view(n, v), flat[n * v :].view(n, v)
    wide = torch.zeros(n, 3 * v)
    for a, b in ((x, out), (out, x), (wide[:, :v], wide[:, v : 2 * v]), (wide[:, 2 * v :], wide[:, :v])):
        no_launch.distillation_step(a, idx, top, out=b)
        no_launch.embed_tokens(idx[:, 0], a, out=b)
        no_launch.embedding_gradient(a, idx[:, 0], n, out=b)
    alias = torch.from_dlpack(flat.numpy()[v : v + n * v].reshape(n, v))   # the same bytes under another storage
    for a, b in ((x, flat[v : v + n * v].view(n, v)), (x, alias), (wide[:, :v], wide[:, 1 : 1 + v]), (wide[:, 2 * v :], wide.view(-1)[-n * v :].view(n, v)),
                 (wide[:, 1 : 1 + v], wide[:, :v])):
        for call in (lambda: no_launch.distillation_step(a, idx, top, out=b), lambda: no_launch.embed_tokens(idx[:, 0], a, out=b),
                     lambda: no_launch.embedding_gradient(a, idx[:, 0], n, out=b)):
            with pytest.raises(ValueError, match="overlap|share memory"):
                call()
    # every byte of every pair of row blocks of one matrix, against their elements
    whole = torch.arange(60)
    for pitch in (5, 7):
        for r0, c0, r1, c1, w0, w1 in ((a, b, c, d, e, f) for a in range(2) for b in range(4) for c in range(3) for d in range(4) for e in (1, 2) for f in (1, 3)):
            p = whole.as_strided((3, w0), (pitch, 1), r0 * pitch + c0)
            q = whole.as_strided((2, w1), (pitch, 1), r1 * pitch + c1)
            if c0 + w0 <= pitch and c1 + w1 <= pitch:
                rows_apart = r1 >= r0 + 3 or r0 >= r1 + 2
                want = bool(set(p.flatten().tolist()) & set(q.flatten().tolist()))
                got = no_launch._share_memory(p, q)
                assert got == want or (got and rows_apart)


def test_temperatures_too_small_for_float32(no_launch, monkeypatch):
    """A positive temperature that float32 rounds to 0 is not the greedy one: it does as 1e-30."""
    x, u = torch.zeros(3, 8), torch.zeros(3)
    calls = []
    monkeypatch.setattr(no_launch, "_call", lambda engine, function, *args: calls.append(args))
    for temperature, want in ((1e-50, 1e-30), (1e-31, 1e-30), (0.0, 0.0), (1e-30, 1e-30), (0.5, 0.5)):
        no_launch.sample_tokens(x, u, temperature=temperature)
        assert ctypes.c_float(calls[-1][6]).value == np.float32(want)
    rows = torch.tensor([1e-50, 0.0, -1e-50], dtype=torch.float64)
    got = no_launch._per_row(rows, "temperature", (3,), x.device)
    assert got.dtype == torch.float32 and got[0] == np.float32(1e-30) and got[1] == 0 and not got[2] > 0


@pytest.mark.parametrize("top_k", [math.inf, -math.inf, math.nan, 0.5])
def test_top_k_that_is_no_whole_number(top_k):
    import ser_amd

    with pytest.raises(ValueError, match="top_k must be a whole number"):
        ser_amd.sample_tokens(torch.zeros(3, 8), torch.zeros(3), top_k=top_k)


def test_oracle_gradient_is_the_derivative():
    """The distillation gradient's formula against central differences of the loss's formula: with step h the
    difference is off by h^2/6 times a third derivative (below 4 T^-1 for softmax terms) plus 2^-53 |L| / h."""
    rng = np.random.default_rng(3)
    for temperature in (0.7, 1.0, 3.0):
        x = rng.standard_normal(9) * 2
        index, teacher = np.asarray([4, 0, 4, -1, 8]), rng.standard_normal(5)
        loss, g = plain.distill_row(x, index, teacher, temperature)
        h = 1e-5
        for j in range(9):
            d = np.zeros(9)
            d[j] = h
            slope = (plain.distill_row(x + d, index, teacher, temperature)[0]
                     - plain.distill_row(x - d, index, teacher, temperature)[0]) / (2 * h)
            assert abs(slope - g[j]) < 1e-9 * max(1.0, abs(loss))
        assert abs(g.sum()) < 1e-12   # q and p both sum to one


def _weights_program(tmp_path):
    """csrc/row_weights.hpp compiled for the host: lines of (top, T, x) in, the weight of x out."""
    clang = Path("/opt/rocm/lib/llvm/bin/clang++")
    if not clang.exists():
        pytest.skip("amdclang++ not available")
    src, exe = tmp_path / "weights.cpp", tmp_path / "weights"
    src.write_text(r'''
#include "row_weights.hpp"
#include <cstdio>
using namespace serhip;
static constexpr PowerTable table;
int main() {
  float top, t, x;
  while (scanf("%g %g %g", &top, &t, &x) == 3)
    printf("%.17g\n", row_weights(top, t, 45).real(x, [](int j) { return table.v[j]; }));
  return 0;
}''')
    subprocess.run([str(clang), "-std=c++17", "-O2", "-ffp-contract=on", "-I", str(ROOT / "ser_amd" / "csrc"), "-o", str(exe), str(src)],
                   check=True)

    def weights(top, t, x):
        lines = "".join(f"{float(np.float32(top))!r} {float(np.float32(t))!r} {float(v)!r}\n" for v in x)
        out = subprocess.run([str(exe)], input=lines, check=True, capture_output=True, text=True).stdout.split()
        return np.asarray(out, dtype=np.float64)

    return weights


def test_weights_of_every_temperature(tmp_path):
    """The weight of every score, from the largest down to the lowest number, at every temperature that is accepted: never
    above 1, never negative, in the order of the scores, and exp((x - top) / T) to the 2^-45 of itself that a series to the third
    power leaves (f^4 / 24 of (ln 2 / 1024)^4) with the roundings of an exponent of up to 2^10 -- or, where that is below 2^-200,
    anything below 2^-190, which no sum notices."""
    weights = _weights_program(tmp_path)
    big = np.finfo(np.float32).max
    for top in (0.0, 1e-30, 1e-3, 1.0, 10.0, 30.0, 6e4, 1e10, 1e11, 1e38, float(big), -1e-3, -7.25, -1e10, -float(big)):
        for t in (1e-30, 1e-12, 1e-10, 1e-9, 1e-8, 1e-7, 1e-6, 1e-5, 1e-4, 1e-2, 0.7, 1.0, 30.0, 1e10, 3e38):
            x = [np.float32(top)]
            for _ in range(6):   # the next numbers below
                if x[-1] > -big:
                    x.append(np.nextafter(x[-1], np.float32(-np.inf)))
            with np.errstate(over="ignore"):
                x += [np.float32(top - d) for d in (t, 50 * t, 500 * t, 1000 * t, 1e-6, 1e-3, 0.5, 5.0, 7000.0, 1e5, 1e9, 1e30, 3e38)]
            x = np.unique(np.asarray([v for v in x if np.isfinite(v)], np.float32))[::-1]
            got = weights(top, t, x)
            far = (x.astype(np.float64) - float(np.float32(top))) / float(np.float32(t))
            with np.errstate(under="ignore"):
                want = np.exp(far)
            assert got[0] == 1.0 and (got >= 0).all() and (got <= 1).all() and (np.diff(got) <= 0).all(), (top, t)
            tiny = want < 2.0**-200
            assert (got[tiny] < 2.0**-190).all(), (top, t)
            # far is rounded twice more on the way, and is below 2^8 here: 2^-44 of the weight with it
            assert (np.abs(got - want)[~tiny] <= want[~tiny] * 2.0**-44).all(), (top, t, got, want)


# ------------------------------------------------------------------------------------------- sampling
def _check_sample(logits, uniform, device_logits=None, **settings):
    """The kernels' tokens and log-probabilities against the oracle, row by row."""
    import ser_amd

    x = logits.cuda() if device_logits is None else device_logits
    on_gpu = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in settings.items()}
    token, logprob = ser_amd.sample_tokens(x, uniform.cuda(), **on_gpu)
    assert token.dtype == torch.int64 and logprob.dtype == torch.float32
    rows, u = _np(logits).reshape(-1, logits.shape[-1]), _np(uniform).reshape(-1)
    got_t, got_l = token.cpu().reshape(-1).numpy(), _np(logprob).reshape(-1)
    for r in range(len(rows)):
        one = {k: (_np(v).reshape(-1)[r] if isinstance(v, torch.Tensor) else float(np.float32(v))) for k, v in settings.items()}
        want_t, want_l = plain.sample_row(rows[r], u[r], **one)
        if got_t[r] != want_t:
            # a goal on the border of two classes, as u = 1/2 has it for classes in groups of equal scores, has two answers:
            # the oracle adds up n weights one after another, off by n 2^-53 of the sum; the kernel's weights are off by 2^-44,
            # and rounded to units of 2^-45 of the largest, up or down (allowed for with 2^-44 in all)
            off = len(rows[r]) * 2.0**-53 + 2.0**-43
            sides = [plain.sample_row(rows[r], u[r] * (1 + d), **one) for d in (-off, off)]
            assert got_t[r] in [t for t, _ in sides], (r, got_t[r], want_t, one)
            want_l = dict(sides)[got_t[r]]
        if np.isinf(want_l):
            assert got_l[r] == want_l
        else:
            # log of a sum of f32 terms: at most V/64 terms one after another, each off by two units; the answer's rounding
            v = rows.shape[1]
            assert abs(got_l[r] - want_l) <= (v / 64 + 64) * 2.0**-23 + abs(want_l) * 2.0**-23, r
    return token


SETTINGS = [
    {}, {"temperature": 0.0}, {"temperature": 0.7, "top_k": 50, "top_p": 0.95}, {"top_k": 1}, {"top_k": 3, "min_p": 0.3},
    {"temperature": 1.3, "top_p": 0.9}, {"top_p": 0.0}, {"top_p": 1e-6}, {"min_p": 0.05}, {"min_p": 1.0}, {"temperature": 2.5, "min_p": 1e-4},
    {"top_k": 10**9, "top_p": 0.5}, {"top_k": 700, "top_p": 0.999, "min_p": 1e-5, "temperature": 4.0},
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [1, 2, 8, 63, 257, 1025, 4099, 20011])
@pytest.mark.parametrize("at", range(len(SETTINGS)))
def test_sampling_matches_the_definition(dtype, v, at):
    n = 5 if v < 20000 else 3
    u = torch.rand((n,), generator=_gen(1000 + v + at))
    _check_sample(_scores(n, v, dtype, 7 * v + at), u, **SETTINGS[at])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [8, 63, 257, 5003, 20011])
@pytest.mark.parametrize("temperature", [1e-30, 1e-12, 1e-9, 1e-8, 1e-6, 1e-4, 1.0])
def test_sampling_small_temperatures_and_large_scores(dtype, v, temperature):
    """Where an octave of the weight is about as far as the next number below the largest score, or far below it: what is left
    are the classes at the largest score, and at T = 1e-4 those next to it."""
    rows = []
    for top in (10.0, 30.0, 6e4, 1e10, -7.25):
        if top > torch.finfo(dtype).max:
            continue
        row = top - 0.001 - 5.0 * torch.rand((v,), generator=_gen(v)).abs()
        row = row.to(dtype)
        best = row.max().clone()
        row[v // 2], row[v - 2] = best, torch.tensor(top, dtype=dtype)   # (no other is larger)
        rows += [row, torch.where(torch.arange(v) % 3 == 1, torch.tensor(top, dtype=dtype), row)]
    x = torch.stack(rows)
    n = x.shape[0]
    for u in (0.03, 0.5013, 0.99999):
        uniform = torch.full((n,), u)
        for settings in ({}, {"top_k": 5}, {"top_p": 0.6}, {"min_p": 0.05}, {"top_k": 40, "top_p": 0.9, "min_p": 0.01}):
            _check_sample(x, uniform, temperature=temperature, **settings)
        _check_sample(x, uniform, temperature=torch.full((n,), temperature), top_p=torch.linspace(0.1, 1.0, n))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [63, 257, 5003, 20011, 70001])
def test_sampling_a_uniform_number_of_zero(dtype, v):
    """u = 0 takes the first class that has any weight, not the first class: here all but the largest are e^-1000 of it, or less."""
    row = (10.0 - 0.0625 - 5.0 * torch.rand((v,), generator=_gen(v))).to(dtype)
    row[v // 2] = row[v - 2] = 10.0
    x = torch.stack([row, torch.where(torch.arange(v) < v - 5, -math.inf, row.float()).to(dtype)])
    for temperature in (1e-30, 1e-9, 1e-5):
        for settings in ({}, {"top_k": v - 1}, {"top_p": 0.999}, {"min_p": 1e-30}):
            _check_sample(x, torch.zeros((2,)), temperature=temperature, **settings)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [40, 5003, 20011, 70001])
def test_sampling_large_temperatures(dtype, v, monkeypatch):
    """Scores further apart than the largest f32, at temperatures where that is a moderate weight.  (The log-probability is
    untempered: below -3.4028236e38 it rounds to -inf in f32.)"""
    exact = plain.sample_row

    def rounded(*arguments, **settings):
        token, logprob = exact(*arguments, **settings)
        with np.errstate(over="ignore"):
            return token, -math.inf if np.float32(logprob) == -np.inf else logprob

    monkeypatch.setattr(plain, "sample_row", rounded)
    x = (3.3e38 * (2.0 * torch.rand((3, v), generator=_gen(v)) - 1.0)).to(dtype)
    x[1, : v // 2] = LOWEST[dtype]
    x[1, v - 1] = torch.finfo(dtype).max
    for temperature in (1e37, 1e38, 3e38):
        for settings in ({}, {"top_p": 0.5}, {"top_p": 0.97}, {"min_p": 0.2}, {"top_k": 2000, "top_p": 0.7}):
            _check_sample(x, torch.tensor([0.2, 0.61, 0.97]), temperature=temperature, **settings)


@gpu
@pytest.mark.parametrize("v", [40, 300, 20011])
def test_sampling_uniform_numbers_out_of_range(v):
    """1 and more draw the last class that is kept, what is below 0, or NaN, the first."""
    x = _scores(6, v, torch.float32, v, spread=1.0)
    u = torch.tensor([1.0, 2.5, math.inf, -0.5, -math.inf, math.nan])
    for settings in ({}, {"top_k": 7}, {"top_p": 0.8}, {"min_p": 0.3}):
        _check_sample(x, u, **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [300, 5003, 20011, 70001])
def test_sampling_among_infinite_scores(dtype, v):
    """More classes at +inf than are kept, in rows whose cut is found from candidates, and in rows where it is not."""
    x = _scores(3, v, dtype, v)
    x[0, :] = math.inf
    x[1, v // 3 :] = math.inf
    x[2, ::2] = math.inf
    x[2, 1::4] = math.nan
    for u in (0.0, 0.2849, 0.999):
        for settings in ({}, {"top_k": 257, "temperature": 1e-6}, {"top_k": 257, "min_p": 0.3}, {"top_p": 0.3}, {"top_p": 0.3, "min_p": 0.1, "temperature": 2.0},
                         {"top_k": v - 2, "top_p": 0.4}, {"min_p": 1.0}):
            _check_sample(x, torch.full((3,), u), **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [65536, 131072, 100003])
def test_sampling_large_vocabularies(dtype, v):
    u = torch.rand((2,), generator=_gen(v))
    for settings in ({}, {"top_k": 40, "temperature": 0.8}, {"top_p": 0.8}, {"min_p": 0.02, "top_p": 0.95}, {"top_k": 5000, "top_p": 0.9}):
        _check_sample(_scores(2, v, dtype, v + 1), u, **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [16383, 16384, 16385, 40009, 70001])
def test_sampling_wide_nuclei(dtype, v):
    """Cuts that keep hundreds to tens of thousands of classes, on both sides of what fits a workgroup's memory: peaked rows,
    flat ones, rows whose classes fall into 13 or 700 groups of equal scores."""
    at = torch.arange(v)
    rows = torch.stack([_scores(1, v, torch.float32, v + 2, spread=1.2)[0], _scores(1, v, torch.float32, v + 3, spread=0.05)[0],
                        (at * 7919 % 13).float() / 4, (at * 104729 % 700).float() / 256, at.float() / v]).to(dtype)
    u = torch.tensor([0.31, 0.77, 0.5, 0.08, 0.99999])
    for settings in ({"top_p": 0.6}, {"top_p": 0.95}, {"top_p": 0.9, "temperature": 2.0}, {"top_p": 0.9999, "temperature": 0.8},
                     {"top_p": 0.7, "min_p": 1e-3}, {"top_p": 0.97, "min_p": 0.2}, {"min_p": 1e-6, "temperature": 1.5},
                     {"top_k": 1024, "top_p": 0.5}, {"top_k": 1025}, {"top_k": 15000, "top_p": 0.9}, {"top_k": 16390, "min_p": 0.1}):
        _check_sample(rows, u, **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,settings", [(5888, {"top_p": 0.97, "temperature": 1.4}), (5889, {"top_p": 0.97, "temperature": 1.4}),
                                        (20011, {}), (20011, {"top_k": 40, "top_p": 0.9}), (20011, {"top_p": 0.9, "temperature": 2.0}),
                                        (20011, {"top_p": 0.95, "temperature": 0.4}), (20011, {"min_p": 0.001, "top_p": 0.99}),
                                        (20011, {"top_k": 600}), (70001, {"top_k": 9}), (70001, {"min_p": 0.01})])
def test_sampling_more_rows_than_compute_units(dtype, v, settings):
    u = torch.rand((260,), generator=_gen(v))
    rows = _scores(4, v, dtype, v + 9).repeat(65, 1)   # (the oracle's time)
    _check_sample(rows, u, **settings)


@gpu
@pytest.mark.parametrize("v", [131073, 300007, 4194305])
def test_sampling_past_131072_classes(v):
    """Ranges of classes that one step of the draw does not narrow to a wave's width."""
    rows = _scores(2, v, torch.bfloat16, v + 1)
    rows[0, v - 40 :] = rows[0].max()   # the last range is shorter than a wave
    u = torch.tensor([0.9, 0.4])
    for settings in ({}, {"top_k": 100}, {"min_p": 0.003}, {"top_p": 0.5}, {"top_k": 900, "top_p": 0.9}):
        _check_sample(rows, u, **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("settings", [{}, {"top_k": 37}, {"top_p": 0.4}, {"top_k": 900, "top_p": 0.5}, {"min_p": 0.5},
                                      {"top_k": 5, "top_p": 0.7, "temperature": 0.3}, {"temperature": 0.0}])
def test_sampling_ties_go_to_the_lowest_index(dtype, settings):
    """Rows of one value, of two, and of a few: the cut falls inside a group of equal scores."""
    v = 3001
    rows = torch.stack([torch.full((v,), -1.5), (torch.arange(v) % 2).float(), (torch.arange(v) * 7919 % 13).float() / 4,
                        torch.where(torch.arange(v) % 5 == 0, 0.0, -0.0)]).to(dtype)
    for u in (0.0, 0.25, 0.5, 0.9999):
        _check_sample(rows, torch.full((4,), u), **settings)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_sampling_masked_rows(dtype):
    """Masked classes at -inf, NaN and the type's lowest value; +inf; rows with nothing left; a row with one class."""
    v = 2500
    x = _scores(9, v, dtype, 5)
    x[0, :] = -math.inf
    x[1, :] = math.nan
    x[2, ::2] = -math.inf
    x[2, 1::4] = math.nan
    x[3, 100:] = LOWEST[dtype]
    x[4, :] = LOWEST[dtype]
    x[5, 17] = math.inf
    x[6, 17:30] = math.inf
    x[7, :] = -math.inf
    x[7, 2499] = -3.0
    x[8, :-1] = math.nan
    for settings in SETTINGS:
        for u in (0.0, 0.3, 0.99999994):
            _check_sample(x, torch.full((9,), u), **settings)


@gpu
def test_sampling_settings_per_row():
    n, v = 24, 5003
    at = torch.arange(n)
    x, u = _scores(n, v, torch.bfloat16, 11), torch.rand((n,), generator=_gen(12))
    temperature = (0.25 + 0.2 * (at % 6)).float()
    temperature[3], temperature[4], temperature[5], temperature[6] = 0.0, -1.0, math.nan, math.inf
    top_k = ((at * 5) % 60).to(torch.int32)
    top_k[7], top_k[8] = -4, 2**31 - 1
    top_p = (0.1 + 0.035 * at).float()
    top_p[9], top_p[10], top_p[11], top_p[12] = 0.0, -1.0, math.nan, 7.0
    min_p = (0.01 * (at % 4)).float()
    min_p[13], min_p[14], min_p[15] = math.nan, -2.0, 9.0
    a = _check_sample(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    b = _check_sample(x.view(4, 6, v), u.view(4, 6), temperature=temperature.view(4, 6), top_k=top_k.view(4, 6).long(),
                      top_p=top_p.view(4, 6), min_p=min_p.view(4, 6))
    assert torch.equal(a, b.view(-1))


@gpu
def test_sampling_follows_the_distribution():
    """A grid of uniform numbers over one row gives each class its share, to a step of the grid."""
    import ser_amd

    v, n = 40, 8000
    row = _scores(1, v, torch.float32, 3, spread=1.0)
    u = (torch.arange(n).double() + 0.5).div(n).float()
    for settings, temperature in (({}, 1.0), ({"temperature": 0.5}, 0.5)):
        token, _ = ser_amd.sample_tokens(row.cuda().expand(n, v), u.cuda(), **settings)
        share = np.bincount(token.cpu().numpy(), minlength=v) / n
        w = np.exp((_np(row)[0] - _np(row).max()) / temperature)
        assert np.abs(share - w / w.sum()).max() <= 1.0 / n + 1e-6
        assert (np.diff(token.cpu().numpy()) >= 0).all()   # index order is the order of the draw


@gpu
def test_sampling_layouts_and_streams():
    import ser_amd

    v = 1031
    u = torch.rand((6,), generator=_gen(2))
    whole = _scores(6 * 5, v, torch.float16, 1).view(6, 5, v)
    want = _check_sample(whole[:, -1].contiguous(), u, top_k=20)
    assert torch.equal(want, _check_sample(whole[:, -1].contiguous(), u, device_logits=whole.cuda()[:, -1], top_k=20))
    wide = torch.zeros((6, v + 9), dtype=torch.float16)
    wide[:, 3 : 3 + v] = whole[:, -1]
    assert torch.equal(want, _check_sample(whole[:, -1].contiguous(), u, device_logits=wide.cuda()[:, 3 : 3 + v], top_k=20))
    columns = whole[:, -1].t().contiguous().cuda().t()   # classes are not contiguous: copied
    assert torch.equal(want, _check_sample(whole[:, -1].contiguous(), u, device_logits=columns, top_k=20))
    token, logprob = ser_amd.sample_tokens(whole[0, -1].cuda(), u[0].cuda(), top_k=20)   # one row without a batch axis
    assert token.shape == () == logprob.shape and token == want[0]
    token, logprob = ser_amd.sample_tokens(torch.zeros((0, 3, v), device="cuda"), torch.zeros((0, 3), device="cuda"))
    assert token.shape == (0, 3) == logprob.shape
    side = torch.cuda.Stream()
    x, uu = whole[:, -1].cuda(), u.cuda()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token, _ = ser_amd.sample_tokens(x, uu, top_k=20)
    side.synchronize()
    assert torch.equal(token, want)


# ---------------------------------------------------------------------------------------- distillation
def _teacher(n, v, k, seed, dtype=torch.float32, index_dtype=torch.int64):
    g = _gen(seed)
    index = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    return index.to(index_dtype), (torch.randn((n, k), generator=g) * 2).to(dtype)


def _distill_bounds(x, index, teacher, temperature, weight, dtype):
    """(losses, gradients, bounds of both) from the oracle."""
    rows, idx, tops = _np(x), index.cpu().numpy(), _np(teacher)
    n, v = rows.shape
    k = idx.shape[1]
    loss, grad, loss_off, grad_off = np.zeros(n), np.zeros((n, v)), np.zeros(n), np.zeros((n, v))
    for r in range(n):
        l, g = plain.distill_row(rows[r], idx[r], tops[r], temperature)
        # rounded to f32, a loss of 4.9e38 (a listed class at the lowest bf16 or f32) is infinite: it is past 3.4e38
        loss[r] = math.copysign(math.inf, l) if abs(l) > float(torch.finfo(torch.float32).max) else l
        w = 1.0 if weight is None else float(weight[r])
        grad[r] = g * w if w != 0 else 0.0
        p = plain.teacher_softmax(idx[r], tops[r], v, temperature)
        top = rows[r].max()
        if p is None or np.isnan(top) or top == np.inf:
            continue
        if top == -np.inf:   # every class masked: q = 0, the teacher's part is there all the same
            far, q = np.zeros(v), np.zeros(v)
        else:
            with np.errstate(over="ignore"):
                far = np.minimum((top - rows[r]) / temperature * 1.4427, 150.0)
                q = np.exp((rows[r] - top) / temperature)
            q /= q.sum()
        sum_off = (v / 64 + 64 + (q * far).sum()) * 2.0**-23      # of S: its terms, their order
        full = np.zeros(v)
        np.add.at(full, idx[r][(idx[r] >= 0) & (idx[r] < v)], p[(idx[r] >= 0) & (idx[r] < v)])
        t_far = np.minimum((np.nanmax(tops[r][np.isfinite(tops[r])]) - np.where(np.isfinite(tops[r]), tops[r], 0)) / temperature, 150).max()
        grad_off[r] = abs(w) * temperature * (q * (sum_off + (far + 6) * 2.0**-23) + full * (k / 16 + 16 + 2 * t_far) * 2.0**-23) \
            + np.abs(grad[r]) * HALF[dtype] * 1.01 + float(torch.finfo(dtype).tiny) * torch.finfo(dtype).eps
        # the loss: log S, and f64 from there; one rounding to f32.  A loss of -log q for a far class is as large as `far`
        loss_off[r] = temperature**2 * (2 * sum_off + 2.0**-40 * (1 + far.max())) + (abs(l) * 2.0**-23 if np.isfinite(l) else 0.0)
    return loss, grad, loss_off, grad_off


def _same(got, want, off):
    got, want = np.asarray(got), np.asarray(want)
    assert (np.isnan(got) == np.isnan(want)).all()
    fine = np.isfinite(want)
    assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all() and np.isfinite(got[fine]).all()
    over = np.abs(got[fine] - want[fine]) - off[fine]
    assert over.size == 0 or over.max() <= 0, (over.max(), np.abs(got[fine] - want[fine]).max())


def _check_distill(x, index, teacher, temperature=1.0, weight=None):
    """distillation_step, distillation_loss, and its autograd gradient against the oracle."""
    import ser_amd

    dx, di, dt = x.cuda(), index.cuda(), teacher.cuda()
    dw = None if weight is None else weight.cuda()
    loss, grad, loss_off, grad_off = _distill_bounds(x, index, teacher, temperature, weight, x.dtype)
    got_loss, got_grad = ser_amd.distillation_step(dx, di, dt, temperature=temperature, row_weight=dw)
    assert got_loss.dtype == torch.float32 and got_grad.dtype == x.dtype and got_grad.shape == x.shape
    _same(_np(got_loss), loss, loss_off)
    _same(_np(got_grad), grad, grad_off)
    leaf = dx.clone().requires_grad_()
    auto = ser_amd.distillation_loss(leaf, di, dt, temperature=temperature)
    (auto_grad,) = torch.autograd.grad(auto, leaf, grad_outputs=torch.ones_like(auto) if dw is None else dw)
    _same(_np(auto), loss, loss_off)
    _same(_np(auto_grad), grad, grad_off)
    with torch.no_grad():
        assert torch.equal(ser_amd.distillation_loss(dx, di, dt, temperature=temperature).nan_to_num(7.0), auto.detach().nan_to_num(7.0))
    again = ser_amd.distillation_step(dx, di, dt, temperature=temperature, row_weight=dw)
    assert torch.equal(again[1].nan_to_num(7.0), got_grad.nan_to_num(7.0)) and torch.equal(again[0].nan_to_num(7.0), got_loss.nan_to_num(7.0))
    inplace = dx.clone()
    _, out = ser_amd.distillation_step(inplace, di, dt, temperature=temperature, row_weight=dw, out=inplace)
    assert out is inplace and torch.equal(out.nan_to_num(7.0), got_grad.nan_to_num(7.0))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (7, 2, 1), (300, 8, 3), (33, 16, 16), (5, 64, 5), (9, 65, 64), (12, 187, 9), (3, 513, 100),
                                   (6, 1025, 7), (4, 2051, 256), (3, 4100, 20), (2, 8200, 300), (5, 20011, 64), (3, 50001, 33), (2, 70001, 17),
                                   (1, 131072, 2048)])
def test_distillation_matches_the_definition(dtype, n, v, k):
    index, teacher = _teacher(n, v, k, 50 + v, dtype=TYPES[(v + 1) % 3], index_dtype=torch.int32 if v % 2 else torch.int64)
    weight = torch.rand((n,), generator=_gen(v)) + 0.1
    _check_distill(_scores(n, v, dtype, v), index, teacher, temperature=(1.0, 2.0, 0.5)[v % 3], weight=weight)


@gpu
@pytest.mark.parametrize("n,v", [(2000, 300), (1500, 1030), (700, 5001), (520, 30011), (130, 70001), (128, 100003)])
def test_distillation_many_rows(n, v):
    """Row counts that fill the device, where a row is not divided."""
    index, teacher = _teacher(n, v, 6, v, dtype=torch.bfloat16)
    _check_distill(_scores(n, v, torch.bfloat16, n), index, teacher, temperature=2.0)


@gpu
@pytest.mark.parametrize("n", [5, 700])
@pytest.mark.parametrize("v", [1, 2, 3, 8, 15, 16, 17, 64, 65])
def test_distillation_lists_longer_than_the_classes(n, v):
    """Few classes, listed again and again, some entries outside them, by few rows and by many."""
    k = 37
    index = torch.randint(-2, v + 2, (n, k), generator=_gen(v), dtype=torch.int32)
    teacher = torch.randn((n, k), generator=_gen(v + 1)) * 2
    teacher[1, 5:] = -math.inf
    weight = torch.rand((n,), generator=_gen(2))
    _check_distill(_scores(n, v, torch.float32, v), index, teacher, temperature=0.8, weight=weight)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [12, 16, 40, 700, 5000, 60001])
def test_distillation_padding_masks_and_repeats(dtype, v):
    n, k = 14, 6
    x = _scores(n, v, dtype, v + 3)
    index, teacher = _teacher(n, v, k, v + 4)
    index[0, 2:] = -1                       # a shorter list
    index[1, :] = -1                        # none at all
    index[2, 0], index[2, 1] = v, v + 7     # outside the classes
    teacher[3, 1] = -math.inf
    teacher[4, :] = -math.inf
    index[5, :] = 11                        # the same class again and again
    index[6, 3] = index[6, 0]
    x[7, :] = LOWEST[dtype]
    x[8, v // 2 :] = LOWEST[dtype]
    x[8, : v // 2] = 1.0
    x[9, 1:] = -math.inf                    # masked classes, the teacher's among them or not
    index[9, :] = 0
    x[10, 3] = -math.inf
    index[10, 1] = 3
    x[11, :] = -math.inf
    x[12, 5] = math.nan
    x[13, 6] = math.inf
    weight = torch.full((n,), 0.25)
    weight[6] = 0.0
    _check_distill(x, index, teacher, temperature=1.5, weight=weight)
    weight[11:] = 0.0                       # whatever the row holds
    _check_distill(x, index, teacher, temperature=1.5, weight=weight)
    x[1, 2] = math.nan                      # a row without entries holds nothing that counts
    _check_distill(x, index, teacher, temperature=1.5, weight=weight)


@gpu
def test_distillation_layouts_and_reductions():
    import ser_amd

    n, v, k = 6, 1037, 8
    index, teacher = _teacher(n, v, k, 1)
    x = _scores(n, v, torch.bfloat16, 2)
    want_loss, want = ser_amd.distillation_step(x.cuda(), index.cuda(), teacher.cuda())
    wide = torch.zeros((n, v + 5), dtype=torch.bfloat16, device="cuda")
    wide[:, 1 : 1 + v] = x.cuda()
    loss, grad = ser_amd.distillation_step(wide[:, 1 : 1 + v], index.cuda(), teacher.cuda())
    assert torch.equal(loss, want_loss) and torch.equal(grad, want)
    ser_amd.distillation_step(wide[:, 1 : 1 + v], index.cuda(), teacher.cuda(), out=wide[:, 1 : 1 + v])
    assert torch.equal(wide[:, 1 : 1 + v], want) and not wide[:, 0].any() and not wide[:, 1 + v :].any()
    loss, grad = ser_amd.distillation_step(x.cuda().view(2, 3, v), index.cuda().view(2, 3, k), teacher.cuda().view(2, 3, k))
    assert torch.equal(loss.view(-1), want_loss) and torch.equal(grad.view(n, v), want)
    one, g1 = ser_amd.distillation_step(x[0].cuda(), index[0].cuda(), teacher[0].cuda())
    assert one.shape == () and g1.shape == (v,)
    # the gradient of a mean arrives as a broadcast number; of leading dimensions, as they are
    leaf = x.cuda().view(2, 3, v).clone().requires_grad_()
    ser_amd.distillation_loss(leaf, index.cuda().view(2, 3, k), teacher.cuda().view(2, 3, k)).mean().backward()
    _, g = ser_amd.distillation_step(x.cuda(), index.cuda(), teacher.cuda(), row_weight=torch.full((n,), 1.0 / n, device="cuda"))
    assert torch.equal(leaf.grad.view(n, v), g)
    empty = ser_amd.distillation_step(x.cuda()[:0], index.cuda()[:0], teacher.cuda()[:0])
    assert empty[0].shape == (0,) and empty[1].shape == (0, v)
    # one row of scores for all (stride 0)
    shared = x.cuda()[:1].expand(n, v)
    loss, grad = ser_amd.distillation_step(shared, index.cuda(), teacher.cuda())
    again = ser_amd.distillation_step(shared.contiguous(), index.cuda(), teacher.cuda())
    assert torch.equal(loss, again[0]) and torch.equal(grad, again[1])
    with pytest.raises(ValueError, match="overlap"):
        ser_amd.distillation_step(x.cuda(), index.cuda(), teacher.cuda(), out=shared)
    big = torch.zeros((n + 1, v), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        ser_amd.distillation_step(big[:n], index.cuda(), teacher.cuda(), out=big[1:])
    with pytest.raises(RuntimeError):   # differentiable once
        leaf = x.float().cuda().requires_grad_()
        (g,) = torch.autograd.grad(ser_amd.distillation_loss(leaf, index.cuda(), teacher.cuda()).sum(), leaf, create_graph=True)
        g.sum().backward()


@gpu
def test_scores_overwritten_by_their_gradient_are_an_error_in_backward():
    import ser_amd

    index, teacher = (t.cuda() for t in _teacher(4, 300, 3, 1))
    leaf = _scores(4, 300, torch.float32, 1).cuda().requires_grad_()
    logits = leaf * 1.0
    loss = ser_amd.distillation_loss(logits, index, teacher)
    ser_amd.distillation_step(logits.detach(), index, teacher, out=logits.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


@gpu
def test_distillation_saved_in_host_memory():
    import ser_amd

    n, v, k = 6, 1037, 8
    index, teacher = (t.cuda() for t in _teacher(n, v, k, 1))
    for x in (_scores(n, v, torch.bfloat16, 2).cuda(), _scores(v, n, torch.bfloat16, 2).cuda().t(), _scores(n, v, torch.float32, 2).cuda()[:1].expand(n, v)):
        leaf = x.detach().requires_grad_()
        (want,) = torch.autograd.grad(ser_amd.distillation_loss(leaf, index, teacher).sum(), leaf)
        with torch.autograd.graph.save_on_cpu():
            loss = ser_amd.distillation_loss(leaf, index, teacher)
        (got,) = torch.autograd.grad(loss.sum(), leaf)
        assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [8.5, 20.0, 100.0, 1000.0])
@pytest.mark.parametrize("n,v,k,masked", [(5, 8, 8, False), (7, 3, 3, False), (600, 32, 32, False), (4, 33, 33, False), (520, 64, 70, False), (3, 300, 300, False),
                                          (2, 2048, 2048, False), (3, 4096, 700, True), (3, 4097, 64, True), (2, 50001, 33, True), (2, 50001, 64, False)])
def test_distillation_at_high_temperatures(dtype, temperature, n, v, k, masked):
    """Lists that cover the classes (all of them, or all that are not masked): the loss stays of the size of their scores' variance,
    a millionth of the T^2 that it is a difference of.  f64 sums, exponentials and logarithms: (V / 64 + 64) 2^-50 of T^2 is a
    hundred units for each of its terms, less than 2^-20 of a loss; and one rounding.  The gradient of a listed class is such a
    difference too, rounded once; of another it is T q, by a 2^x in f32."""
    import ser_amd

    g = _gen(v + k)
    index = torch.stack([torch.cat([torch.randperm(v, generator=g)[: min(k, v)], torch.randint(0, v, (max(0, k - v),), generator=g)]) for _ in range(n)])
    teacher = (torch.randn((n, k), generator=g) * 2).to(dtype)
    x = _scores(n, v, dtype, v)
    if masked:
        x = torch.full_like(x, -math.inf).scatter_(1, index, x.gather(1, index))
    weight = torch.rand((n,), generator=g) + 0.1
    dx, di, dt, dw = x.cuda(), index.cuda(), teacher.cuda(), weight.cuda()
    loss, grad = ser_amd.distillation_step(dx, di, dt, temperature=temperature, row_weight=dw)
    leaf = dx.clone().requires_grad_()
    auto = ser_amd.distillation_loss(leaf, di, dt, temperature=temperature)
    (auto_grad,) = torch.autograd.grad(auto, leaf, grad_outputs=dw)
    assert torch.equal(auto, loss) and torch.equal(auto_grad, grad)
    inplace = dx.clone()
    ser_amd.distillation_step(inplace, di, dt, temperature=temperature, row_weight=dw, out=inplace)
    assert torch.equal(inplace, grad)
    t = float(np.float32(temperature))
    for r in range(0, n, max(1, n // 20)):
        want, want_grad = plain.distill_row(_np(x)[r], index[r].numpy(), _np(teacher)[r], t)
        w, off = float(weight[r]), (v / 64 + 64) * 2.0**-50
        assert abs(float(loss[r]) - want) <= abs(want) * 2.0**-24 * 1.01 + t * t * off, (r, float(loss[r]), want)
        far = np.minimum((_np(x)[r].max() - _np(x)[r]) / t, 150.0)
        bound = np.abs(want_grad) * w * ((far * 1.45 + 6) * 2.0**-23 + HALF[dtype] * 1.01) + w * t * off + float(torch.finfo(dtype).tiny) * torch.finfo(dtype).eps
        _same(_np(grad)[r], want_grad * w, bound)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [9.0, 100.0, 1000.0])
@pytest.mark.parametrize("n,v,k,masked", [(1, 65537, 40, True), (3, 100003, 300, False), (63, 70001, 6, True), (2, 300007, 2048, True)])
def test_distillation_of_few_long_rows_at_high_temperatures(dtype, temperature, n, v, k, masked):
    """Rows that are divided among workgroups.  The loss is held to f64 as elsewhere; the gradient has S rounded to f32 between its
    two kernels, which moves it by T q 2^-24."""
    import ser_amd

    index, teacher = _teacher(n, v, k, v, dtype=dtype)
    x = _scores(n, v, dtype, v)
    if masked:   # but for the listed classes, and whole pieces of the row
        x = torch.full_like(x, -math.inf).scatter_(1, index, x.gather(1, index))
        x[0, : v // 2] = -math.inf
        index[0] = torch.where(index[0] < v // 2, -1, index[0])
    if n == 63:
        x[5, 9], x[6, 60000], x[7, :], index[8, :] = math.nan, math.inf, -math.inf, -1
    weight = torch.rand((n,), generator=_gen(1)) + 0.1
    dx, di, dt, dw = x.cuda(), index.cuda(), teacher.cuda(), weight.cuda()
    loss, grad = ser_amd.distillation_step(dx, di, dt, temperature=temperature, row_weight=dw)
    leaf = dx.clone().requires_grad_()
    auto = ser_amd.distillation_loss(leaf, di, dt, temperature=temperature)
    (auto_grad,) = torch.autograd.grad(auto, leaf, grad_outputs=dw)
    assert torch.equal(auto.nan_to_num(7.0), loss.nan_to_num(7.0)) and torch.equal(auto_grad.nan_to_num(7.0), grad.nan_to_num(7.0))
    inplace = dx.clone()
    ser_amd.distillation_step(inplace, di, dt, temperature=temperature, row_weight=dw, out=inplace)
    assert torch.equal(inplace.nan_to_num(7.0), grad.nan_to_num(7.0))
    t = float(np.float32(temperature))
    for r in range(min(n, 9)):
        row = _np(x)[r]
        want, want_grad = plain.distill_row(row, index[r].numpy(), _np(teacher)[r], t)
        w, off = float(weight[r]), (v / 64 + 64) * 2.0**-50
        _same(np.asarray([float(loss[r])]), np.asarray([want]), np.asarray([abs(want) * 2.0**-24 * 1.01 + t * t * off]))
        if not np.isfinite(row.max()):
            _same(_np(grad)[r], want_grad * w, np.abs(np.nan_to_num(want_grad)) * w * (HALF[dtype] * 1.01 + 2.0**-22))
            continue
        far = np.minimum((row.max() - row) / t, 150.0)
        q = np.exp((row - row.max()) / t)
        q /= q.sum()
        bound = np.abs(want_grad) * w * ((far * 1.45 + 6) * 2.0**-23 + HALF[dtype] * 1.01) + w * t * (q * 2.0**-23 + off) \
            + float(torch.finfo(dtype).tiny) * torch.finfo(dtype).eps
        _same(_np(grad)[r], want_grad * w, bound)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [12, 40, 700, 5000])
def test_distillation_masks_at_high_temperatures(dtype, v):
    n, k = 11, 6
    x = _scores(n, v, dtype, v + 3)
    index, teacher = _teacher(n, v, k, v + 4)
    index[0, 2:] = -1
    index[1, :] = -1
    index[2, 0], index[2, 1] = v, v + 7
    teacher[3, 1] = -math.inf
    teacher[4, :] = -math.inf
    index[5, :] = 11
    x[6, 1:] = -math.inf
    index[6, :] = 0
    x[7, :] = -math.inf
    x[8, 5] = math.nan
    x[9, 6] = math.inf
    x[10, :] = LOWEST[dtype]
    weight = torch.full((n,), 0.25)
    _check_distill(x, index, teacher, temperature=20.0, weight=weight)
    weight[5:9] = 0.0
    x[1, 2] = math.nan
    _check_distill(x, index, teacher, temperature=1000.0, weight=weight)


@gpu
@pytest.mark.parametrize("dtype,n,v", [(torch.float32, 128, 32769), (torch.float32, 129, 49152), (torch.float32, 128, 49153), (torch.float32, 128, 65536),
                                       (torch.float32, 128, 65537), (torch.float16, 128, 65537), (torch.float16, 128, 98304), (torch.float16, 128, 98305),
                                       (torch.float16, 128, 131072), (torch.bfloat16, 128, 98305)])
def test_distillation_longest_held_rows(dtype, n, v):
    """Rows of 12 and 16 vectors a thread, at both ends of what these hold, and the first that nothing does."""
    index, teacher = _teacher(n, 700, 5, v, dtype=torch.float32)
    index += v - 700   # the row's end, where the vectors are not whole
    _check_distill(_scores(n, v, dtype, n), index, teacher, temperature=1.5)


@gpu
@pytest.mark.parametrize("v", [8, 700, 30011])
def test_distillation_gradient_against_differences(v):
    """The kernel's gradient against differences of the kernel's own loss along random directions.  f32: the two losses
    are off by 2 T^2 (V/64 + 128) 2^-23 together, divided by the step 2h; the cubic term is below h^2."""
    import ser_amd

    n, k, temperature, h = 3, 4, 1.5, 0.125
    index, teacher = _teacher(n, v, k, 9)
    x = _scores(n, v, torch.float32, 8, spread=1.5).cuda()
    d = torch.sign(torch.randn((n, v), generator=_gen(10))).cuda()
    _, g = ser_amd.distillation_step(x, index.cuda(), teacher.cuda(), temperature=temperature)
    up = ser_amd.distillation_loss(x + h * d, index.cuda(), teacher.cuda(), temperature=temperature).double()
    down = ser_amd.distillation_loss(x - h * d, index.cuda(), teacher.cuda(), temperature=temperature).double()
    off = temperature**2 * (v / 64 + 128) * 2.0**-22 / (2 * h) + h * h
    assert ((up - down) / (2 * h) - (g.double() * d.double()).sum(1)).abs().max().item() <= off


@gpu
def test_classifier_distillation():
    """The fast profile's classifier against a teacher that names its likeliest emotions."""
    from ser_amd import GpuEmotionClassifier

    rng = np.random.default_rng(4)
    gpu_model = GpuEmotionClassifier(classes=np.arange(8), coefs=[rng.standard_normal((20, 12)), rng.standard_normal((12, 8))],
                                     intercepts=[rng.standard_normal(12), rng.standard_normal(8)])
    x = rng.standard_normal((50, 20))
    index = torch.stack([torch.randperm(8, generator=_gen(i))[:3] for i in range(50)])
    teacher = torch.randn((50, 3), generator=_gen(99))
    loss, grad = gpu_model.distillation_device(x, index.cuda(), teacher.cuda(), temperature=2.0)
    scores = torch.from_numpy(np.log(gpu_model.predict_proba(x))).float()
    want = _distill_bounds(scores, index, teacher, 2.0, None, torch.float32)
    # the scores themselves are f32: half a step each moves a row's loss by at most T 2^-24 max |score| times 2
    slack = 4 * 2.0 * 2.0**-24 * scores.abs().max().item()
    _same(_np(loss), want[0], want[2] + slack)
    _same(_np(grad), want[1], want[3] + slack)


@gpu
@pytest.mark.parametrize("n_out", [1, 2, 8])
@pytest.mark.parametrize("scale", [1.0, 40.0, 3000.0])
def test_classifier_distillation_of_confident_models(n_out, scale):
    """Scores far apart: the probability of the other class rounds to 0 (of two classes from a logit of 37 on, of more from
    745), the distance of the scores does not."""
    from ser_amd import GpuEmotionClassifier

    rng = np.random.default_rng(5)
    w, b = rng.standard_normal((6, n_out)) * scale, rng.standard_normal(n_out)
    n_classes = max(2, n_out)
    model = GpuEmotionClassifier(classes=np.arange(n_classes), coefs=[w], intercepts=[b], out_activation="logistic" if n_out == 1 else "softmax")
    x = rng.standard_normal((60, 6))
    logits = x @ w + b
    scores = np.concatenate([np.zeros_like(logits), logits], 1) if n_out == 1 else logits
    scores = scores - scores.max(1, keepdims=True)
    index = torch.stack([torch.randperm(n_classes, generator=_gen(i))[:2] for i in range(60)])
    teacher = torch.randn((60, 2), generator=_gen(98))
    loss, grad = model.distillation_device(x, index.cuda(), teacher.cuda(), temperature=1.5)
    want = _distill_bounds(torch.from_numpy(scores), index, teacher, 1.5, None, torch.float32)
    # the distances are f32: half a step each moves a row's loss by at most T 2^-24 max |distance| times 2, as much again for the
    # 6 products of a score in f64 and the loss's own rounding
    slack = 4 * 1.5 * 2.0**-24 * np.abs(scores).max()
    assert np.isfinite(want[0]).all()
    _same(_np(loss), want[0], want[2] + slack)
    _same(_np(grad), want[1], want[3] + slack)
    label, proba = model.predict_device(x)
    scored, raw = model._forward(x, 2)
    assert torch.equal(label, scored) and raw.shape == proba.shape
    torch.testing.assert_close(torch.softmax(raw, 1), proba, rtol=1e-9, atol=1e-15)


# ------------------------------------------------------------------------------------------- embedding
@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,d", [(1, 1), (5, 3), (300, 16), (77, 187), (1000, 64), (50, 512), (33, 1025), (11, 4104)])
def test_embedding_lookup(dtype, v, d):
    import ser_amd

    table = torch.randn((v, d), generator=_gen(v + d)).to(dtype)
    scale = math.sqrt(d) * 1.0001
    for shape, token_dtype in (((1,), torch.int64), ((7,), torch.int32), ((3, 65), torch.int64), ((0,), torch.int64), ((), torch.int32)):
        tok = torch.randint(-2, v + 2, shape, generator=_gen(d), dtype=torch.int64).to(token_dtype)
        got = ser_amd.embed_tokens(tok.cuda(), table.cuda(), scale=scale).cpu()
        inside = ((tok >= 0) & (tok < v)).unsqueeze(-1)
        # the product is exact in f64 (24 + 24 bits).  The kernel rounds it to f32 and that to the table's type, or (the
        # f16 multiply that rounds its f32 product itself) to the type at once: 2^-24 and half a step, no more
        want = torch.where(inside, table[tok.long().clamp(0, v - 1)].double() * float(np.float32(scale)), 0.0)
        off = want.abs() * (2.0**-24 + HALF[dtype]) * (1 + 2.0**-20) + float(torch.finfo(dtype).tiny) * torch.finfo(dtype).eps
        assert got.shape == (*shape, d) and got.dtype == dtype and (got.double() - want).abs().le(off).all()
        assert not got[~inside.expand_as(got)].any()


@gpu
def test_embedding_layouts():
    import ser_amd

    wide = torch.randn((40, 100), generator=_gen(1)).cuda()
    tok = torch.tensor([0, 39, 5, -1, 40, 5, 2**40], device="cuda")
    want = ser_amd.embed_tokens(tok, wide[:, 3:80].contiguous(), scale=2.0)
    assert torch.equal(want, ser_amd.embed_tokens(tok, wide[:, 3:80], scale=2.0))
    assert torch.equal(want, ser_amd.embed_tokens(tok, wide[:, 3:80].t().contiguous().t(), scale=2.0))
    assert not want[[3, 4, 6]].any() and torch.equal(want[1], 2.0 * wide[39, 3:80])
    pairs = torch.stack([tok, tok * 0], 1)   # a strided column of tokens
    assert torch.equal(want, ser_amd.embed_tokens(pairs[:, 0], wide[:, 3:80], scale=2.0))
    out = torch.full((7, 90), 5.0, device="cuda")
    assert ser_amd.embed_tokens(tok, wide[:, 3:80], scale=2.0, out=out[:, 1:78]).data_ptr() == out[:, 1:78].data_ptr()
    assert torch.equal(out[:, 1:78], want) and (out[:, 0] == 5).all() and (out[:, 78:] == 5).all()
    with pytest.raises(ValueError, match="share memory"):
        ser_amd.embed_tokens(tok, wide, out=wide[:7])


def _check_embedding_gradient(tok, grad, v, scale=1.0, out_dtype=None, **kwargs):
    import ser_amd

    got = ser_amd.embedding_gradient(grad.cuda(), tok.cuda(), v, scale=scale, dtype=out_dtype, **kwargs)
    d = grad.shape[-1]
    want, size, count = plain.embedding_gradient(_np(grad).reshape(-1, d), tok.reshape(-1).numpy(), v, float(np.float32(scale)))
    out_dtype = out_dtype or grad.dtype
    assert got.shape == (v, d) and got.dtype == out_dtype
    off = (count[:, None] + 2) * 2.0**-24 * size + np.abs(want) * HALF[out_dtype] * 1.01 \
        + float(torch.finfo(out_dtype).tiny) * torch.finfo(out_dtype).eps
    _same(_np(got), want, off)
    assert torch.equal(got, ser_amd.embedding_gradient(grad.cuda(), tok.cuda(), v, scale=scale, dtype=out_dtype, **kwargs))
    return got


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(0, 5, 7), (1, 1, 1), (1, 40, 16), (3, 100, 187), (64, 7, 33), (127, 1, 20), (128, 1, 8), (129, 1, 8), (300, 1, 65),
                                   (1000, 3, 40), (2047, 500, 24), (2048, 500, 24), (2049, 3000, 24), (5000, 50, 520), (20000, 9000, 12),
                                   (70000, 300, 5), (300, 100000, 9), (4096, 60000, 6), (4097, 70000, 6), (140000, 5000, 4), (300000, 140000, 3)])
def test_embedding_gradient_matches_the_definition(dtype, n, v, d):
    tok = torch.randint(-1, v + 1, (n,), generator=_gen(n + v), dtype=torch.int64)
    tok[::5] = v // 2   # a frequent one
    grad = torch.randn((n, d), generator=_gen(d)).to(dtype)
    _check_embedding_gradient(tok, grad, v, scale=1.25)
    _check_embedding_gradient(tok.to(torch.int32), grad, v, scale=-3.0, out_dtype=torch.float32)


@gpu
@pytest.mark.parametrize("lengths", [(32,), (33,), (31, 33, 1), (64, 64, 5), (1, 33, 31, 32), (5, 27, 33, 33, 2, 100), (96, 1, 31, 65), (128,), (129,), (127, 129, 1), (1, 129, 127, 128), (256, 256, 1, 300), (5, 123, 129, 129, 2, 400), (130, 130, 130, 130),
                                     (1000, 1, 1, 1, 700), (64, 64, 128, 128, 129), (2048, 2049)])
@pytest.mark.parametrize("shuffled", [False, True])
def test_embedding_gradient_runs_at_tile_borders(lengths, shuffled):
    """Runs of equal tokens that begin and end at, before and after the borders of the tiles that long runs are cut into."""
    tok = torch.repeat_interleave(torch.arange(len(lengths)) * 2 + 1, torch.tensor(lengths))
    if shuffled:
        tok = tok[torch.randperm(tok.numel(), generator=_gen(1))]
    v = 2 * len(lengths) + 2
    grad = torch.randn((tok.numel(), 70), generator=_gen(2))
    _check_embedding_gradient(tok, grad, v)
    padded = torch.cat([torch.full((333,), -1), tok, torch.full((200,), v)])   # long runs of padding are no row
    _check_embedding_gradient(padded, torch.randn((padded.numel(), 70), generator=_gen(3)), v)


@gpu
@pytest.mark.parametrize("v", [254, 255, 256, 1022, 1023, 1024, 65534, 65535, 65536, (1 << 20) - 1, 1 << 20, (1 << 22) + 5])
def test_embedding_gradient_number_of_sort_passes(v):
    for n in (4000, 5000):   # by one workgroup, by many
        tok = torch.randint(0, v, (n,), generator=_gen(v), dtype=torch.int64)
        tok[:3] = torch.tensor([0, v - 1, v])
        _check_embedding_gradient(tok, torch.randn((n, 3), generator=_gen(1)), v)


@gpu
def test_embedding_gradient_of_a_million_tokens():
    """So many that the sort's counts are added up by a kernel of their own."""
    n, v = 1100000, 3001
    tok = torch.randint(-1, v + 1, (n,), generator=_gen(1), dtype=torch.int64)
    tok[::7] = 5
    _check_embedding_gradient(tok, torch.randn((n, 2), generator=_gen(2)), v)


@gpu
def test_embedding_gradient_accumulates_and_layouts():
    import ser_amd

    n, v, d = 900, 60, 37
    tok = torch.randint(0, 50, (n,), generator=_gen(1), dtype=torch.int64)
    tok[::3] = 7
    grad = torch.randn((n, d), generator=_gen(2)).to(torch.bfloat16)
    base = torch.randn((v, d + 4), generator=_gen(3))
    out = base.clone().cuda()
    got = ser_amd.embedding_gradient(grad.cuda(), tok.cuda(), v, scale=0.5, out=out[:, 2 : 2 + d], accumulate=True)
    assert got.data_ptr() == out[:, 2:].data_ptr()
    want, size, count = plain.embedding_gradient(_np(grad), tok.numpy(), v, 0.5)
    off = (count[:, None] + 2) * 2.0**-24 * (size + np.abs(_np(base)[:, 2 : 2 + d]))
    _same(_np(out)[:, 2 : 2 + d], want + _np(base)[:, 2 : 2 + d], off)
    assert torch.equal(out[:, :2].cpu(), base[:, :2]) and torch.equal(out[:, 2 + d :].cpu(), base[:, 2 + d :])
    assert torch.equal(out[50:].cpu(), base[50:])   # rows no token names
    # one gradient row for all tokens (a broadcast), and a transposed one
    _check_embedding_gradient(tok, grad[:1].expand(n, d), v)
    assert torch.equal(ser_amd.embedding_gradient(grad.cuda().t().contiguous().t(), tok.cuda(), v), ser_amd.embedding_gradient(grad.cuda(), tok.cuda(), v))
    assert torch.equal(ser_amd.embedding_gradient(grad.cuda().view(30, 30, d), tok.cuda().view(30, 30), v), ser_amd.embedding_gradient(grad.cuda(), tok.cuda(), v))
    # NaN and infinity stay in their rows
    grad[4, 0], grad[5, 1] = math.nan, math.inf
    got = ser_amd.embedding_gradient(grad.cuda(), tok.cuda(), v).cpu()
    assert got[tok[4], 0].isnan() and got[tok[5], 1] == math.inf
    assert int((~got.isfinite()).sum()) == 2


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v,d", [(40, 3, 70001), (500, 9, 13), (5000, 40, 187), (3, 7, 5), (200, 1, 1029)])
def test_embedding_gradient_accumulates_in_its_own_type(dtype, n, v, d):
    """Short and long runs, vectors that reach past a row and rows shorter than one: added to what is there, with one rounding."""
    import ser_amd

    tok = torch.randint(-1, max(1, v - 1), (n,), generator=_gen(n), dtype=torch.int64)   # the last row gets nothing, where there are two
    grad = torch.randn((n, d), generator=_gen(d)).to(dtype)
    base = torch.randn((v, d), generator=_gen(3)).to(dtype)
    out = base.clone().cuda()
    got = ser_amd.embedding_gradient(grad.cuda(), tok.cuda(), v, scale=0.75, out=out, accumulate=True)
    assert got is out
    want, size, count = plain.embedding_gradient(_np(grad), tok.numpy(), v, 0.75)
    want = want + _np(base)
    off = (count[:, None] + 2) * 2.0**-24 * (size + np.abs(_np(base))) + np.abs(want) * HALF[dtype] * 1.01
    _same(_np(got), want, off)
    if v > 1:
        assert torch.equal(got[v - 1].cpu(), base[v - 1])


@gpu
def test_tables_and_scores_of_one_row():
    """Rows of stride 0: one row of a table, or of scores, for all."""
    import ser_amd

    row = torch.randn((1, 8), generator=_gen(1)).cuda()
    tok = torch.tensor([0, 4, 5, -1], device="cuda")
    assert torch.equal(ser_amd.embed_tokens(tok, row.expand(5, 8)), ser_amd.embed_tokens(tok, row.expand(5, 8).contiguous()))
    index, teacher = (t.cuda() for t in _teacher(700, 8, 3, 2))
    for temperature in (2.0, 20.0):
        got = ser_amd.distillation_step(row.expand(700, 8), index, teacher, temperature=temperature)
        want = ser_amd.distillation_step(row.expand(700, 8).contiguous(), index, teacher, temperature=temperature)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_embedding_autograd():
    import ser_amd

    table = torch.randn((30, 20), generator=_gen(1), dtype=torch.float32).cuda().requires_grad_()
    tok = torch.tensor([[1, 2, 1], [29, -1, 30]], device="cuda")
    y = ser_amd.embed_tokens(tok, table, scale=3.0)
    g = torch.randn(y.shape, generator=_gen(2)).cuda()
    y.backward(g)
    assert torch.equal(table.grad, ser_amd.embedding_gradient(g, tok, 30, scale=3.0))
    # linear in the table: the gradient is the difference quotient, up to f32
    d = torch.randn((30, 20), generator=_gen(3)).cuda()
    with torch.no_grad():
        slope = ((ser_amd.embed_tokens(tok, d, scale=3.0) * g).double().sum() - (table.grad.double() * d.double()).sum()).abs()
    assert slope <= 2.0**-20 * (3 * (g.abs().sum() * d.abs().max()))
    table.grad = None
    ser_amd.embed_tokens(tok, table, scale=3.0).sum().backward()   # a broadcast gradient
    assert torch.equal(table.grad, ser_amd.embedding_gradient(torch.ones_like(g), tok, 30, scale=3.0))


# --------------------------------------------------------------------------------- together, and in use
def _train_step(tokens, table, head, uniform, index, teacher):
    """Draw, look up, score, distil, and both gradients that reach the shared table: the operators as a loop uses them."""
    import ser_amd

    h = ser_amd.embed_tokens(tokens, table, scale=0.5)
    logits = torch.tanh(h.float()) @ head
    drawn, logprob = ser_amd.sample_tokens(logits, uniform, temperature=0.8, top_k=30, top_p=0.95)
    weight = torch.full(tokens.shape, 1.0 / tokens.numel(), device=tokens.device)
    loss, dlogits = ser_amd.distillation_step(logits, index, teacher, temperature=2.0, row_weight=weight)
    dh = (dlogits @ head.t()) * (1 - torch.tanh(h.float()) ** 2)
    dtable = ser_amd.embedding_gradient(dh, tokens, table.shape[0], scale=0.5)
    ser_amd.embedding_gradient(dh, drawn, table.shape[0], scale=0.1, out=dtable, accumulate=True)
    return drawn, logprob, loss, dlogits, dtable


def _train_inputs(seed, n=48, v=400, d=32, k=5):
    index, teacher = _teacher(n, v, k, seed)
    return [t.cuda() for t in (torch.randint(-1, v, (n,), generator=_gen(seed), dtype=torch.int64), torch.randn((v, d), generator=_gen(seed + 1)),
                               torch.randn((d, v), generator=_gen(seed + 2)), torch.rand((n,), generator=_gen(seed + 3)), index, teacher)]


@gpu
def test_operators_together():
    import ser_amd

    tokens, table, head, uniform, index, teacher = _train_inputs(5)
    drawn, logprob, loss, dlogits, dtable = _train_step(tokens, table, head, uniform, index, teacher)
    h = ser_amd.embed_tokens(tokens, table, scale=0.5)
    logits = torch.tanh(h) @ head
    for r in range(tokens.numel()):
        t, _ = plain.sample_row(_np(logits)[r], _np(uniform)[r], temperature=float(np.float32(0.8)), top_k=30, top_p=float(np.float32(0.95)))
        assert t == int(drawn[r])
    # autograd through the same operators gives the same table gradient as the explicit calls
    leaf = table.clone().requires_grad_()
    scores = torch.tanh(ser_amd.embed_tokens(tokens, leaf, scale=0.5)) @ head
    auto = ser_amd.distillation_loss(scores, index, teacher, temperature=2.0)
    auto.mean().backward()
    assert torch.equal(auto.detach(), loss)
    explicit = ser_amd.embedding_gradient((dlogits @ head.t()) * (1 - torch.tanh(h) ** 2), tokens, table.shape[0], scale=0.5)
    # the same formula in another order of f32 products: 32 + 400 terms
    torch.testing.assert_close(leaf.grad, explicit, rtol=1e-4, atol=1e-6)


@gpu
def test_operators_in_a_graph():
    """Captured once and replayed with new inputs, with eager calls of the same operators between the replays."""
    state = _train_inputs(20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _train_step(*state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _train_step(*state)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        out2 = _train_step(*state)
    for seed in (21, 22, 23, 24):
        fresh = _train_inputs(seed)
        for a, b in zip(state, fresh):
            a.copy_(b)
        want = [t.clone() for t in _train_step(*fresh)]
        torch.cuda.synchronize()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        for got, got2, w in zip(out, out2, want):
            assert torch.equal(got, w) and torch.equal(got2, w), seed


@gpu
def test_operators_from_two_threads():
    """Two threads, each on its own stream, at once: nothing is shared."""
    states = [_train_inputs(s, n=200, v=3001) for s in (31, 32)]
    want = [[t.clone() for t in _train_step(*s)] for s in states]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = _train_step(*states[i])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as e:  # pragma: no cover - reported below
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@gpu
def test_offsets_beyond_32_bits():
    """Rows, tables and gradients whose elements are counted past 2^31."""
    import ser_amd

    n, v = 33000, 65552
    x = torch.zeros((n, v), dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 1 << 31
    last = _scores(3, v, torch.bfloat16, 1)
    x[-3:] = last.cuda()
    index, teacher = _teacher(n, 8, 2, 2)
    index[-3:] += 65000
    u = torch.rand((n,), generator=_gen(3))
    token, _ = ser_amd.sample_tokens(x, u.cuda(), top_k=9)
    for r in range(3):
        assert int(token[n - 3 + r]) == plain.sample_row(_np(last)[r], _np(u)[n - 3 + r], top_k=9)[0]
    assert int(token[0]) == plain.sample_row(np.zeros(v), float(u[0]), top_k=9)[0]
    want_loss, want, loss_off, off = _distill_bounds(last, index[-3:], teacher[-3:], 1.0, None, torch.bfloat16)
    loss, grad = ser_amd.distillation_step(x, index.cuda(), teacher.cuda(), out=x)
    _same(_np(loss[-3:]), want_loss, loss_off)
    _same(_np(grad[-3:]), want, off)
    del x, grad
    d, v = 2048, 1100000
    table = torch.zeros((v, d), dtype=torch.bfloat16, device="cuda")
    table[-1] = torch.arange(d).to(torch.bfloat16).cuda()
    assert torch.equal(ser_amd.embed_tokens(torch.tensor([v - 1, 0], device="cuda"), table)[0], table[-1])
    g = torch.randn((3, d), generator=_gen(4)).to(torch.bfloat16).cuda()
    ser_amd.embedding_gradient(g, torch.tensor([0, v - 1, v - 2], device="cuda"), v, out=table)
    assert torch.equal(table[[0, v - 1, v - 2]], g) and not table[1 : v - 2].any()


@gpu
def test_a_gpu_and_a_cpu_tensor_do_not_mix():
    import ser_amd

    x = torch.zeros((2, 8), device="cuda")
    with pytest.raises(ValueError, match="device|on cpu"):
        ser_amd.sample_tokens(x, torch.zeros(2))
    with pytest.raises(ValueError, match="on cpu"):
        ser_amd.distillation_loss(x, torch.zeros((2, 1), dtype=torch.int64), torch.zeros((2, 1)).cuda())
    with pytest.raises(ValueError, match="on cpu"):
        ser_amd.embed_tokens(torch.zeros(2, dtype=torch.int64), x)


@gpu
def test_one_row_of_any_stride():
    """The distance to the next row of a tensor with one row means nothing: torch allows any number there."""
    import ser_amd

    x = _scores(1, 70, torch.float32, 8).cuda()
    odd = x.as_strided((1, 70), (1, 1))
    u = torch.rand((1,), generator=_gen(1)).cuda()
    assert odd.is_contiguous() and torch.equal(ser_amd.sample_tokens(x, u)[0], ser_amd.sample_tokens(odd, u)[0])
    index, teacher = (t.cuda() for t in _teacher(1, 70, 3, 2))
    want = ser_amd.distillation_step(x, index, teacher)
    out = torch.empty((70,), device="cuda").as_strided((1, 70), (1, 1))
    got = ser_amd.distillation_step(odd, index, teacher, out=out)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], out)
    token = torch.zeros((1,), dtype=torch.int64, device="cuda")
    assert torch.equal(ser_amd.embed_tokens(token, odd, out=out), x)
    assert torch.equal(ser_amd.embedding_gradient(odd, token, 1, out=out), x)


@gpu
def test_autograd_in_a_graph():
    """Forward and backward of both differentiable operators, captured with torch.autograd.grad and replayed."""
    import ser_amd

    n, v, d = 37, 611, 24
    tokens = torch.randint(-1, v, (n,), generator=_gen(5)).cuda()
    table, head = (torch.randn(s, generator=_gen(6)).cuda() for s in ((v, d), (d, v)))
    index, teacher = (t.cuda() for t in _teacher(n, v, 4, 7))
    weight = torch.rand((n,), generator=_gen(8)).cuda()

    def step(leaf):
        x = ser_amd.embed_tokens(tokens, leaf, scale=2.0) @ head
        loss = ser_amd.distillation_loss(x, index, teacher, temperature=1.5)
        return [loss.detach(), *torch.autograd.grad(loss, leaf, grad_outputs=weight)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(table.clone().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    captured = table.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(captured)
    for seed in (1, 2, 3):
        with torch.no_grad():
            captured.copy_(torch.randn((v, d), generator=_gen(seed)))
        want = [t.clone() for t in step(captured.detach().clone().requires_grad_())]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        # the matrix products between them are the library's, which may choose another order in a graph: n terms of f32
        for got, w in zip(out, want):
            assert torch.allclose(got, w, rtol=v * 2.0**-22, atol=float(w.abs().max()) * v * 2.0**-24), seed
