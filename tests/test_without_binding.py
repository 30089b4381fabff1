"""The backend where the extension module cannot be had (no C compiler, no Python headers, another interpreter): the library's functions are then called
through ctypes, and everything else is as it was."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys
sys.modules["minml_b200._binding"] = None  # what an import of a module that is not there comes to
import pytest
import tests.test_binding as t, tests.test_large_workspace as w
from minml_b200 import backend as B
assert type(B._binding).__name__ == "CtypesCalls"
t.test_refusals()
t.test_a_refused_call_leaves_its_arguments_alone()
w.test_a_workspace_above_two_gigabytes_is_described()
print("as with it")
"""


def test_the_backend_imports_and_refuses_alike():
    run = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True)
    assert run.returncode == 0 and "as with it" in run.stdout, run.stderr[-2000:]


def test_the_library_is_built_without_a_compiler_for_the_module(monkeypatch, capsys):
    from minml_b200 import build as b
    try:
        b.find_nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    monkeypatch.setenv("CC", "/nonexistent/compiler")
    with pytest.raises(RuntimeError, match="extension module"):
        b.build_binding(force=True)
    before = b.build_binding
    monkeypatch.setattr(b, "build_binding", lambda force=False: before(force=True))
    assert b.build() == b.LIB and os.path.exists(b.LIB)
    assert "extension module" in capsys.readouterr().err


def test_the_module_belongs_to_one_interpreter():
    """Its file name has the interpreter's tag, so that another one neither loads it nor takes it for its own."""
    import importlib.machinery
    import sysconfig
    from minml_b200 import build as b
    assert os.path.basename(b.BINDING) == "_binding" + sysconfig.get_config_var("EXT_SUFFIX")
    assert any(b.BINDING.endswith(s) for s in importlib.machinery.EXTENSION_SUFFIXES)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_both_ways_give_the_same_bits(ctx, monkeypatch, dtype):
    from minml_b200 import backend as B
    gen = torch.Generator(device="cuda").manual_seed(1)

    def n(*shape, scale=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)
    tokens, embed, hidden, vocab = 90, 64, 72, 300
    x, ext, dy, w, b = n(tokens, embed), n(tokens, embed), n(tokens, embed), n(embed), n(embed)
    w1, w2, wv = n(2 * hidden, embed, scale=0.1), n(embed, hidden, scale=0.1), n(vocab, embed, scale=0.1)
    targets = torch.randint(-1, vocab, (tokens,), device="cuda", generator=gen, dtype=torch.int32)
    weights = torch.rand(tokens, device="cuda", generator=gen)

    def everything():
        f32 = dict(device="cuda", dtype=torch.float32)
        y, dx, y2, dx2, dx3 = (x.clone() for _ in range(5))
        stats, saved, loss, lse, dw, db = torch.empty((tokens, 2), **f32), torch.empty((tokens, 2 * hidden), **f32), torch.empty(tokens, **f32), torch.empty(tokens, **f32), w.float().clone(), b.float().clone()
        dw1, dw2, dwv = w1.clone(), w2.clone(), wv.clone()
        ws = torch.empty(max(B.layernormBackwardGetWorkspaceSize(ctx, x.shape), B.gatedFeedForwardGetWorkspaceSize(ctx, x.shape, w1.shape, dtype, True),
                             B.softmaxCrossEntropyGetWorkspaceSize(ctx, x.shape, wv.shape, dtype, True)), device="cuda", dtype=torch.uint8)
        torch.cuda.synchronize()
        B.layernormForwardTraining(ctx, x, y, w, b, stats, ext)
        B.layernormBackward(ctx, x, dy, dx, w, stats, dw, db, ext=ext, beta_dx=0.5, beta_dw=-2.0, workspace=ws)
        B.gatedFeedForwardForward(ctx, x, w1, w2, y2, "gelu", beta=0.25, saved=saved, workspace=ws)
        B.gatedFeedForwardBackward(ctx, x, w1, w2, dy, dx2, dw1, dw2, "gelu", saved=saved, beta_dx=1.5, beta_dw=0.75, workspace=ws)
        B.softmaxCrossEntropyForward(ctx, x, wv, targets, loss, lse, ws)
        B.softmaxCrossEntropyBackward(ctx, x, wv, targets, lse, dx3, dwv, 8.0, row_weights=weights, beta_dx=0.5, beta_dw=3.0, workspace=ws)
        ctx.synchronize()
        return y, stats, dx, dw, db, y2, dx2, dw1, dw2, loss, lse, dx3, dwv
    one = everything()
    monkeypatch.setattr(B, "_binding", B.CtypesCalls())
    assert all(torch.equal(p, q) for p, q in zip(one, everything()))
    with pytest.raises(B.BackendError, match="needs a workspace"):
        B.gatedFeedForwardForward(ctx, x, w1, w2, x.clone())
