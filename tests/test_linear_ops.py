"""CPU checks of dropout, the linear layer and the loss head: the generator against its published
known answers, and the refusals that no kernel has to see (the C ABI's and the wrappers')."""
import ast
import ctypes
import inspect
import os
import re

import numpy as np
import pytest

import linear_ops_ref as ref

torch = pytest.importorskip("torch")

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


@pytest.mark.parametrize("ctr,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((ref.LOW,) * 4, (ref.LOW,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_known_answers(ctr, key, want):
    """The known-answer vectors published with the generator."""
    assert tuple(int(v) for v in ref.philox(ctr, key)) == want


def test_mask_frequency():
    """Kept share within 5 standard deviations of the quantised probability."""
    n = 512 * 1024
    for p in (0.1, 0.5):
        keep, scale = ref.keep_mask(5, 11, 512, 1024, p)
        q = 1 / scale
        assert abs(keep.double().mean().item() - q) < 5 * np.sqrt(q * (1 - q) / n)


def _written_out_step():
    """The sites of the training step that INTEGRATION.md writes out, and what it adds to the offset."""
    from llmgpu import ops
    md = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    code, = [c for c in re.findall(r"```python\n(.*?)```", md, re.S) if "dropout_fwd" in c]
    sites, adds = set(), []
    for n in ast.walk(ast.parse(code)):
        if isinstance(n, ast.Call) and ast.unparse(n.func).startswith("ops."):
            sig = inspect.signature(getattr(ops, n.func.attr))
            a = sig.bind(*n.args, **{k.arg: k.value for k in n.keywords}).arguments
            if "rng" in a:
                sites.add(ast.literal_eval(a["site"]) if "site" in a else 0)
        elif isinstance(n, ast.AugAssign) and ast.unparse(n.target) == "rng[1]":
            adds.append(ast.literal_eval(n.value))
    return sites, adds


def test_no_mask_of_the_written_out_step_comes_back():
    """A mask goes by offset + site: the steps' sums (and so the masks of one shape) are all different."""
    sites, adds = _written_out_step()
    assert sites == {0, 1} and len(adds) == 1 and adds[0] > max(sites)
    masks = [ref.keep_mask(3, step * adds[0] + s, 16, 64, 0.5)[0] for step in range(4) for s in sites]
    assert not any(torch.equal(a, b) for i, a in enumerate(masks) for b in masks[:i])


def test_sites_and_offsets_add_up():
    """What that rule is for: site 1 of a step has the mask of site 0 at the next offset."""
    a, b = ref.keep_mask(3, 5 + 1, 16, 64, 0.5)[0], ref.keep_mask(3, 6 + 0, 16, 64, 0.5)[0]
    assert torch.equal(a, b)


def _lib():
    from llmgpu import load
    return load()


P = 0x1000  # a made-up device address: every call below is refused before it is used
REFUSED = (-1, -3)  # the checks' own codes; a launch or a tensor map that failed has others


@pytest.mark.parametrize("bad", [dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(rows=-1),
                                 dict(cols=(1 << 30) + 1), dict(x=None), dict(out=None),
                                 dict(rng=None), dict(ldx=7), dict(ldo=7), dict(resid=P, ldr=7)])
def test_dropout_refusals(bad):
    a = dict(x=P, ldx=8, resid=None, ldr=0, out=P, ldo=8, rows=4, cols=8, p=0.5, rng=P)
    a.update(bad)
    assert _lib().llmgpu_op_dropout(a["x"], 0, a["ldx"], a["resid"], a["ldr"], a["out"], 0, a["ldo"],
                                    a["rows"], a["cols"], a["p"], a["rng"], 0, None) in REFUSED


@pytest.mark.parametrize("bad", [dict(x_f32=1), dict(out_f32=1), dict(ldx=16), dict(ldo=16),
                                 dict(x=2 * P, resid=P, ldr=16)])
def test_dropout_over_another_layout_is_refused(bad):
    """out may be x or resid where every element keeps its place: one type, one row stride."""
    a = dict(x=P, x_f32=0, ldx=8, resid=None, ldr=0, out_f32=0, ldo=8)
    a.update(bad)
    assert _lib().llmgpu_op_dropout(a["x"], a["x_f32"], a["ldx"], a["resid"], a["ldr"], P, a["out_f32"],
                                    a["ldo"], 4, 8, 0.5, P, 0, None) in REFUSED


@pytest.mark.parametrize("M", [4, 40])
def test_linear_over_a_residual_of_another_stride_is_refused(M):
    assert _lib().llmgpu_op_linear_fwd(P, 16, P, 16, 0, None, 0, 0.0, None, 0, 2 * P, 24, None, 0, 2 * P, 0,
                                       16, M, 16, 16, None, None, None) in REFUSED


def test_empty_calls_do_nothing():
    lib = _lib()
    assert lib.llmgpu_op_dropout(None, 0, 8, None, 0, None, 0, 8, 0, 8, 0.5, None, 0, None) == 0
    assert lib.llmgpu_op_linear_fwd(None, 8, P, 8, 0, None, 0, 0.0, None, 0, None, 0, None, 0, None,
                                    0, 8, 0, 8, 8, None, None, None) == 0
    assert lib.llmgpu_op_linear_ce_fwd(None, 8, P, 8, 0, None, 0, 8, 8, 0.0, None, None, None, None,
                                       None) == 0
    assert lib.llmgpu_op_linear_bwd_work(0, 8, 8) == 0
    assert lib.llmgpu_op_linear_ce_fwd_work(0, 8) == 0
    assert lib.llmgpu_op_linear_ce_bwd_work(0, 8, 8, 0) == 0


@pytest.mark.parametrize("bad", [dict(act=4), dict(act=-1), dict(K=0), dict(N=0), dict(M=-1),
                                 dict(p=2.0), dict(p=0.5), dict(x=None), dict(w=None),
                                 dict(out=None), dict(ldx=8), dict(ldw=8), dict(ldo=8),
                                 dict(resid=P, ldr=8), dict(pre=P, ld_pre=8), dict(x=P + 2),
                                 dict(ldx=17), dict(w=P + 8), dict(w_mn=1, ldw=8),
                                 dict(work=P + 8)])
def test_linear_fwd_refusals(bad):
    a = dict(x=P, ldx=16, w=P, ldw=16, w_mn=0, act=0, p=0.0, resid=None, ldr=0, pre=None, ld_pre=0,
             out=P, ldo=16, M=4, N=16, K=16, work=P)
    a.update(bad)
    rc = _lib().llmgpu_op_linear_fwd(a["x"], a["ldx"], a["w"], a["ldw"], a["w_mn"], None, a["act"],
                                     a["p"], None, 0, a["resid"], a["ldr"], a["pre"], a["ld_pre"],
                                     a["out"], 0, a["ldo"], a["M"], a["N"], a["K"], a["work"], None,
                                     None)
    assert rc in REFUSED


@pytest.mark.parametrize("bad", [dict(act=5), dict(act=1, pre=None), dict(p=0.5), dict(dy=None),
                                 dict(work=None), dict(work=P + 8), dict(lddy=8), dict(ldx=8),
                                 dict(lddx=8), dict(lddw=8), dict(acc=1), dict(N=0), dict(K=-1)])
def test_linear_bwd_refusals(bad):
    a = dict(dy=P, lddy=16, ldx=16, pre=None, act=0, p=0.0, lddx=16, lddw=16, acc=0, M=4, N=16, K=16,
             work=P)
    a.update(bad)
    rc = _lib().llmgpu_op_linear_bwd(a["dy"], 1, a["lddy"], P, a["ldx"], P, 16, 0, a["pre"], 16,
                                     a["act"], a["p"], None, 0, P, 0, a["lddx"], P, 0, a["lddw"], P,
                                     a["acc"], a["M"], a["N"], a["K"], a["work"], None, None)
    assert rc in REFUSED


def test_linear_bwd_refuses_a_workspace_off_16_bytes():
    """Where dy itself is the products' operand (bf16, no activation, dropout or bias gradient), the
    workspace holds the planes of the products split along K alone."""
    assert _lib().llmgpu_op_linear_bwd(P, 0, 16, P, 16, P, 16, 0, None, 0, 0, 0.0, None, 0, P, 0, 16,
                                       P, 0, 16, None, 0, 32, 16, 16, P + 8, None, None) in REFUSED


@pytest.mark.parametrize("bad", [dict(smoothing=1.0), dict(smoothing=-0.1), dict(V=0), dict(C=0),
                                 dict(V=(1 << 30) + 1), dict(targets=None), dict(work=None),
                                 dict(lse=None), dict(ldx=8), dict(ldw=8), dict(x=P + 2),
                                 dict(rows=-1)])
def test_loss_head_refusals(bad):
    a = dict(x=P, ldx=16, ldw=16, targets=P, rows=4, C=16, V=32, smoothing=0.0, lse=P, work=P)
    a.update(bad)
    lib = _lib()
    assert lib.llmgpu_op_linear_ce_fwd(a["x"], a["ldx"], P, a["ldw"], 0, a["targets"], a["rows"],
                                       a["C"], a["V"], a["smoothing"], P, a["lse"], a["work"], None,
                                       None) in REFUSED
    assert lib.llmgpu_op_linear_ce_bwd(a["x"], a["ldx"], P, a["ldw"], 0, a["targets"], a["lse"], None,
                                       1.0, a["rows"], a["C"], a["V"], a["smoothing"], P, 0, 16, P, 0,
                                       16, 0, 0, a["work"], None, None) in REFUSED


@pytest.mark.parametrize("bad", [dict(piece=100), dict(piece=-256), dict(acc=1), dict(lddx=8),
                                 dict(lddw=8)])
def test_loss_head_bwd_refusals(bad):
    a = dict(piece=0, acc=0, lddx=16, lddw=16)
    a.update(bad)
    lib = _lib()
    assert lib.llmgpu_op_linear_ce_bwd(P, 16, P, 16, 0, P, P, None, 1.0, 4, 16, 32, 0.0, P, 0,
                                       a["lddx"], P, 0, a["lddw"], a["acc"], a["piece"], P, None,
                                       None) in REFUSED
    if "piece" in bad:
        assert lib.llmgpu_op_linear_ce_bwd_work(4, 16, 32, bad["piece"]) < 0


@pytest.mark.parametrize("at", ["M", "N", "K"])
def test_sizes_past_2_30_are_refused(at):
    """Tile counts and column offsets are 32-bit: nothing is launched, and no workspace named."""
    big = (1 << 30) + 8
    d = dict(M=32, N=16, K=16)
    d[at] = big
    M, N, K = d["M"], d["N"], d["K"]
    lib, ld = _lib(), big
    assert lib.llmgpu_op_linear_fwd(P, ld, P, ld, 0, None, 0, 0.0, None, 0, None, 0, None, 0, P, 0, ld,
                                    M, N, K, P, None, None) in REFUSED
    assert lib.llmgpu_op_linear_bwd(P, 1, ld, P, ld, P, ld, 0, None, 0, 0, 0.0, None, 0, P, 0, ld, P, 0,
                                    ld, P, 0, M, N, K, P, None, None) in REFUSED
    assert lib.llmgpu_op_linear_ce_fwd(P, ld, P, ld, 0, P, M, K, N, 0.0, P, P, P, None, None) in REFUSED
    assert lib.llmgpu_op_linear_ce_bwd(P, ld, P, ld, 0, P, P, None, 1.0, M, K, N, 0.0, P, 0, ld, P, 0, ld,
                                       0, 0, P, None, None) in REFUSED
    assert lib.llmgpu_op_linear_fwd_work(M, N, K) == lib.llmgpu_op_linear_bwd_work(M, N, K) == 0
    assert lib.llmgpu_op_linear_ce_bwd_work(M, K, N, 0) == 0


def test_workspace_covers_any_piece():
    """The workspace holds at least the gradient of one piece and a copy of x; a piece past the
    vocabulary is the whole of it."""
    f = _lib().llmgpu_op_linear_ce_bwd_work
    for p in (256, 512, 2048, 4096, 8192):
        assert f(100, 64, 5000, p) >= 100 * (min(p, 5000) + 64) * 2
    assert f(100, 64, 5000, 8192) == f(100, 64, 5000, 1 << 20) == f(100, 64, 5000, 0)


def test_linear_forward_workspace():
    """Room for two f32 planes of the result at least where K is split, 0 where it is not; the
    backward's size is another, which may be smaller."""
    fwd, bwd = _lib().llmgpu_op_linear_fwd_work, _lib().llmgpu_op_linear_bwd_work
    for M, N, K in ((256, 512, 4096), (40, 130, 2101), (17, 8, 1 << 20)):
        assert fwd(M, N, K) >= 2 * M * N * 4
    assert bwd(256, 512, 4096) < fwd(256, 512, 4096)
    for M, N, K in ((16, 512, 4096), (256, 512, 512), (8192, 4096, 1024)):
        assert fwd(M, N, K) == 0


def test_block_call_refusals():
    """llmgpu_op_call: an unknown operator, no block, an integer past its argument's type, and the
    refusals of the calls themselves."""
    from llmgpu import ops
    lib = _lib()

    def call(name, *args):
        op, pack = ops._BLOCKS[name]
        return lib.llmgpu_op_call(op, pack(*args))
    drop = [P, 0, 8, 0, 0, P, 0, 8, 4, 8, P, 0, 0, 0.5]
    assert lib.llmgpu_op_call(0, None) == -1 and lib.llmgpu_op_call(99, b"\0" * 256) == -1
    assert call("llmgpu_op_dropout", *drop[:8], 0, *drop[9:]) == 0  # no rows
    for i, bad in ((0, 0), (2, 7), (8, 1 << 33), (9, (1 << 30) + 1), (10, 0), (13, 1.5)):
        assert call("llmgpu_op_dropout", *drop[:i], bad, *drop[i + 1:]) == -1
    fwd = [P, 16, P, 16, 0, 0, 0, 0, 0, 0, 0, 0, 0, P, 0, 16, 4, 16, 16, 0, 0, 0, 0.0]
    assert call("llmgpu_op_linear_fwd", *fwd[:16], 0, *fwd[17:]) == 0
    for i, bad in ((0, 0), (0, P + 2), (1, 8), (6, 4), (16, 1 << 40), (18, 0), (22, 2.0)):
        assert call("llmgpu_op_linear_fwd", *fwd[:i], bad, *fwd[i + 1:]) in REFUSED
    bwd = [P, 1, 16, P, 16, P, 16, 0, 0, 16, 0, 0, 0, P, 0, 16, P, 0, 16, P, 0, 4, 16, 16, P, 0, 0, 0.0]
    for i, bad in ((0, 0), (2, 8), (10, 1), (20, 1), (22, 1 << 32), (24, 0), (27, 0.5)):
        assert call("llmgpu_op_linear_bwd", *bwd[:i], bad, *bwd[i + 1:]) in REFUSED
    cef = [P, 16, P, 16, 0, P, 4, 16, 32, P, P, P, 0, 0, 0.0]
    for i, bad in ((0, 0), (5, 0), (6, -1), (8, 1 << 35), (11, 0), (14, 1.0)):
        assert call("llmgpu_op_linear_ce_fwd", *cef[:i], bad, *cef[i + 1:]) in REFUSED
    ceb = [P, 16, P, 16, 0, P, P, 0, 4, 16, 32, P, 0, 16, P, 0, 16, 0, 0, P, 0, 0, 1.0, 0.0]
    for i, bad in ((0, 0), (6, 0), (17, 1), (18, 100), (19, 0), (23, -0.5)):
        assert call("llmgpu_op_linear_ce_bwd", *ceb[:i], bad, *ceb[i + 1:]) in REFUSED


def test_error_word_refusals():
    assert _lib().llmgpu_op_error_word(None) != 0 and _lib().llmgpu_op_take_error(None) != 0


def test_wrappers_refuse_cpu_tensors():
    from llmgpu import ops
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.dropout_fwd(x, 0.5, rng)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.linear_fwd(x, w)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.linear_bwd(x, x, w)
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.linear_cross_entropy_fwd(x, w, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.linear_cross_entropy_bwd(x, w, torch.zeros(4, dtype=torch.int32), torch.zeros(4))
