"""The token embedding, dropout, layer norm and masked attention on the CPU: the float64 definitions the GPU tests compare
with (against differences and published values), the torch formulation, and every refusal of the Python layer and of the C
entry points (no kernel is launched)."""
from __future__ import annotations

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import orda_ce_kernel as orda
from orda_ce_kernel import _native
from orda_ce_kernel.ops._random import kept_factors
from tests._layers import check
from tests._step import attention64, dropout64, embedding64, kept, norm64, philox, seen

ROOT = Path(__file__).resolve().parents[1]


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale


# ------------------------------------------------------------------- definitions
def test_philox_against_its_authors_values():
    """The known answers that its authors publish for 10 rounds."""
    ones = (1 << 64) - 1
    assert philox(0, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox(ones, ones, ones) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox(0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


@pytest.mark.parametrize("shape,p,seed,site", [((3, 7), 0.3, 5, 0), ((40,), 0.5, (1 << 64) - 3, (1 << 63) + 9), ((2, 8), 1.0, 1, 2),
                                               ((9, 3), 0.0, 0, 0), ((1,), 1e-6, 3, 1)])
def test_kept_elements(shape, p, seed, site):
    want = kept(shape, p, seed, site)
    assert torch.equal(kept_factors(shape, p, seed, None, site, torch.device("cpu")).double(), want.float().double())
    as_tensor = torch.tensor([seed - (1 << 64) if seed >> 63 else seed])
    assert torch.equal(kept_factors(shape, p, 0, as_tensor, site, torch.device("cpu")).double(), want.float().double())


def differences(value, grads, tensors, seed=3):
    """Gradients' products with random directions against central differences; the truncation is below h^2 times the third
    derivative along the direction (below 1e4 here)."""
    h, g = 1e-5, torch.Generator().manual_seed(seed)
    for name, t in tensors.items():
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        hi, lo = value({**tensors, name: t + h * d}), value({**tensors, name: t - h * d})
        assert abs(float(hi - lo) / (2 * h) - float((grads[name][0] * d).sum())) < 1e4 * h * h + 1e-7, name


def test_gradients_of_the_definitions_against_differences():
    F = torch.float32
    dy, ds, keep = randn(4, 6, seed=1), randn(4, 6, seed=2), kept((4, 6), 0.3, 9)
    t = {"x": randn(4, 6, seed=3), "residual": randn(4, 6, seed=4), "w": randn(6, seed=5), "bias": randn(6, seed=6)}

    def norm(a):
        out = norm64(F, **a, keep=keep)
        return (out["y"][0] * dy).sum() + (out["s"][0] * ds).sum()

    differences(norm, norm64(F, **t, keep=keep, dy=dy, ds=ds), t)
    u = {n: t[n] for n in ("x", "w")}
    differences(lambda a: (norm64(F, **a)["y"][0] * dy).sum(), norm64(F, **u, dy=dy), u)
    u = {n: t[n] for n in ("x", "residual")}
    differences(lambda a: (dropout64(F, a["x"], keep, a["residual"])["y"][0] * dy).sum(), dropout64(F, **u, keep=keep, dy=dy), u)
    ids, w = torch.tensor([2, 0, 2, -100]), {"w": randn(5, 6, seed=7)}
    differences(lambda a: (embedding64(F, F, ids, a["w"], 1.7)["y"][0] * dy).sum(), embedding64(F, F, ids, **w, scale=1.7, dy=dy), w)
    q = {"q": randn(2, 5, 4, 3, seed=8), "k": randn(2, 5, 2, 3, seed=9), "v": randn(2, 5, 2, 3, seed=10)}
    do = randn(2, 5, 4, 3, seed=11)
    for kw in (dict(), dict(causal=False, softcap=1.5), dict(slopes=torch.tensor([0.5, 0.1, 1.0, 0.0], dtype=torch.float64)),
               dict(documents=torch.tensor([[0, 0, 3, 3, -1], [1, 2, 2, 1, 1]]), prefix=torch.tensor([2, 4]), softcap=4.0)):
        differences(lambda a, kw=kw: (attention64(torch.float16, **a, **kw)["y"][0] * do).sum(),
                    attention64(torch.float16, **q, **kw, dy=do), q)


def test_masks_by_hand():
    docs = torch.tensor([[0, 0, 1, -1]])
    assert seen(1, 4, True, docs, torch.tensor([2])).int().tolist() == [[[1, 1, 0, 0], [1, 1, 0, 0], [0, 0, 1, 0], [0, 0, 0, 0]]]
    assert seen(1, 3, True, None, torch.tensor([-5])).int().tolist() == [[[1, 0, 0], [1, 1, 0], [1, 1, 1]]]


# ------------------------------------------------------------------- torch formulation
def test_torch_formulation_and_its_gradients():
    """In fp32 within the kernels' bounds."""
    F = torch.float32
    dy, ds = randn(4, 9, seed=1).float(), randn(4, 9, seed=2).float()
    t = {"x": randn(4, 9, seed=3), "residual": randn(4, 9, seed=4), "w": randn(9, seed=5), "bias": randn(9, seed=6)}
    leaves = {n: v.float().requires_grad_(True) for n, v in t.items()}
    wide = {n: v.detach().double() for n, v in leaves.items()}
    y, s = orda.layer_norm(leaves["x"], leaves["w"], leaves["bias"], leaves["residual"], p=0.25, seed=7, site=3)
    got = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), (dy, ds))))
    check({"y": y, "s": s, **got}, norm64(F, **wide, keep=kept((4, 9), 0.25, 7, 3), dy=dy.double(), ds=ds.double()))
    y = orda.counter_dropout(leaves["x"], 0.25, leaves["residual"], seed=7, site=3)
    got = dict(zip(("x", "residual"), torch.autograd.grad(y, (leaves["x"], leaves["residual"]), dy)))
    check({"y": y, **got}, dropout64(F, wide["x"], kept((4, 9), 0.25, 7, 3), wide["residual"], dy.double()))
    ids, w = torch.tensor([[2, 0], [2, -100]], dtype=torch.int32), randn(5, 9, seed=8).float().requires_grad_(True)
    y = orda.token_embedding(ids, w, scale=3.0, padding_idx=0)
    (g,) = torch.autograd.grad(y, w, dy.view(2, 2, 9))
    check({"y": y, "w": g}, embedding64(F, F, ids.reshape(-1).long(), w.detach().double(), 3.0, 0, dy.double()))


@pytest.mark.parametrize("kw", [dict(), dict(causal=False), dict(softcap=2.0, slopes=torch.tensor([0.5, 0.25, 0.0, 1.0])),
                                dict(documents=torch.tensor([[0, 0, 1, 1, -1], [4, 4, 4, 4, 4]]), prefix=torch.tensor([3, 0]))])
def test_torch_attention(kw):
    t = {n: randn(2, 5, h, 6, seed=i).half().float() for i, (n, h) in enumerate((("q", 4), ("k", 2), ("v", 2)))}
    dy = randn(2, 5, 4, 6, seed=9).half().float()
    leaves = {n: v.requires_grad_(True) for n, v in t.items()}
    y = orda.masked_attention(**leaves, **kw)
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    wide = {n: v.detach().double() for n, v in leaves.items()}
    kw64 = {n: v.double() if n == "slopes" else v for n, v in kw.items()}
    check({"y": y, **got}, attention64(torch.float16, **wide, **kw64, dy=dy.double()))


def test_padding_may_hold_anything_in_torch():
    docs = torch.tensor([[0, 0, -1]])
    q = torch.randn(1, 3, 2, 4)
    q[0, 2] = math.nan
    leaf = q.clone().requires_grad_(True)
    y = orda.masked_attention(leaf, leaf, leaf, documents=docs)
    y.sum().backward()
    assert torch.equal(y[0, 2], torch.zeros(2, 4)) and torch.isfinite(leaf.grad).all() and not leaf.grad[0, 2].any()


def test_empty_tensors():
    x = torch.zeros(0, 4, requires_grad=True)
    w = torch.ones(4, requires_grad=True)
    y, s = orda.layer_norm(x, w, None, torch.zeros(0, 4), p=0.5, seed=1)
    (y.sum() + s.sum()).backward()
    assert y.shape == s.shape == (0, 4) and not w.grad.any()
    assert orda.counter_dropout(x, 0.5, seed=2).shape == (0, 4)
    e = torch.ones(3, 4, requires_grad=True)
    y = orda.token_embedding(torch.zeros(2, 0, dtype=torch.int64), e)
    y.sum().backward()
    assert y.shape == (2, 0, 4) and not e.grad.any()
    assert orda.masked_attention(*(torch.zeros(2, 0, 1, 8) for _ in range(3))).shape == (2, 0, 1, 8)


def test_seeds_come_from_torchs_generator():
    x = torch.ones(64)
    torch.manual_seed(5)
    a, b = orda.counter_dropout(x, 0.5), orda.counter_dropout(x, 0.5)
    torch.manual_seed(5)
    assert torch.equal(a, orda.counter_dropout(x, 0.5)) and not torch.equal(a, b)
    assert not torch.equal(orda.counter_dropout(x, 0.5, seed=1), orda.counter_dropout(x, 0.5, seed=1, site=1))
    assert torch.equal(orda.counter_dropout(x, 0.0), x) and not orda.counter_dropout(x * math.inf, 1.0).any()


# ------------------------------------------------------------------- refusals
X, W1, IDS = torch.zeros(3, 8), torch.zeros(8), torch.zeros(3, dtype=torch.int64)
Q = torch.zeros(2, 3, 4, 8)


@pytest.mark.parametrize("call,error,match", [
    (lambda: orda.token_embedding(IDS.float(), X), ValueError, "ids must be an int32 or int64"),
    (lambda: orda.token_embedding([1], X), ValueError, "ids must be an int32 or int64"),
    (lambda: orda.token_embedding(IDS, W1), ValueError, "weight must have shape"),
    (lambda: orda.token_embedding(IDS, torch.zeros(0, 8)), ValueError, "weight must have shape"),
    (lambda: orda.token_embedding(IDS, torch.zeros(3, 0)), ValueError, "features > 0"),
    (lambda: orda.token_embedding(IDS, X.double()), ValueError, "must be bfloat16"),
    (lambda: orda.token_embedding(IDS, X.to("meta")), ValueError, "ids are on"),
    (lambda: orda.token_embedding(IDS, X, scale=math.inf), ValueError, "scale must be finite"),
    (lambda: orda.token_embedding(IDS, X, padding_idx=3), ValueError, "padding_idx must be in"),
    (lambda: orda.token_embedding(IDS, X, padding_idx=-1), ValueError, "padding_idx must be in"),
    (lambda: orda.token_embedding(IDS, X, backend="hip"), RuntimeError, "requires the HIP extension"),
    (lambda: orda.counter_dropout(X, 1.5), ValueError, "p must be in"),
    (lambda: orda.counter_dropout(X, math.nan), ValueError, "p must be in"),
    (lambda: orda.counter_dropout(X, 0.5, torch.zeros(3, 7)), ValueError, "residual must have shape"),
    (lambda: orda.counter_dropout(X, 0.5, seed=-1), ValueError, "seed must be"),
    (lambda: orda.counter_dropout(X, 0.5, seed=1 << 64), ValueError, "seed must be"),
    (lambda: orda.counter_dropout(X, 0.5, seed=True), ValueError, "seed must be"),
    (lambda: orda.counter_dropout(X, 0.5, seed=torch.zeros(2, dtype=torch.int64)), ValueError, "seed tensor"),
    (lambda: orda.counter_dropout(X, 0.5, seed=torch.zeros(1)), ValueError, "seed tensor"),
    (lambda: orda.counter_dropout(X, 0.5, seed=torch.zeros(1, dtype=torch.int64, device="meta")), ValueError, "seed tensor"),
    (lambda: orda.counter_dropout(X, 0.5, site=-1), ValueError, "site must be"),
    (lambda: orda.counter_dropout(X.long(), 0.5), ValueError, "must be bfloat16"),
    (lambda: orda.counter_dropout(X, 0.5, backend="hip"), RuntimeError, "requires the HIP extension"),
    (lambda: orda.layer_norm(X, torch.zeros(7)), ValueError, "weight must have shape"),
    (lambda: orda.layer_norm(X, W1, torch.zeros(1, 8)), ValueError, "bias must have shape"),
    (lambda: orda.layer_norm(X, W1, None, torch.zeros(8)), ValueError, "residual must have shape"),
    (lambda: orda.layer_norm(X, W1, eps=-1.0), ValueError, "eps must be"),
    (lambda: orda.layer_norm(X, W1, eps=math.nan), ValueError, "eps must be"),
    (lambda: orda.layer_norm(X, W1, p=0.5), ValueError, "p > 0 needs residual"),
    (lambda: orda.layer_norm(X, W1, None, X, p=2.0), ValueError, "p must be in"),
    (lambda: orda.layer_norm(torch.zeros(3, 0), torch.zeros(0)), ValueError, "features > 0"),
    (lambda: orda.layer_norm(X, W1.to("meta")), ValueError, "weight is on meta"),
    (lambda: orda.layer_norm(X, W1, backend="hip"), RuntimeError, "requires the HIP extension"),
    (lambda: orda.masked_attention(Q[0], Q, Q), ValueError, "q must have shape"),
    (lambda: orda.masked_attention(Q, Q[:, :, :3], Q[:, :, :3]), ValueError, "kv_heads a divisor"),
    (lambda: orda.masked_attention(Q, Q[:, :, :0], Q[:, :, :0]), ValueError, "kv_heads a divisor"),
    (lambda: orda.masked_attention(Q, Q[:, :2], Q[:, :2]), ValueError, "k must have shape"),
    (lambda: orda.masked_attention(Q, Q, Q[..., :4]), ValueError, "v must have shape"),
    (lambda: orda.masked_attention(Q, Q, Q, slopes=torch.zeros(3)), ValueError, "slopes must have shape"),
    (lambda: orda.masked_attention(Q, Q, Q, slopes=torch.zeros(4, requires_grad=True)), ValueError, "slopes are constants"),
    (lambda: orda.masked_attention(Q, Q, Q, documents=torch.zeros(2, 3)), ValueError, "documents must be an int32"),
    (lambda: orda.masked_attention(Q, Q, Q, documents=torch.zeros(3, 2, dtype=torch.int32)), ValueError, "documents must have shape"),
    (lambda: orda.masked_attention(Q, Q, Q, prefix=torch.zeros(3, dtype=torch.int32)), ValueError, "prefix must have shape"),
    (lambda: orda.masked_attention(Q, Q, Q, softcap=-1.0), ValueError, "softcap must be"),
    (lambda: orda.masked_attention(Q, Q, Q, softcap=math.inf), ValueError, "softcap must be"),
    (lambda: orda.masked_attention(Q, Q, Q, scale=math.nan), ValueError, "scale must be finite"),
    (lambda: orda.masked_attention(Q, Q.to("meta"), Q), ValueError, "k is on meta"),
    (lambda: orda.masked_attention(Q, Q, Q, backend="hip"), RuntimeError, "requires the HIP extension"),
])
def test_python_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


# ------------------------------------------------------------------- C ABI
VERSION = _native.ABI_VERSION


def message():
    return _native.library().orda_last_error().decode()


def embedding(**kw):
    return _native.Embedding(**{**dict(abi_version=VERSION, dtype=0, out_dtype=0, wide_ids=1, tokens=4, vocab=10, hidden=8, ldw=8,
                                       ldg=8, padding_idx=-1, scale=1.0), **kw})


def norm(**kw):
    return _native.LayerNorm(**{**dict(abi_version=VERSION, dtype=0, param_dtype=0, eps=1e-5, rows=4, cols=8, ldx=8, ldr=8, ld_s=8,
                                       ld_dy=8, ld_ds=8), **kw})


def rows(**kw):
    return _native.RowsProblem(**{**dict(abi_version=VERSION, dtype=0, rows=4, cols=8, ldx=8, ldr=8), **kw})


def drop(p=0.5, **kw):
    return _native.Dropout(p=p, **kw)


I3 = ctypes.c_int64 * 3


def attention(**kw):
    dense, kv = I3(5 * 4 * 16, 4 * 16, 16), I3(5 * 2 * 16, 2 * 16, 16)
    return _native.Attention(**{**dict(abi_version=VERSION, dtype=0, heads=4, kv_heads=2, head_dim=16, causal=1, batch=3, length=5,
                                       q_stride=dense, k_stride=kv, v_stride=kv, g_stride=dense, documents_stride=5, scale=0.25,
                                       softcap=0.0), **kw})


def refused(rc, code, text):
    assert rc == code and text in message(), (rc, message())


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=3), "abi_version"), (dict(dtype=3), "dtype"), (dict(out_dtype=-1), "out_dtype"), (dict(reserved=1), "reserved"),
    (dict(tokens=0), "tokens"), (dict(tokens=(1 << 30) + 1), "tokens"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 31) - 1), "vocab"),
    (dict(hidden=0), "hidden"), (dict(hidden=(1 << 21) + 1), "hidden"), (dict(scale=math.inf), "scale"),
])
def test_embedding_problems_are_refused(kw, match):
    lib, p = _native.library(), ctypes.byref(embedding(**kw))
    assert lib.orda_embedding_workspace_bytes(p) == 0 and match in message()
    refused(lib.orda_embedding_forward(p, 256, 256, 256, None), -1, match)
    refused(lib.orda_embedding_backward(p, 256, 256, 256, 256, 1 << 30, None), -1, match)


def test_embedding_operands_are_checked():
    lib, p = _native.library(), ctypes.byref(embedding())
    f, b = lib.orda_embedding_forward, lib.orda_embedding_backward
    refused(f(None, 256, 256, 256, None), -1, "NULL")
    refused(f(p, None, 256, 256, None), -1, "ids")
    refused(f(p, 260, 256, 256, None), -1, "ids")
    refused(f(p, 256, 257, 256, None), -1, "weight")
    refused(f(p, 256, 256, None, None), -1, "y is required")
    refused(f(ctypes.byref(embedding(ldw=7)), 256, 256, 256, None), -1, "ldw")
    refused(f(ctypes.byref(embedding(ldw=(1 << 22) + 1)), 256, 256, 256, None), -1, "ldw")
    refused(b(ctypes.byref(embedding(ldg=7)), 256, 256, 256, 256, 1 << 30, None), -1, "ldg")
    refused(b(p, 256, 256, 264, 256, 1 << 30, None), -1, "grad_weight")
    refused(b(p, 256, None, 256, 256, 1 << 30, None), -1, "grad_output")
    need = lib.orda_embedding_workspace_bytes(p)
    refused(b(p, 256, 256, 256, 256, need - 1, None), -2, "workspace")
    refused(b(p, 256, 256, 256, None, need, None), -2, "workspace")


def test_dropout_calls_are_checked():
    lib, d = _native.library(), ctypes.byref(drop())
    f = lib.orda_dropout_add
    refused(f(None, d, 256, None, 256, None), -1, "NULL")
    refused(f(ctypes.byref(rows()), None, 256, None, 256, None), -1, "NULL")
    for kw, text in ((dict(abi_version=0), "abi_version"), (dict(dtype=5), "dtype"), (dict(rows=0), "rows"), (dict(cols=0), "cols"),
                     (dict(rows=1 << 20, cols=1 << 23), "2^42"), (dict(ldx=7), "ldx"), (dict(ldx=(1 << 22) + 1), "ldx")):
        refused(f(ctypes.byref(rows(**kw)), d, 256, None, 256, None), -1, text)
    refused(f(ctypes.byref(rows(ldr=7)), d, 256, 256, 256, None), -1, "ldr")
    p = ctypes.byref(rows())
    refused(f(p, d, 257, None, 256, None), -1, "x must be aligned")
    refused(f(p, d, None, None, 256, None), -1, "x is required")
    refused(f(p, d, 256, None, None, None), -1, "y is required")
    for q in (-0.1, 1.1, math.nan):
        refused(f(p, ctypes.byref(drop(q)), 256, None, 256, None), -1, "p must be in")
    refused(f(p, ctypes.byref(drop(0.5, seed_on_device=260)), 256, None, 256, None), -1, "seed_on_device")


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=3), "abi_version"), (dict(dtype=3), "dtype"), (dict(param_dtype=1), "param_dtype"), (dict(dtype=2, param_dtype=0), "param_dtype"),
    (dict(rows=0), "rows"), (dict(rows=(1 << 30) + 1), "rows"), (dict(cols=0), "cols"), (dict(cols=(1 << 21) + 1), "cols"),
    (dict(eps=-1.0), "eps"), (dict(eps=math.inf), "eps"),
])
def test_layer_norm_problems_are_refused(kw, match):
    lib, p = _native.library(), ctypes.byref(norm(**kw))
    assert lib.orda_layer_norm_workspace_bytes(p) == 0 and match in message()
    refused(lib.orda_layer_norm_forward(p, None, 256, None, 256, None, 256, None, None, None), -1, match)
    refused(lib.orda_layer_norm_backward(p, None, 256, None, 256, 256, 256, None, 256, None, None, None, 256, 1 << 30, None), -1, match)


def test_layer_norm_operands_are_checked():
    lib, p = _native.library(), ctypes.byref(norm())
    f, b = lib.orda_layer_norm_forward, lib.orda_layer_norm_backward
    big = 1 << 30
    refused(f(None, None, 256, None, 256, None, 256, None, None, None), -1, "NULL")
    refused(f(p, None, None, None, 256, None, 256, None, None, None), -1, "x is required")
    refused(f(p, None, 256, 257, 256, None, 256, None, None, None), -1, "residual must be aligned")
    refused(f(p, None, 256, None, None, None, 256, None, None, None), -1, "weight is required")
    refused(f(p, None, 256, None, 256, 257, 256, None, None, None), -1, "bias must be aligned")
    refused(f(p, None, 256, None, 256, None, 256, None, 260, None), -1, "stats must be aligned")
    refused(f(ctypes.byref(norm(ldx=7)), None, 256, None, 256, None, 256, None, None, None), -1, "ldx")
    refused(f(ctypes.byref(norm(ldr=7)), None, 256, 256, 256, None, 256, None, None, None), -1, "ldr")
    refused(f(p, ctypes.byref(drop(3.0)), 256, 256, 256, None, 256, None, None, None), -1, "p must be in")
    refused(b(p, None, None, None, 256, 256, 256, None, 256, None, None, None, 256, big, None), -1, "s is required")
    refused(b(p, None, 256, None, None, 256, 256, None, 256, None, None, None, 256, big, None), -1, "stats is required")
    refused(b(p, None, 256, None, 256, 256, None, None, 256, None, None, None, 256, big, None), -1, "grad_y is required")
    refused(b(p, None, 256, 256, 256, 256, 256, None, 256, None, None, None, 256, big, None), -1, "computed again only")
    refused(b(ctypes.byref(norm(ld_s=7)), None, 256, None, 256, 256, 256, None, 256, None, None, None, 256, big, None), -1, "ld_s")
    refused(b(ctypes.byref(norm(ld_dy=7)), None, 256, None, 256, 256, 256, None, 256, None, None, None, 256, big, None), -1, "ld_dy")
    refused(b(ctypes.byref(norm(ld_ds=7)), None, 256, None, 256, 256, 256, 256, 256, None, None, None, 256, big, None), -1, "ld_ds")
    refused(b(p, None, 256, None, 256, 256, 256, None, 256, 256, None, None, 256, big, None), -1, "are one")
    need = lib.orda_layer_norm_workspace_bytes(p)
    refused(b(p, None, 256, None, 256, 256, 256, None, 256, None, 256, None, 256, need - 1, None), -2, "workspace")
    refused(b(p, None, 256, None, 256, 256, 256, None, None, None, None, 256, None, need, None), -2, "workspace")


@pytest.mark.parametrize("kw,match", [
    (dict(abi_version=3), "abi_version"), (dict(dtype=2), "bf16 or fp16"), (dict(length=0), "length"), (dict(length=(1 << 24) + 1), "length"),
    (dict(batch=0), "batch"), (dict(batch=65536), "batch"), (dict(heads=0), "heads"), (dict(kv_heads=0), "kv_heads"),
    (dict(kv_heads=3), "multiple of kv_heads"), (dict(kv_heads=8), "kv_heads"), (dict(head_dim=12), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(causal=2), "causal"), (dict(scale=math.nan), "scale"), (dict(softcap=-1.0), "softcap"),
    (dict(q_stride=I3(320, 64, 12)), "strides of q"), (dict(k_stride=I3(160, -32, 16)), "strides of k"),
    (dict(v_stride=I3(160, (1 << 22) + 8, 16)), "2^22"), (dict(batch=60000, length=1 << 24), "workgroups"),
])
def test_attention_problems_are_refused(kw, match):
    lib, p = _native.library(), ctypes.byref(attention(**kw))
    assert lib.orda_attention_saved_bytes(p, 1, 1) == 0 and match in message()
    assert lib.orda_attention_workspace_bytes(p) == 0 and match in message()
    refused(lib.orda_attention_forward(p, 256, 256, 256, None, None, None, 256, 256, 1 << 30, 1, None), -1, match)


def test_attention_operands_are_checked():
    lib, p, big = _native.library(), ctypes.byref(attention()), 1 << 30
    f, b = lib.orda_attention_forward, lib.orda_attention_backward
    good = [p, 256, 256, 256, None, None, None, 256, 256, big, 1, None]

    def forward(**at):
        a = list(good)
        for i, v in at.items():
            a[int(i[1:])] = v
        return f(*a)

    refused(forward(_0=None), -1, "NULL")
    for i, name in ((1, "q"), (2, "k"), (3, "v"), (7, "out")):
        refused(forward(**{f"_{i}": None}), -1, f"{name} is required")
        refused(forward(**{f"_{i}": 264}), -1, f"{name} must be aligned")
    for i, name in ((4, "slopes"), (5, "documents"), (6, "prefix")):
        refused(forward(**{f"_{i}": 258}), -1, f"{name} must be aligned")
    refused(forward(_0=ctypes.byref(attention(documents_stride=4)), _5=256), -1, "documents_stride")
    refused(forward(_8=None), -2, "saved")
    refused(forward(_8=264), -1, "saved must be aligned")
    refused(forward(_9=lib.orda_attention_saved_bytes(p, 0, 1) - 1), -2, "saved")
    refused(forward(_9=lib.orda_attention_saved_bytes(p, 1, 0) - 1, _5=256, _10=0), -2, "saved")
    good = [p, 256, 256, 256, None, 0, None, 256, 256, big, 256, 256, 256, 256, 256, big, None]

    def backward(**at):
        a = list(good)
        for i, v in at.items():
            a[int(i[1:])] = v
        return b(*a)

    for i, name in ((1, "q"), (7, "out"), (10, "grad_output")):
        refused(backward(**{f"_{i}": None}), -1, f"{name} is required")
    for i, name in ((11, "grad_q"), (12, "grad_k"), (13, "grad_v")):
        refused(backward(**{f"_{i}": 264}), -1, f"{name} must be aligned")
    refused(backward(_0=ctypes.byref(attention(g_stride=I3(320, 60, 16)))), -1, "strides of grad_output")
    refused(backward(_8=None), -2, "saved")
    refused(backward(_15=lib.orda_attention_workspace_bytes(p) - 1), -2, "workspace")


def test_struct_layouts_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("no gcc")
    names = {"orda_embedding_t": _native.Embedding, "orda_dropout_t": _native.Dropout, "orda_rows_problem_t": _native.RowsProblem,
             "orda_layer_norm_t": _native.LayerNorm, "orda_attention_t": _native.Attention}
    lines = [f'printf("{t}.{f} %zu\\n", offsetof({t}, {f}));' for t, c in names.items() for f, _ in c._fields_]
    lines += [f'printf("{t} %zu\\n", sizeof({t}));' for t in names]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "orda_ce.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "probe"
    subprocess.run([gcc, "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for t, c in names.items():
        assert int(got[t]) == ctypes.sizeof(c)
        assert all(int(got[f"{t}.{f}"]) == getattr(c, f).offset for f, _ in c._fields_)
