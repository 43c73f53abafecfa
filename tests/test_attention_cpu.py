"""The attention library without a GPU: it loads and exports what include/pbattn.h
declares, refuses bad arguments before any launch, and its matrix results are read
late enough; the host API's refusals; the oracle against closed forms and
differences."""
import ctypes
import os
import re
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from oracle import attention as oa
from pseudobrain_amd import _lib, build
from pseudobrain_amd import attention as at
from tests import test_mfma_hazards as hazards

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "pbattn.h")
FAKE = 0x1000  # never dereferenced: every call below fails validation first


def declared_functions():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(pbattn_\w+)\s*\(", text)))


def test_header_library_and_signatures_agree():
    assert declared_functions() == sorted(_lib.ATTN_SIGNATURES)
    lib = _lib.attn_lib()
    for name in declared_functions():
        assert isinstance(getattr(lib, name), ctypes._CFuncPtr), name
    text = open(HEADER).read()
    assert lib.pbattn_abi_version() == _lib.ATTN_ABI_VERSION
    assert re.search(r"#define PBATTN_ABI_VERSION (\d+)", text).group(1) == str(_lib.ATTN_ABI_VERSION)
    assert re.search(r"#define PBATTN_MAX_DRAFT (\d+)", text).group(1) == str(at.MAX_DRAFT)


def strides(*values):
    return (ctypes.c_int64 * len(values))(*values)


QKV = (8192, 512, 128) * 3


def fwd(**over):
    args = dict(q=FAKE, k=FAKE, v=FAKE, dtype=1, strides=strides(*QKV), cu_q=None, cu_k=None, nseq=1, o=FAKE, lse=None,
                B=1, Tq=16, Tk=16, Hq=4, Hk=4, D=128, scale=0.1, window=0, sinks=0, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_window_fwd(*args.values())


def bwd(**over):
    args = dict(q=FAKE, k=FAKE, v=FAKE, dtype=1, strides=strides(*QKV), cu_q=None, cu_k=None, nseq=1, o=FAKE, lse=FAKE,
                go=FAKE, glse=None, dq=FAKE, dk=FAKE, dv=FAKE, B=1, Tq=16, Tk=16, Hq=4, Hk=4, D=128, scale=0.1,
                window=0, sinks=0, ws=FAKE, ws_bytes=1 << 40, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_window_bwd(*args.values())


BAD_WINDOW_CALLS = [
    (dict(dtype=3), _lib.ERR_INVALID_ARGUMENT),
    (dict(q=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(v=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(k=FAKE + 8), _lib.ERR_INVALID_ARGUMENT),                 # 16-byte alignment
    (dict(strides=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(*QKV[:8], 60)), _lib.ERR_INVALID_ARGUMENT),  # rows off 16 bytes
    (dict(strides=strides(*QKV[:7], -512, 128)), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(*QKV[:7], 1 << 23, 128)), _lib.ERR_UNSUPPORTED),  # token stride of 16 MiB
    (dict(Hq=6), _lib.ERR_INVALID_ARGUMENT),
    (dict(Hk=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(Tq=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(Tk=1 << 30), _lib.ERR_UNSUPPORTED),
    (dict(nseq=2), _lib.ERR_INVALID_ARGUMENT),                     # N must equal B without boundaries
    (dict(cu_q=FAKE, B=2, nseq=2), _lib.ERR_INVALID_ARGUMENT),     # boundaries need B == 1
    (dict(cu_q=FAKE, Tk=20), _lib.ERR_INVALID_ARGUMENT),           # one set of boundaries, two lengths
    (dict(cu_k=FAKE), _lib.ERR_INVALID_ARGUMENT),
    (dict(D=96), _lib.ERR_UNSUPPORTED),
    (dict(scale=float("nan")), _lib.ERR_INVALID_ARGUMENT),
    (dict(scale=float("inf")), _lib.ERR_INVALID_ARGUMENT),
    (dict(sinks=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(o=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(o=FAKE + 8), _lib.ERR_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("over,code", BAD_WINDOW_CALLS)
def test_window_calls_reject(over, code):
    assert fwd(**over) == code
    assert bwd(**over) == code


@pytest.mark.parametrize("over", [dict(lse=None), dict(go=None), dict(go=FAKE + 4), dict(dq=None), dict(dk=None),
                                  dict(ws=None), dict(ws=FAKE + 8), dict(ws_bytes=8)])
def test_window_bwd_rejects(over):
    assert bwd(**over) == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("heads,head", [
    (32, (0x7ffffff0 - 256) // 2 // 31 // 8 * 8 + 8),  # one step of 16 bytes past the limit
    (32, 1 << 27),                                     # wraps in 32 bits: 31 of 256 MiB
    (64, 1 << 27),                                     # a group of more heads than a tile
    (2, 1 << 31), (2, 1 << 59)])
def test_rows_of_q_past_32_bits_are_refused_and_copied(heads, head):
    """The gradient kernels reach 32 rows of q by 32-bit offsets: the C ABI refuses heads farther
    apart than that, the host API makes q dense. (Only refused calls are made: others would launch.)"""
    assert bwd(Hq=heads, Hk=1, strides=strides(0, 512, head, *QKV[3:])) == _lib.ERR_UNSUPPORTED
    k, v = (torch.empty(1, 16, 1, 128, dtype=torch.bfloat16, device="meta") for _ in range(2))
    for step in (head, head - 8):
        if step * heads * 2 >= 1 << 62:
            continue  # no such tensor
        q = torch.empty_strided((1, 16, heads, 128), (0, 512, step, 1), dtype=torch.bfloat16, device="meta")
        kept = at._window_operands(q, k, v)
        assert kept[0] is q and list(kept[3])[:3] == [0, 512, step]  # the forward reads it in place
        got = at._window_operands(q, k, v, gradients=True)
        copied = got[0] is not q
        assert copied == (step == head or head >= 1 << 27)
        assert list(got[3])[:3] == ([0, heads * 128, 128] if copied else [0, 512, step])


def test_a_head_of_its_own_may_lie_anywhere():
    """One head a group: its stride is no part of a tile."""
    q = torch.empty_strided((1, 16, 2, 128), (0, 128, 1 << 31, 1), dtype=torch.bfloat16, device="meta")
    k, v = (torch.empty(1, 16, 2, 128, dtype=torch.bfloat16, device="meta") for _ in range(2))
    assert at._window_operands(q, k, v, gradients=True)[0] is q


def test_empty_window_calls_are_ok():
    for empty in (dict(B=0, nseq=0), dict(Tq=0), dict(cu_q=FAKE, nseq=0)):
        assert fwd(**empty) == _lib.OK and bwd(**empty) == _lib.OK


def test_backward_workspace():
    size = _lib.attn_lib().pbattn_window_bwd_workspace_size
    plain = size(4, 2048, 2048, 32, 8, 128, 4, 1, 0, 1024, 0)
    assert plain >= 4 * 2048 * 32 * 8
    assert size(4, 2048, 2048, 32, 8, 128, 4, 1, 0, 1024, 4) > plain      # the sinks' parts
    assert size(4, 2048, 2048, 32, 8, 128, 4, 1, 0, 2048, 4) == size(4, 2048, 2048, 32, 8, 128, 4, 1, 0, 0, 0)
    assert size(1, 64, 64, 3, 2, 128, 1, 1, 0, 0, 0) == 0                 # heads
    assert size(1, 64, 64, 4, 2, 96, 1, 1, 0, 0, 0) == 0                  # width


def test_backward_workspace_of_short_documents():
    """Sequences no longer than the window have no sinks beyond it: 8,192 tokens in 1,000 documents, window
    128, 64 sinks, 8 key heads of 128. At most 63 of them are longer, with two parts each beside one per 256
    tokens, of 2 x 64 x 8 x 128 float32 values: 83 MB."""
    size = _lib.attn_lib().pbattn_window_bwd_workspace_size
    plain = size(1, 8192, 8192, 32, 8, 128, 1000, 1, 1, 128, 0)
    packed = size(1, 8192, 8192, 32, 8, 128, 1000, 1, 1, 128, 64)
    assert 0 < packed - plain <= (2 * 63 + 32 + 1) * 2 * 64 * 8 * 128 * 4
    # few long ones: two parts of each beside one per 256 tokens
    assert size(1, 8192, 8192, 32, 8, 128, 2, 1, 1, 128, 64) - plain <= (2 * 2 + 32 + 1) * 2 * 64 * 8 * 128 * 4


def decode(**over):
    args = dict(q=FAKE, k=FAKE, v=FAKE, dtype=1, strides=strides(16 * 256, 256, 128), page=16, pages=8, table=FAKE,
                max_pages=4, lengths=FAKE, o=FAKE, lse=None, B=2, T=1, Hq=4, Hk=2, D=128, scale=0.1, window=0, sinks=0,
                ws=FAKE, ws_bytes=1 << 40, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_paged_decode(*args.values())


def test_decoding_of_more_threads_than_a_launch_has_is_refused():
    """2^24 workgroups of 256 threads, in the parts' join or their own launch: told before either."""
    assert decode(B=1 << 22, Hq=16, Hk=4) == _lib.ERR_UNSUPPORTED
    assert decode(B=1 << 23, Hq=2, Hk=2) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("over,code", [
    (dict(dtype=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(T=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(T=17), _lib.ERR_INVALID_ARGUMENT),
    (dict(Hq=5), _lib.ERR_INVALID_ARGUMENT),
    (dict(page=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(pages=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(16 * 256, 255, 128)), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(16 * 256 + 8, 256, 128)), _lib.ERR_INVALID_ARGUMENT),  # page stride not in whole tokens
    (dict(strides=strides(16 * 256, 0, 128)), _lib.ERR_INVALID_ARGUMENT),
    (dict(pages=1 << 28), _lib.ERR_UNSUPPORTED),                                 # rows past 31 bits
    (dict(lengths=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(table=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(o=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(q=FAKE + 2), _lib.ERR_INVALID_ARGUMENT),
    (dict(D=80), _lib.ERR_UNSUPPORTED),
    (dict(sinks=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(scale=float("inf")), _lib.ERR_INVALID_ARGUMENT),
    (dict(ws=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(ws_bytes=100), _lib.ERR_INVALID_ARGUMENT),
])
def test_paged_decode_rejects(over, code):
    assert decode(**over) == code
    assert decode(B=0) == _lib.OK


def write(**over):
    args = dict(k=FAKE, v=FAKE, dtype=1, kv=strides(256, 128, 256, 128), kc=FAKE, vc=FAKE,
                strides=strides(16 * 256, 256, 128), page=16, pages=8, slots=FAKE, N=3, Hk=2, D=128, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_paged_write(*args.values())


@pytest.mark.parametrize("over,code", [
    (dict(dtype=7), _lib.ERR_INVALID_ARGUMENT),
    (dict(N=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(page=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(k=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(vc=FAKE + 4), _lib.ERR_INVALID_ARGUMENT),
    (dict(slots=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(kv=strides(256, 128, 250, 128)), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(16 * 256, 256, -128)), _lib.ERR_INVALID_ARGUMENT),
    (dict(D=60), _lib.ERR_UNSUPPORTED),  # 120 bytes are no whole 16-byte units
])
def test_paged_write_rejects(over, code):
    assert write(**over) == code
    assert write(N=0) == _lib.OK and write(pages=0) == _lib.OK


# ----------------------------------------------------------------------------
# The host API's refusals.
# ----------------------------------------------------------------------------
def tensors(tq=8, tk=8, hq=4, hk=2, d=64, batch=1):
    return torch.zeros(batch, tq, hq, d), torch.zeros(batch, tk, hk, d), torch.zeros(batch, tk, hk, d)


@pytest.mark.parametrize("kw,over,message", [
    (dict(hq=3), {}, "multiple of the key heads"),
    (dict(d=300), {}, "above 256"),
    (dict(batch=2), dict(cu_seqlens=torch.tensor([0, 8])), "B == 1"),
    (dict(tk=9), dict(cu_seqlens=torch.tensor([0, 8])), "cu_seqlens_k"),
    ({}, dict(cu_seqlens_k=torch.tensor([0, 8])), "needs cu_seqlens"),
    ({}, dict(cu_seqlens=torch.tensor([0, 8]), cu_seqlens_k=torch.tensor([0, 4, 8])), "shape"),
    ({}, dict(cu_seqlens=torch.zeros(1, 2)), "1-D"),
])
def test_window_attention_refuses_shapes(kw, over, message):
    with pytest.raises(ValueError, match=message):
        at.window_attention(*tensors(**kw), 1.0, **over)


def test_window_attention_refuses_cpu_tensors_and_bad_values():
    with pytest.raises(RuntimeError, match="no CPU path"):
        at.window_attention(*tensors(), 1.0)
    with pytest.raises(ValueError, match="window must be"):
        at._window_args(0, 0)
    with pytest.raises(ValueError, match="sinks"):
        at._window_args(None, -1)
    with pytest.raises(ValueError, match="float64"):
        at._dtype_code(torch.float64)
    with pytest.raises(ValueError, match="one shape"):
        q, k, v = tensors()
        at.window_attention(q, k, v[:, :4], 1.0)


def test_paged_calls_refuse():
    q, cache = torch.zeros(2, 1, 4, 64), torch.zeros(5, 16, 2, 64)
    table, lengths = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        at.paged_decode_attention(q, cache, cache, table, lengths, 1.0)
    with pytest.raises(RuntimeError, match="no backward"):
        at.paged_decode_attention(q.requires_grad_(True), cache, cache, table, lengths, 1.0)
    with pytest.raises(RuntimeError, match="no backward"):
        at.paged_cache_write(torch.zeros(2, 2, 64, requires_grad=True), torch.zeros(2, 2, 64), cache, cache, lengths)
    for bad in (torch.zeros(5, 16, 2, 65)[..., :64], torch.zeros(5, 16, 2, 128)[..., ::2],
                torch.zeros(5 * 16 * 128 + 16 * 4)[: 5 * (16 * 128 + 12)].as_strided((5, 16, 2, 64), (16 * 128 + 12, 128, 64, 1))):
        with pytest.raises(ValueError, match="strides"):
            at._caches(bad, bad)
    with pytest.raises(ValueError, match="strides"):
        at._caches(cache, torch.zeros(5, 2, 16, 64).transpose(1, 2))
    with pytest.raises(ValueError, match="one shape"):
        at._caches(cache, cache[:4])
    heads_first = cache.transpose(1, 2).contiguous().transpose(1, 2)
    sizes, steps, *_ = at._caches(heads_first, heads_first)
    assert sizes == (5, 16, 2, 64) and list(steps) == [2048, 64, 1024]


def misaligned(tokens, heads, d, dtype, lead=()):
    """Columns of wider rows: strides of whole 16 bytes, a base 8 bytes off."""
    skip = 8 // dtype.itemsize
    z = torch.randn(*lead, tokens, heads * d + 16 // dtype.itemsize).to(dtype)
    x = z[..., skip:skip + heads * d].unflatten(-1, (heads, d))
    assert x.data_ptr() % 16 == 8 and all(s * dtype.itemsize % 16 == 0 for s in x.stride()[:-1])
    return x


def read_by(tensor, steps):
    """The tensor's rows as a kernel finds them by its stride array."""
    return tensor.as_strided(tensor.shape, (*steps, 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_are_those_of_the_tensors_passed_on(dtype):
    """A view copied for its base's alignment gives its rows another distance."""
    q, k, v = (misaligned(5, h, 64, dtype, (2,)) for h in (4, 2, 2))
    *got, steps = at._window_operands(q, k, v)
    for i, (x, y) in enumerate(zip(got, (q, k, v))):
        assert list(steps)[3 * i:3 * i + 3] == list(x.stride())[:3] and x.data_ptr() % 16 == 0
        assert torch.equal(read_by(x, list(steps)[3 * i:3 * i + 3]), y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_written_rows_strides_are_those_of_the_tensors_passed_on(dtype, monkeypatch):
    calls = []
    monkeypatch.setattr(at, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(at, "_launch", lambda where, fn, dev, *args: calls.append(args))
    k, v = (misaligned(5, 2, 64, dtype) for _ in range(2))
    cache = torch.zeros(3, 16, 2, 64, dtype=dtype)
    at.paged_cache_write(k, v, cache, cache.clone(), torch.arange(5))
    (k_at, v_at, code, steps, *_), = calls
    # (an aligned view's tensor is passed as it is, a copy densely)
    assert k_at % 16 == 0 and v_at % 16 == 0 and list(steps) == [128, 64, 128, 64]


def test_a_stale_attention_library_is_named(tmp_path):
    src = tmp_path / "stub.cpp"
    src.write_text('extern "C" int pbattn_abi_version(void) { return 0; }\n')
    lib = tmp_path / "libstub.so"
    subprocess.run(["g++", "-shared", "-fPIC", str(src), "-o", str(lib)], check=True)
    with pytest.raises(RuntimeError, match="ABI version 0.*rebuild it"):
        _lib._load_attn(str(lib))


def test_forward_mode_tangents_are_refused(monkeypatch):
    """The kernels have no forward-mode derivative: no result without its tangent."""
    import torch.autograd.forward_ad as forward_ad
    monkeypatch.setattr(at, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(at, "_launch", lambda *args: None)
    q, k, v = tensors()
    cache, slots = torch.zeros(5, 16, 2, 64), torch.arange(8)
    table, lengths = torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with torch.no_grad():
        at.window_attention(q, k, v, 1.0)
    with forward_ad.dual_level():
        at.window_attention(q, k, v, 1.0)  # no tangent among the inputs
        for i in range(3):
            x = [q, k, v]
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                at.window_attention(*x, 1.0)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            at.paged_decode_attention(forward_ad.make_dual(q, q)[:, :1], cache, cache, table, lengths, 1.0)
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            at.paged_cache_write(forward_ad.make_dual(k[0], k[0]), v[0], cache, cache, slots)
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda t: at.window_attention(t, k, v, 1.0), (q,), (q,))


@pytest.mark.filterwarnings("ignore")
def test_jit_trace_records_the_op(monkeypatch):
    """Not the empty output that the launch fills."""
    monkeypatch.setattr(at, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(at, "_launch", lambda *args: None)
    q, k, v = tensors()
    graph = torch.jit.trace(lambda q, k, v: at.window_attention(q, k, v, 1.0, 4, 1), (q, k, v), check_trace=False).graph
    assert "pbgdn::window_attention" in str(graph) and "aten::empty" not in str(graph)


def paged_inputs(dtype=torch.bfloat16, device=None):
    q, k, v = (torch.zeros(2, 1, h, 64, dtype=dtype, device=device) for h in (4, 2, 2))
    kc, vc = (torch.zeros(5, 16, 2, 64, dtype=dtype, device=device) for _ in range(2))
    table, lengths = torch.zeros(2, 3, dtype=torch.int32, device=device), torch.ones(2, dtype=torch.int32, device=device)
    return q, k[:, 0], v[:, 0], kc, vc, table, lengths, torch.arange(2, device=device)


def paged_step(q, k, v, kc, vc, table, lengths, slots, out=None):
    at.paged_cache_write(k, v, kc, vc, slots)
    return at.paged_decode_attention(q, kc, vc, table, lengths, 0.125, 8, 1, return_lse=True, out=out)


def test_paged_calls_under_fake_tensors():
    """Inside the mode, and with fake tensors outside of it."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = paged_inputs()
        o, lse = paged_step(*x)
        assert o.shape == x[0].shape and o.dtype == x[0].dtype and lse.shape == (2, 1, 4)
        out = torch.empty_like(x[0])
        assert paged_step(*x, out=out)[0] is out
        with pytest.raises(ValueError, match="out must"):
            paged_step(*x, out=out.float())
    assert paged_step(*x)[0].shape == x[0].shape


def test_paged_calls_are_traced_as_ops(monkeypatch):
    """make_fx of real tensors: the ops, not the outputs that the launches fill."""
    from torch.fx.experimental.proxy_tensor import make_fx
    monkeypatch.setattr(at, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(at, "_launch", lambda *args: None)
    monkeypatch.setattr(at, "_decode_plan", lambda *args: ((2, 1, 4, 2, 64), 8, 1, 256))  # (asks for the device)
    for mode in ("real", "fake", "symbolic"):
        code = make_fx(lambda *x: paged_step(*x), tracing_mode=mode)(*paged_inputs()).code
        assert "pbgdn.paged_cache_write_" in code and "pbgdn.paged_decode_attention" in code
        assert "empty" not in code


def test_a_cache_write_counts_as_one(monkeypatch):
    """The caches' versions rise, so that autograd notices a cache it has saved."""
    monkeypatch.setattr(at, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(at, "_launch", lambda *args: None)
    q, k, v, kc, vc, *_, slots = paged_inputs()
    w = torch.ones(64, dtype=kc.dtype, requires_grad=True)
    loss = (kc * w).sum() + (vc * w).sum()
    before = kc._version, vc._version
    at.paged_cache_write(k, v, kc, vc, slots)
    assert kc._version > before[0] and vc._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # (tensors without a version)
        kc, vc = kc.clone(), vc.clone()
        at.paged_cache_write(k, v, kc, vc, slots)


def test_ops_infer_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k, v = (torch.empty(2, 9, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
        o, lse = torch.ops.pbgdn.window_attention(q, k, v, 0.1, None, 0, None, None)
        assert o.shape == q.shape and o.dtype == q.dtype and lse.shape == (2, 9, 4) and lse.dtype == torch.float32
        grads = torch.ops.pbgdn.window_attention_backward(q, k, v, o, lse, o, None, 0.1, 3, 1, None, None)
        assert [g.shape for g in grads] == [q.shape, k.shape, v.shape]
        cache = torch.empty(5, 16, 2, 64, dtype=torch.bfloat16)
        o, lse = torch.ops.pbgdn.paged_decode_attention(q[:, :1], cache, cache, torch.empty(2, 3, dtype=torch.int32),
                                                        torch.empty(2, dtype=torch.int32), 0.1, None, 0)
        assert o.shape == (2, 1, 4, 64) and lse.shape == (2, 1, 4)


# ----------------------------------------------------------------------------
# The kernels' code: no read of a matrix product's result before it is there
# (hipcc's own distances in straight-line code: 12 wait states for the 32x32x16
# products, 18 for 32x32x2 float32).
# ----------------------------------------------------------------------------
def test_no_mfma_result_is_read_early(monkeypatch):
    for op, need in (("v_mfma_f32_32x32x16_bf16", 12), ("v_mfma_f32_32x32x16_f16", 12), ("v_mfma_f32_32x32x2_f32", 18)):
        monkeypatch.setitem(hazards.NEED, op, need)
    sources = [s for s in build.ATTN_SOURCES if s.startswith("attn_")]
    with tempfile.TemporaryDirectory() as tmp:
        def compile_one(src):
            out = os.path.join(tmp, src + ".s")
            subprocess.run([build.hipcc(), *build.HIPCC_FLAGS, f"-I{build.INCLUDE}", "--cuda-device-only", "-S",
                            os.path.join(build.CSRC, src), "-o", out], check=True, capture_output=True)
            with open(out) as f:
                return f.read()

        with ThreadPoolExecutor(max_workers=len(sources)) as pool:
            listings = list(pool.map(compile_one, sources))
    problems = []
    for src, asm in zip(sources, listings):
        assert "v_mfma" in asm, src
        problems += [f"{src}: {name[-60:]}: '{prod}' read by '{rd}' after {w}"
                     for name, prod, rd, w in hazards.short_reads(asm)]
    assert not problems, "\n".join(problems[:20])


def test_narrow_decoding_keeps_its_registers(tmp_path):
    """The 64-wide 16-bit decoding kernels: no register spilled, and few enough of them for three waves
    a SIMD (168 of 512; two waves take 10 to 15% more time)."""
    out = tmp_path / "decode.s"
    subprocess.run([build.hipcc(), *build.HIPCC_FLAGS, f"-I{build.INCLUDE}", "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, "attn_decode.hip"), "-o", str(out)], check=True, capture_output=True)
    meta = out.read_text().split("amdhsa.kernels:")[1]
    found = 0
    for entry in re.split(r"\n  - \.", meta)[1:]:
        name = re.search(r"\.name:\s+(\S+)", entry).group(1)
        if not re.search(r"decode_kernelILi[12]ELi64E", name):
            continue
        number = {k: int(re.search(rf"{k}:\s+(\d+)", entry).group(1)) for k in ("vgpr_count", "vgpr_spill_count")}
        assert number["vgpr_spill_count"] == 0 and number["vgpr_count"] <= 168, (name, number)
        found += 1
    assert found == 4


# ----------------------------------------------------------------------------
# The oracle.
# ----------------------------------------------------------------------------
def test_oracle_masks_by_definition():
    for tq, tk, window, sinks in [(5, 5, None, 0), (4, 9, 3, 2), (6, 2, 2, 1), (1, 1, 1, 5)]:
        seen = oa.visible(tq, tk, window, sinks)
        for i in range(tq):
            for j in range(tk):
                p = tk - tq + i
                assert seen[i, j] == (j <= p and (window is None or j > p - window or j < sinks))


def test_oracle_closed_forms():
    rng = np.random.default_rng(0)
    v = rng.standard_normal((6, 1, 4))
    r = oa.attention(np.zeros((6, 2, 4)), rng.standard_normal((6, 1, 4)), v, 1.0, 3, 1)
    for i in range(6):  # equal scores: the mean of what is seen
        seen = [j for j in range(i + 1) if j > i - 3 or j < 1]
        np.testing.assert_allclose(r["o"][i, 1], v[seen, 0].mean(0), rtol=1e-14)
        np.testing.assert_allclose(r["lse"][i, 0], np.log(len(seen)), atol=1e-14)
    r = oa.attention(np.ones((3, 1, 4)), np.ones((1, 1, 4)), np.ones((1, 1, 4)), 1.0)
    assert (r["o"][:2] == 0).all() and np.isneginf(r["lse"][:2]).all() and (r["o"][2] == 1).all()


@pytest.mark.parametrize("tq,tk,window,sinks", [(5, 5, None, 0), (4, 9, 3, 2), (5, 3, 2, 1)])
def test_oracle_gradients_against_differences(tq, tk, window, sinks):
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal(s) for s in ((tq, 4, 3), (tk, 2, 3), (tk, 2, 3)))
    go, glse = rng.standard_normal(q.shape), rng.standard_normal((tq, 4))

    def loss(q, k, v):
        r = oa.attention(q, k, v, 0.7, window, sinks)
        return (r["o"] * go).sum() + (np.where(np.isfinite(r["lse"]), r["lse"], 0) * glse).sum()

    r = oa.attention(q, k, v, 0.7, window, sinks, go, glse)
    for n, x in zip(("dq", "dk", "dv"), (q, k, v)):
        for at_ in np.ndindex(x.shape):
            keep, ends = x[at_], []
            for step in (1e-5, -1e-5):
                x[at_] = keep + step
                ends.append(loss(q, k, v))
            x[at_] = keep
            # the difference's own error: 1e-10 (third derivatives) and 1e-16 / 1e-5
            np.testing.assert_allclose((ends[0] - ends[1]) / 2e-5, r[n][at_], atol=1e-8)


def test_numbers_past_32_bits_do_not_wrap_around():
    """Lengths, tables and boundaries of 64 bits: what 32 do not hold stays as large, or as small, as they go."""
    x = torch.tensor([[5, 2**32 + 3, -2**32 + 5], [2**62, -2**63, -1]])
    want = torch.tensor([[5, 2**31 - 1, -2**31], [2**31 - 1, -2**31, -1]], dtype=torch.int32)
    for y in (x, x.t().contiguous().t()):
        got = at._boundaries(y)
        assert got.dtype == torch.int32 and got.is_contiguous() and torch.equal(got, want)
    assert torch.equal(at._boundaries(x[:, ::2]), want[:, ::2]) and at._boundaries(want) is want
    assert torch.equal(at._boundaries(torch.tensor([3, 4], dtype=torch.int16)), torch.tensor([3, 4], dtype=torch.int32))
