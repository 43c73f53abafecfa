"""Norms and rotation without a GPU: the oracle against differences and rotations of
plane vectors, the C ABI's and the host API's refusals."""
import numpy as np
import pytest
import torch

from oracle import rope as orp
from pseudobrain_amd import _lib
from pseudobrain_amd import rope
from tests.test_attention_cpu import FAKE, strides


def inputs(d=16, rotary=8, tokens=5, heads=3, seed=0):
    rng = np.random.default_rng(seed)
    x, g = rng.standard_normal((2, 1, tokens, heads, d))
    w = 1 + 0.3 * rng.standard_normal(d)
    angle = rng.uniform(-3, 3, (7, rotary // 2))
    return x, g, w, np.cos(angle), np.sin(angle), np.array([[0, 6, -1, 3, 7]])[:, :tokens]


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_by_complex_numbers(interleaved):
    x, _, w, cos, sin, pos = inputs()
    y = orp.rows(x, w, cos, sin, pos, 1e-6, interleaved, "float32")["y"]
    for t, p in enumerate(pos[0]):
        for h in range(3):
            if not 0 <= p < 7:
                assert not y[0, t, h].any()
                continue
            v = x[0, t, h] / np.sqrt((x[0, t, h] ** 2).mean() + 1e-6) * w
            for i in range(4):
                a, b = (2 * i, 2 * i + 1) if interleaved else (i, 4 + i)
                turned = (v[a] + 1j * v[b]) * (cos[p, i] + 1j * sin[p, i])
                np.testing.assert_allclose([y[0, t, h, a], y[0, t, h, b]], [turned.real, turned.imag], rtol=1e-12)
            np.testing.assert_allclose(y[0, t, h, 8:], v[8:], rtol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 2, 16])
def test_oracle_gradients_by_differences(interleaved, rotary):
    x, g, w, cos, sin, pos = inputs(rotary=rotary)
    got = orp.rows(x, w, cos, sin, pos, 1e-3, interleaved, "float32", g)

    def loss(x, w):
        return (orp.rows(x, w, cos, sin, pos, 1e-3, interleaved, "float32")["y"] * g).sum()

    step = 1e-6
    rng = np.random.default_rng(1)
    for _ in range(30):
        at = tuple(rng.integers(n) for n in x.shape)
        e = np.zeros_like(x)
        e[at] = step
        np.testing.assert_allclose((loss(x + e, w) - loss(x - e, w)) / (2 * step), got["dx"][at], atol=1e-8)
    for i in range(16):
        e = np.zeros_like(w)
        e[i] = step
        np.testing.assert_allclose((loss(x, w + e) - loss(x, w - e)) / (2 * step), got["dw"][i], atol=1e-7)


def test_tables():
    cos, sin = rope.rope_tables(5, 6, 100.0, device="cpu")
    want = np.arange(5)[:, None] * 100.0 ** (-np.arange(0, 6, 2) / 6)
    np.testing.assert_allclose(cos.numpy(), np.cos(want), atol=2.0 ** -24)
    np.testing.assert_allclose(sin.numpy(), np.sin(want), atol=2.0 ** -24)
    assert rope.rope_tables(3, 0, device="cpu")[0].shape == (3, 0)
    far = rope.rope_tables(262144, 4, device="cpu")[0][-1]  # (the angle itself in float32 would be off by 2^-7)
    np.testing.assert_allclose(far.numpy(), np.cos(262143 * np.array([1.0, 0.01])), atol=2.0 ** -24)
    for bad in ((5, 3), (5, -2), (-1, 4)):
        with pytest.raises(ValueError):
            rope.rope_tables(*bad, device="cpu")


def forward(**over):
    args = dict(q=FAKE, k=FAKE, dtype=1, strides=strides(4096, 512, 128, 1024, 256, 128), qw=FAKE, kw=FAKE, wdt=1, offset=0.0,
                cos=FAKE, sin=FAKE, rows=9, pos=FAKE, pos64=0, ps=strides(0, 1), qo=FAKE, ko=FAKE, B=1, T=8, Hq=4, Hk=2, D=128,
                R=64, eps=1e-6, interleaved=0, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_qk_norm_rope(*args.values())


def backward(**over):
    args = dict(q=FAKE, k=FAKE, dtype=1, strides=strides(4096, 512, 128, 1024, 256, 128), qw=FAKE, kw=FAKE, wdt=1, offset=0.0,
                cos=FAKE, sin=FAKE, rows=9, pos=FAKE, pos64=0, ps=strides(0, 1), gq=FAKE, gk=FAKE, dq=FAKE, dk=FAKE, dqw=FAKE,
                dkw=FAKE, B=1, T=8, Hq=4, Hk=2, D=128, R=64, eps=1e-6, interleaved=0, ws=FAKE, ws_bytes=1 << 40, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_qk_norm_rope_bwd(*args.values())


BOTH = [
    (dict(dtype=3), _lib.ERR_INVALID_ARGUMENT),
    (dict(wdt=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(R=63), _lib.ERR_INVALID_ARGUMENT),
    (dict(R=130), _lib.ERR_INVALID_ARGUMENT),
    (dict(R=-2), _lib.ERR_INVALID_ARGUMENT),
    (dict(D=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(D=264), _lib.ERR_UNSUPPORTED),
    (dict(Hk=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(B=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(T=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(rows=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(eps=-1e-6), _lib.ERR_INVALID_ARGUMENT),
    (dict(eps=float("nan")), _lib.ERR_INVALID_ARGUMENT),
    (dict(eps=float("inf")), _lib.ERR_INVALID_ARGUMENT),
    (dict(offset=float("nan")), _lib.ERR_INVALID_ARGUMENT),
    (dict(interleaved=2), _lib.ERR_INVALID_ARGUMENT),
    (dict(pos64=2), _lib.ERR_INVALID_ARGUMENT),
    (dict(pos64=1, pos=FAKE + 4), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(4096, 512, -128, 1024, 256, 128)), _lib.ERR_INVALID_ARGUMENT),
    (dict(ps=strides(0, -1)), _lib.ERR_INVALID_ARGUMENT),
    (dict(q=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(q=FAKE + 1), _lib.ERR_INVALID_ARGUMENT),
    (dict(kw=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(wdt=0, qw=FAKE + 2), _lib.ERR_INVALID_ARGUMENT),
    (dict(cos=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(sin=FAKE + 2), _lib.ERR_INVALID_ARGUMENT),
    (dict(pos=None), _lib.ERR_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("over,code", BOTH + [
    (dict(qo=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(ko=FAKE + 8), _lib.ERR_INVALID_ARGUMENT),
])
def test_forward_rejects(over, code):
    assert forward(**over) == code
    assert forward(B=0) == _lib.OK and forward(T=0) == _lib.OK


@pytest.mark.parametrize("over,code", BOTH + [
    (dict(gq=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(gk=FAKE + 8), _lib.ERR_INVALID_ARGUMENT),
    (dict(dk=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(dqw=FAKE + 2), _lib.ERR_INVALID_ARGUMENT),
    (dict(ws=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(ws_bytes=64), _lib.ERR_INVALID_ARGUMENT),
])
def test_backward_rejects(over, code):
    assert backward(**over) == code
    assert backward(B=0) == _lib.OK and backward(T=0) == _lib.OK


def test_workspace_size():
    size = _lib.attn_lib().pbattn_qk_norm_rope_bwd_workspace_size
    assert size(0) == size(257) == size(-1) == 0 and size(128) == 2 * size(64) > 0


def tensors(batch=2, tokens=3, hq=4, hk=2, d=32, rotary=16, dtype=torch.float32):
    return dict(q=torch.zeros(batch, tokens, hq, d, dtype=dtype), k=torch.zeros(batch, tokens, hk, d, dtype=dtype),
                q_weight=torch.ones(d, dtype=dtype), k_weight=torch.ones(d, dtype=dtype), cos=torch.zeros(9, rotary // 2),
                sin=torch.zeros(9, rotary // 2), positions=torch.zeros(tokens, dtype=torch.int64))


def test_calls_refuse():
    with pytest.raises(RuntimeError, match="no CPU path"):
        rope.qk_norm_rope(**tensors())
    for over, message in (
            (dict(q=torch.zeros(2, 3, 128)), "expected q"), (dict(k=torch.zeros(2, 4, 2, 32)), "expected q"),
            (dict(k=torch.zeros(2, 3, 2, 64)), "expected q"), (dict(k=torch.zeros(2, 3, 0, 32)), "at least one head"),
            (dict(q_weight=torch.ones(31)), "weight"), (dict(k=torch.zeros(2, 3, 2, 32).half()), "one dtype"),
            (dict(k_weight=torch.ones(32).half()), "their weights one"), (dict(cos=torch.zeros(9, 8).half()), "float32 tables"),
            (dict(sin=torch.zeros(8, 8)), "one shape"), (dict(cos=torch.zeros(9, 17), sin=torch.zeros(9, 17)), "more values"),
            (dict(positions=torch.zeros(3)), "int32 or int64"), (dict(positions=torch.zeros(4).long()), "broadcasts"),
            (dict(positions=torch.zeros(3, 3).long()), "broadcasts"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps")):
        with pytest.raises(ValueError, match=message):
            rope.qk_norm_rope(**{**tensors(), **over})
    for over in (dict(q=torch.zeros(1, 1, 4, 32).expand(1, 2**32, 4, 32), k=torch.zeros(1, 1, 2, 32).expand(1, 2**32, 2, 32)),
                 dict(cos=torch.zeros(1, 8).expand(2**32, 8), sin=torch.zeros(1, 8).expand(2**32, 8))):
        with pytest.raises(ValueError, match="less than"):  # (sizes that 32-bit counts call zero)
            rope.qk_norm_rope(**{**tensors(), "positions": torch.zeros(1).long(), **over})
    with pytest.raises(ValueError, match="above 256"):
        rope.qk_norm_rope(**tensors(d=264))
    with pytest.raises(ValueError, match="float64"):
        rope.qk_norm_rope(**tensors(dtype=torch.float64))
    with pytest.raises(RuntimeError, match="no gradient for its tables"):
        rope.qk_norm_rope(**{**tensors(), "sin": torch.zeros(9, 8, requires_grad=True)})


def test_forward_mode_tangents_are_refused(monkeypatch):
    import torch.autograd.forward_ad as forward_ad
    monkeypatch.setattr(rope, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(rope, "_launch", lambda *args: None)
    with forward_ad.dual_level():
        rope.qk_norm_rope(**tensors())  # no tangent among the inputs
        for name in ("q", "k", "q_weight", "k_weight", "cos"):
            t = tensors()
            t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                rope.qk_norm_rope(**t)


def test_strides_passed_on(monkeypatch):
    """Columns of one projection's output are read in place, transposed rows are copied."""
    calls = []
    monkeypatch.setattr(rope, "_one_device", lambda *t: t[0].device)
    monkeypatch.setattr(rope, "_launch", lambda where, fn, dev, *args: calls.append(args))
    t = tensors()
    qkv = torch.zeros(2, 3, 8 * 32)
    q, k, _ = (x.unflatten(-1, (-1, 32)) for x in qkv.split([128, 64, 64], -1))
    rope.qk_norm_rope(**{**t, "q": q, "k": k, "positions": torch.zeros(2, 1, dtype=torch.int32)})
    (q_at, k_at, code, steps, *rest), = calls
    assert (q_at, k_at) == (q.data_ptr(), k.data_ptr()) and list(steps) == [768, 256, 32] * 2
    assert list(rest[9]) == [1, 0]
    rope.qk_norm_rope(**{**t, "q": torch.zeros(2, 3, 32, 4).transpose(2, 3)})
    assert list(calls[1][3]) == [384, 128, 32, 192, 64, 32] and list(calls[1][13]) == [0, 1]
