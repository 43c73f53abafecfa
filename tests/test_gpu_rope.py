"""qk_norm_rope and its gradients on the device against the float64 oracle
(oracle/rope.py), element by element within its error bounds: widths and rotated parts,
types, strides, padding, positions far out, rows at the ends of the types' ranges."""
import numpy as np
import pytest
import torch

from oracle import rope as orp
from pseudobrain_amd import _lib, rope
from tests.test_gpu_window_attention import NAMES, compare, f64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(batch, tokens, hq, hk, d, rotary, dtype, seed, wdtype=None, table=50, size=2.0):
    gen = torch.Generator().manual_seed(seed)
    q, k, gq, gk = (torch.randn(batch, tokens, h, d, generator=gen) * s
                    for h, s in ((hq, size), (hk, size), (hq, 0.3), (hk, 0.3)))
    qw, kw = (1 + 0.2 * torch.randn(2, d, generator=gen)).to(wdtype or dtype).to(DEV)
    angle = (torch.rand(table, rotary // 2, generator=gen) - 0.5) * 12
    positions = torch.randint(table, (batch, tokens), generator=gen)
    q, k, gq, gk = (x.to(dtype).to(DEV) for x in (q, k, gq, gk))
    return dict(q=q, k=k, qw=qw, kw=kw, cos=angle.cos().to(DEV), sin=angle.sin().to(DEV), pos=positions.to(DEV), gq=gq, gk=gk)


def check(where, x, eps=1e-6, offset=0.0, interleaved=False, grads=True):
    q, k, qw, kw = (x[n].detach().requires_grad_(grads) for n in ("q", "k", "qw", "kw"))
    print(f"[{where}] q {tuple(q.shape)} k {tuple(k.shape)} R {2 * x['cos'].shape[1]} {q.dtype} {qw.dtype}", flush=True)
    out = rope.qk_norm_rope(q, k, qw, kw, x["cos"], x["sin"], x["pos"], eps, weight_offset=offset, interleaved=interleaved)
    got = torch.autograd.grad(out, (q, k, qw, kw), (x["gq"], x["gk"])) if grads else None
    torch.cuda.synchronize()
    pos = np.broadcast_to(f64(x["pos"]).astype(np.int64), q.shape[:2])
    for i, (v, w, g) in enumerate(((q, qw, x["gq"]), (k, kw, x["gk"]))):
        w64 = f64(w.detach()) + offset
        ref = orp.rows(f64(v.detach()), w64, f64(x["cos"]), f64(x["sin"]), pos, eps, interleaved, NAMES[q.dtype],
                       f64(g) if grads else None, NAMES[qw.dtype])
        name = "qk"[i]
        assert out[i].dtype == v.dtype and out[i].is_contiguous()
        compare(f"{where} {name}", out[i].detach(), ref["y"], ref["y_tol"])
        if grads:
            compare(f"{where} d{name}", got[i], ref["dx"], ref["dx_tol"])
            compare(f"{where} d{name} weight", got[2 + i], ref["dw"], ref["dw_tol"])
            assert got[i].dtype == v.dtype and got[2 + i].dtype == w.dtype
    return out, got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 64), (64, 16), (128, 128), (128, 64), (256, 64), (256, 256), (96, 32), (16, 16), (128, 0)])
def test_widths_and_types(d, rotary, dtype, interleaved):
    check("widths", make(2, 9, 5, 3, d, rotary, dtype, d + rotary), interleaved=interleaved)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(1, 0), (2, 2), (5, 4), (33, 10), (70, 70), (72, 36), (100, 48), (255, 254), (256, 100)])
def test_odd_widths(d, rotary, dtype, interleaved):
    """Widths and rotated parts that do not go into whole units."""
    check("odd", make(2, 7, 3, 2, d, rotary, dtype, d + rotary), interleaved=interleaved)


@pytest.mark.parametrize("hq,hk", [(1, 1), (32, 8), (16, 2), (7, 40), (3, 17)])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (64, 1), (1, 777), (3, 50)])
def test_heads_and_tokens(hq, hk, batch, tokens):
    check("heads", make(batch, tokens, hq, hk, 64, 32, torch.bfloat16, hq + tokens))


@pytest.mark.parametrize("wdtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 128), (torch.float16, 40)])
def test_weights_of_other_types(dtype, d, wdtype):
    x = make(2, 6, 4, 2, d, 24, dtype, 3, wdtype)
    check("weights", x)
    x["qw"], x["kw"] = x["qw"] - 1, x["kw"] - 1
    check("weights about zero", x, offset=1.0)


def test_many_rows():
    """Sums of the weights' gradients over more rows than the workgroups take at once."""
    check("many", make(4, 2048, 8, 4, 64, 64, torch.float32, 4))
    check("many, odd", make(2, 1100, 4, 4, 50, 20, torch.float32, 5))


@pytest.mark.parametrize("d", [64, 50])
def test_positions_of_padding_and_shapes(d):
    """Positions outside the tables give zeros and no gradient, whatever the rows hold; positions
    of one row for all, one for each batch row, 32 and 64 bits, strided."""
    x = make(3, 8, 4, 2, d, 32, torch.bfloat16, 6, table=20)
    x["pos"][0, 3], x["pos"][1, 0], x["pos"][2] = -1, 20, 2 ** 40
    for n in ("q", "k", "gq", "gk"):
        x[n][0, 3], x[n][2] = torch.nan, torch.inf
    out, got = check("padding", x)
    for y in (*out, *got[:2]):
        assert torch.count_nonzero(y[0, 3]) == 0 and torch.count_nonzero(y[2]) == 0
    x = make(3, 8, 4, 2, d, 32, torch.bfloat16, 7, table=20)
    for pos in (x["pos"][0], x["pos"][:1], x["pos"][:, :1], x["pos"].int(), x["pos"].t().contiguous().t(), x["pos"][0, :1],
                torch.stack((x["pos"], x["pos"]), -1)[..., 0]):
        check("shapes", {**x, "pos": pos})
    check("no table", {**x, "cos": x["cos"][:0], "sin": x["sin"][:0]})


def test_strided_and_unaligned_inputs():
    """Columns of a projection, heads before tokens, rows repeated over heads, rows off the
    alignment, gradients of one value."""
    for d in (64, 36):
        x = make(2, 10, 4, 2, d, 24 if d == 36 else 32, torch.bfloat16, 8)
        qkv = torch.randn(2, 10, 8 * d, device=DEV).to(torch.bfloat16)
        q, k, _ = (y.unflatten(-1, (-1, d)) for y in qkv.split([4 * d, 2 * d, 2 * d], -1))
        check("columns", {**x, "q": q, "k": k})
        check("heads first", {**x, "q": x["q"].transpose(1, 2).contiguous().transpose(1, 2)})
        check("repeated", {**x, "q": x["q"][:, :, :1].expand(-1, -1, 4, -1), "k": x["k"][:1].expand(2, -1, -1, -1)})
        off = torch.randn(2, 10, 4 * d + 8, device=DEV).to(torch.bfloat16)[..., 3:4 * d + 3].unflatten(-1, (4, d))
        check("off", {**x, "q": off})
        check("last axis strided", {**x, "k": x["k"].transpose(2, 3).contiguous().transpose(2, 3)})
        one = torch.ones((), device=DEV, dtype=torch.bfloat16)
        check("gradient of one value", {**x, "gq": one.expand_as(x["gq"]), "gk": one.expand_as(x["gk"])})


@pytest.mark.parametrize("dtype,size", [(torch.float32, 1e15), (torch.float32, 1e-15), (torch.bfloat16, 1e15),
                                        (torch.float16, 3e3), (torch.float16, 1e-4)])
@pytest.mark.parametrize("d", [64, 50])
def test_large_and_small_rows(dtype, size, d):
    x = make(1, 6, 2, 2, d, 20 if d == 50 else 32, dtype, 9)
    x["q"], x["k"] = x["q"] / 4 * size, x["k"] / 4 * size
    x["q"][0, 2] = 0
    check("sizes", x, eps=1e-6)


@pytest.mark.parametrize("dtype,size", [(torch.float32, 2.0**127), (torch.bfloat16, 2.0**127), (torch.float32, 1e25),
                                        (torch.float32, 1e-25), (torch.bfloat16, 1e-30)])
@pytest.mark.parametrize("d", [64, 50, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_whose_squares_float32_does_not_hold(dtype, size, d, interleaved):
    """Rows near the ends of the range among ordinary ones, with an eps of no weight beside them."""
    x = make(1, 6, 8, 3, d, 20 if d == 50 else 32, dtype, 15)
    for n in ("q", "k"):
        x[n] /= x[n].abs().max()
        x[n][0, 1:3] = (x[n][0, 1:3].float() * size).to(dtype)
        x[n][0, 4, 1] = (x[n][0, 4, 1].float() * size).to(dtype)
    check("ends of the range", x, eps=0.0 if size < 1 else 1e-6, interleaved=interleaved)


def test_ordinary_values_of_eps_count_beside_small_rows():
    """Tiny rows under an ordinary eps, and an eps of their own size (as the float32 that the kernels
    take: 1e-44 lies between two that are 2^-149 apart)."""
    x = make(1, 6, 4, 2, 64, 32, torch.float32, 16)
    x["q"], x["k"] = x["q"] * 1e-25, x["k"] * 1e-22
    for eps in (1e-6, 1e-35, 1e-44):
        check("eps", x, eps=float(np.float32(eps)))


@pytest.mark.parametrize("d", [64, 50])
def test_a_bad_value_stays_in_its_row(d):
    """An infinity or NaN reaches its own row alone, an infinity no value that is not rotated with it."""
    x = make(1, 6, 4, 2, d, 16, torch.float32, 10)
    clean, _ = check("clean", x)
    bad = {n: v.clone() for n, v in x.items()}
    bad["q"][0, 2, 1, 40], bad["k"][0, 4, 0, 3] = torch.inf, torch.nan
    q, k = rope.qk_norm_rope(*(bad[n] for n in ("q", "k", "qw", "kw", "cos", "sin", "pos")))
    want = torch.zeros(d, device=DEV)
    want[40] = torch.nan  # x r = 0 for the others
    torch.testing.assert_close(q[0, 2, 1], want, equal_nan=True, rtol=0, atol=0)
    assert torch.isnan(k[0, 4, 0]).all()
    q[0, 2, 1], k[0, 4, 0] = clean[0][0, 2, 1], clean[1][0, 4, 0]
    assert torch.equal(q, clean[0]) and torch.equal(k, clean[1])


def test_offsets_past_32_bits():
    """Rows of a projection's output beyond 4 GiB."""
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GiB of free device memory")
    x = make(1, 140000, 2, 1, 64, 64, torch.bfloat16, 11, table=200000)
    wide = torch.zeros(1, 140000, 16384, dtype=torch.bfloat16, device=DEV)  # 4.6 GB
    q, k = wide[..., :128].unflatten(-1, (2, 64)), wide[..., 128:192].unflatten(-1, (1, 64))
    q.copy_(x["q"]), k.copy_(x["k"])
    args = [x[n] for n in ("qw", "kw", "cos", "sin", "pos")]
    for a, b in zip(rope.qk_norm_rope(q, k, *args), rope.qk_norm_rope(x["q"], x["k"], *args)):
        assert torch.equal(a, b)


def test_empty_calls():
    for batch, tokens in ((0, 4), (2, 0)):
        x = make(batch, tokens, 4, 2, 64, 32, torch.float32, 12)
        q, k, qw, kw = (x[n].requires_grad_(True) for n in ("q", "k", "qw", "kw"))
        out = rope.qk_norm_rope(q, k, qw, kw, x["cos"], x["sin"], x["pos"])
        grads = torch.autograd.grad(out, (q, k, qw, kw), (x["gq"], x["gk"]))
        assert out[0].shape == q.shape and grads[0].shape == q.shape
        assert torch.count_nonzero(grads[2]) == 0 and torch.count_nonzero(grads[3]) == 0


def test_gradients_of_one_output_and_of_some_inputs():
    x = make(2, 5, 4, 2, 64, 32, torch.float32, 13)
    args = [x[n].detach().requires_grad_(True) for n in ("q", "k", "qw", "kw")]
    tables = x["cos"], x["sin"], x["pos"]
    both = torch.autograd.grad(rope.qk_norm_rope(*args, *tables), args, (x["gq"], torch.zeros_like(x["gk"])))
    q, _ = rope.qk_norm_rope(*args, *tables)
    one = torch.autograd.grad(q, args, x["gq"], materialize_grads=True)
    assert all(torch.equal(a, b) for a, b in zip(both, one))
    q, k = rope.qk_norm_rope(x["q"], x["k"], args[2], x["kw"], *tables)
    assert q.requires_grad and k.requires_grad
    dw, = torch.autograd.grad(q, args[2], x["gq"])
    assert torch.equal(dw, both[2])
    with pytest.raises(RuntimeError):  # once
        out = rope.qk_norm_rope(*args, *tables)
        g, = torch.autograd.grad(out[0].sum(), args[0], create_graph=True)
        g.sum().backward()


def test_equal_runs_and_graph_replay():
    """A training step captured and replayed several times among eager work, each replay bit-equal."""
    x = make(2, 300, 8, 4, 64, 32, torch.bfloat16, 14)
    leaves = [x[n] for n in ("q", "k", "qw", "kw")]

    def step():
        args = [t.detach().requires_grad_(True) for t in leaves]
        out = rope.qk_norm_rope(*args, x["cos"], x["sin"], x["pos"])
        return (*(y.detach() for y in out), *torch.autograd.grad(out, args, (x["gq"], x["gk"])))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        for y in out:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(out, want, step()):
            assert torch.equal(a, b) and torch.equal(c, b)


@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_training_equals_eager(dynamic):
    x = make(2, 20, 4, 2, 64, 32, torch.bfloat16, 15)

    def step(q, k, qw, kw, cos, sin, pos):
        a, b = rope.qk_norm_rope(q * 2, k, qw, kw, cos, sin, pos, weight_offset=0.5)
        return a * 3, b

    results = []
    for fn in (step, torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=dynamic)):
        args = [x[n].detach().requires_grad_(True) for n in ("q", "k", "qw", "kw")]
        out = fn(*args, x["cos"], x["sin"], x["pos"])
        results.append((*out, *torch.autograd.grad(out, args, (x["gq"], x["gk"]))))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_op_passes_the_opcheck():
    x = make(1, 4, 2, 1, 64, 32, torch.float32, 16)
    args = [x[n].requires_grad_(n in ("q", "k", "qw", "kw")) for n in ("q", "k", "qw", "kw", "cos", "sin", "pos")]
    torch.library.opcheck(rope.qk_norm_rope_op, (*args, 1e-6, 0.0, False),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))


DEBUG = {
    "units": lambda: test_widths_and_types(128, 64, torch.bfloat16, False),
    "odd": lambda: test_odd_widths(33, 10, torch.float32, True),
    "many": test_many_rows,
}


@pytest.mark.parametrize("case", DEBUG)
def test_under_the_debug_build(case):
    with _lib.debug_library():
        DEBUG[case]()
