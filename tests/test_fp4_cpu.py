"""The 4-bit cache without a GPU: its format (oracle/fp4.py) against its definition's
properties, the C ABI's and the host API's refusals, and its kernels' matrix results
read late enough."""
import subprocess

import numpy as np
import pytest
import torch

from oracle import fp4 as of
from pseudobrain_amd import _lib, build
from pseudobrain_amd import fp4 as fc
from tests import test_mfma_hazards as hazards
from tests.test_attention_cpu import FAKE, HEADER, read_by, strides


def test_limits_agree_with_the_header():
    text = open(HEADER).read()
    assert f"#define PBATTN_MAX_REQUESTS {fc.MAX_REQUESTS}\n" in text


# ----------------------------------------------------------------------------
# The format.
# ----------------------------------------------------------------------------
def test_values_are_kept_to_half_a_step():
    """No value is off by more than half the distance of its neighbours, and what is held is kept."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)) * 2.0 ** rng.integers(-30, 30, (200, 1))
    data, scales = of.quantise(x)
    y = of.values(data, scales)
    s = np.repeat(2.0 ** (scales.astype(float) - 127), 32, -1)
    size = np.abs(x) / s
    assert size.max() < 7 and (np.abs(y).reshape(-1, 32).max(-1) >= 4 * s[:, ::32].reshape(-1)).all()
    step = np.where(size < 2, 0.5, np.where(size < 4, 1.0, 2.0))
    assert (np.abs(y - x) <= step / 2 * s).all()
    again = of.quantise(y)
    np.testing.assert_array_equal(of.values(*again), y)


def test_ties_scales_and_ends():
    x = np.zeros((9, 32))
    x[0, :8] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]       # ties, by a scale of 1
    x[1, :2] = [7.0, 1.0]                                        # 7 would be cut: a scale of 2
    x[2, :2] = [6.99, 1.0]                                       # 6.99 is 6
    x[3, 0] = 3.3e38                                             # past the largest scale: cut to 6 2^125
    x[4, 0] = 1e-45                                              # below half a step of the smallest
    x[5, 0] = np.inf
    x[6, 0] = np.nan
    x[8, 0] = -6.0
    data, scales = of.quantise(x)
    y = of.values(data, scales)
    assert scales[:, 0].tolist() == [127, 128, 127, 252, 2, 255, 255, 2, 127]
    np.testing.assert_array_equal(y[0, :8], [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0])
    np.testing.assert_array_equal(y[1, :2], [8.0, 1.0])
    assert y[2, 0] == 6.0 and y[3, 0] == 6 * 2.0 ** 125 and y[4, 0] == 0 and y[7, 0] == 0 and y[8, 0] == -6
    assert np.isnan(y[5]).all() and np.isnan(y[6]).all()
    assert data[0, 0] == 0x06 and data[8, 0] == 0x0f  # value 0 in the lower half; a negative value's code


def test_pages_by_multiplication():
    """The decoding kernel's j / page: the upper half of 2 j m, shifted, is the quotient for
    every 0 <= j < 2^31 (shown by j at and around multiples of the page, and at the ends)."""
    rng = np.random.default_rng(3)
    pages = [1, 2, 3, 7, 16, 100, 528, 4097, 2 ** 20 - 1, 2 ** 30 + 1, 2 ** 31 - 1, *rng.integers(1, 2 ** 31, 200).tolist()]
    for page in pages:
        shift = (page - 1).bit_length()
        m = (1 << (31 + shift)) // page + 1
        assert m < 2 ** 32
        top = (2 ** 31 - 1) // page * page
        some = [x * page for x in rng.integers(0, top // page + 1, 50).tolist()]
        for j in {0, 1, 2 ** 31 - 1, *(x + d for x in (top, *some) for d in (-1, 0, 1))}:
            if 0 <= j < 2 ** 31:
                assert ((2 * j * m) >> 32) >> shift == j // page


# ----------------------------------------------------------------------------
# The C ABI.
# ----------------------------------------------------------------------------
ROWS = strides(16 * 128, 128, 64)  # codes [8, 16, 2, 64]


def decode(**over):
    args = dict(q=FAKE, dtype=1, k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, strides=ROWS, page=16, pages=8, table=FAKE, max_pages=4,
                lengths=FAKE, o=FAKE, lse=None, B=2, T=1, Hq=4, Hk=2, D=128, scale=0.1, window=0, sinks=0, ws=FAKE,
                ws_bytes=1 << 40, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_fp4_decode(*args.values())


CACHE = [
    (dict(strides=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(16 * 128, 120, 64)), _lib.ERR_INVALID_ARGUMENT),         # not whole rows
    (dict(strides=strides(16 * 128 + 64, 128, 64)), _lib.ERR_INVALID_ARGUMENT),    # page stride not in whole tokens
    (dict(strides=strides(16 * 128, 0, 64)), _lib.ERR_INVALID_ARGUMENT),
    (dict(strides=strides(16 * 128, 128, -64)), _lib.ERR_INVALID_ARGUMENT),
    (dict(k=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(vs=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(ks=FAKE + 8), _lib.ERR_INVALID_ARGUMENT),
    (dict(v=FAKE + 4), _lib.ERR_INVALID_ARGUMENT),
    (dict(page=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(pages=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(D=80), _lib.ERR_UNSUPPORTED),
    (dict(D=512), _lib.ERR_UNSUPPORTED),
    (dict(dtype=3), _lib.ERR_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("over,code", CACHE + [
    (dict(T=0), _lib.ERR_INVALID_ARGUMENT),
    (dict(T=17), _lib.ERR_INVALID_ARGUMENT),
    (dict(Hq=5), _lib.ERR_INVALID_ARGUMENT),
    (dict(pages=1 << 28), _lib.ERR_UNSUPPORTED),  # rows past 31 bits
    (dict(lengths=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(table=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(o=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(q=FAKE + 2), _lib.ERR_INVALID_ARGUMENT),
    (dict(sinks=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(scale=float("nan")), _lib.ERR_INVALID_ARGUMENT),
    (dict(ws=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(ws_bytes=100), _lib.ERR_INVALID_ARGUMENT),
])
def test_decode_rejects(over, code):
    assert decode(**over) == code
    assert decode(B=0) == _lib.OK


def test_a_join_of_more_threads_than_a_launch_has_is_refused():
    """2^24 workgroups of 256 threads: told before the parts are worked out."""
    assert decode(B=1 << 22, Hq=32, Hk=4) == _lib.ERR_UNSUPPORTED


def write(**over):
    args = dict(kn=FAKE, vn=FAKE, dtype=1, kv=strides(256, 128, 256, 128), k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, strides=ROWS,
                page=16, pages=8, slots=FAKE, N=3, Hk=2, D=128, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_fp4_write(*args.values())


@pytest.mark.parametrize("over,code", CACHE + [
    (dict(N=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(kn=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(vn=FAKE + 4), _lib.ERR_INVALID_ARGUMENT),
    (dict(slots=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(kv=strides(256, 128, 250, 128)), _lib.ERR_INVALID_ARGUMENT),
    (dict(Hk=1 << 24), _lib.ERR_UNSUPPORTED),  # a token of 2^31 values
])
def test_write_rejects(over, code):
    assert write(**over) == code
    assert write(N=0) == _lib.OK and write(pages=0) == _lib.OK


def read(**over):
    args = dict(k=FAKE, v=FAKE, ks=FAKE, vs=FAKE, strides=ROWS, page=16, pages=8, table=FAKE, max_pages=4, lengths=FAKE,
                ko=FAKE, vo=FAKE, dtype=1, cu=FAKE, B=2, tokens=20, Hk=2, D=128, stream=None)
    args.update(over)
    return _lib.attn_lib().pbattn_fp4_read(*args.values())


@pytest.mark.parametrize("over,code", CACHE + [
    (dict(B=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(B=fc.MAX_REQUESTS + 1), _lib.ERR_UNSUPPORTED),
    (dict(tokens=-1), _lib.ERR_INVALID_ARGUMENT),
    (dict(ko=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(vo=FAKE + 8), _lib.ERR_INVALID_ARGUMENT),
    (dict(cu=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(lengths=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(table=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(Hk=1 << 24), _lib.ERR_UNSUPPORTED),
    (dict(tokens=2**31 - 1), _lib.ERR_UNSUPPORTED),  # more threads than a launch has
])
def test_read_rejects(over, code):
    assert read(**over) == code


# ----------------------------------------------------------------------------
# The host API.
# ----------------------------------------------------------------------------
def empty(pages=5, page=16, heads=2, width=64, heads_first=False):
    return fc.fp4_cache(pages, page, heads, width, "cpu", heads_first)


def test_calls_refuse():
    q, cache = torch.zeros(2, 1, 4, 64), empty()
    table, lengths = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fc.paged_decode_attention_fp4(q, cache, table, lengths, 1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fc.paged_cache_read_fp4(cache, table, lengths, 10)
    with pytest.raises(RuntimeError, match="no CPU path"):
        fc.paged_cache_write_fp4(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64), cache, lengths)
    with pytest.raises(RuntimeError, match="no backward"):
        fc.paged_decode_attention_fp4(q.requires_grad_(True), cache, table, lengths, 1.0)
    with pytest.raises(RuntimeError, match="no backward"):
        fc.paged_cache_write_fp4(torch.zeros(2, 2, 64, requires_grad=True), torch.zeros(2, 2, 64), cache, lengths)
    for bad in (dict(width=96), dict(page=0), dict(heads=0), dict(pages=-1)):
        with pytest.raises(ValueError):
            empty(**bad)


def test_call_shapes_are_checked(monkeypatch):
    monkeypatch.setattr(fc, "_one_device", lambda *t: torch.device("cuda", 0))
    monkeypatch.setattr(fc, "_launch", lambda *args: pytest.fail("launched"))
    cache, table, lengths = empty(), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for q, message in ((torch.zeros(2, 1, 4, 128), "head width"), (torch.zeros(2, 1, 3, 64), "multiple"),
                       (torch.zeros(2, 17, 4, 64), "1 to 16"), (torch.zeros(2, 4, 64), "expected q"),
                       (torch.zeros(3, 1, 4, 64), "expected page_table")):
        with pytest.raises(ValueError, match=message):
            fc._decode_plan(q.shape, q.dtype, fc._fp4(cache)[0], table.shape, lengths.shape, None, 0, 0)
    with pytest.raises(ValueError, match="float64"):
        fc.paged_cache_read_fp4(cache, table, lengths, 4, torch.float64)
    with pytest.raises(ValueError, match="tokens"):
        fc.paged_cache_read_fp4(cache, table, lengths, -1)
    with pytest.raises(ValueError, match="lengths"):
        fc.paged_cache_read_fp4(cache, table, lengths[:1], 4)
    long = table[:, :1].expand(2, 2**32)  # (more pages than a 32-bit count says)
    with pytest.raises(ValueError, match="expected page_table"):
        fc.paged_cache_read_fp4(cache, long, lengths, 4)
    with pytest.raises(ValueError, match="expected page_table"):
        fc.paged_decode_attention_fp4(torch.zeros(2, 1, 4, 64), cache, long, lengths, 1.0)
    with pytest.raises(ValueError, match="less than"):
        fc.paged_cache_write_fp4(*[torch.zeros(1, 2, 64).expand(2**32, 2, 64)] * 2, cache, lengths[:1].expand(2**32))
    many = fc.MAX_REQUESTS + 1
    with pytest.raises(ValueError, match="at most"):
        fc.paged_cache_read_fp4(cache, table[:1].expand(many, 3), lengths[:1].expand(many), 4)
    k = torch.zeros(2, 2, 64)
    with pytest.raises(ValueError, match="slots"):
        fc.paged_cache_write_fp4(k, k, cache, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="int32 or int64"):
        fc.paged_cache_write_fp4(k, k, cache, torch.zeros(2))
    with pytest.raises(ValueError, match="float64"):
        fc.paged_cache_write_fp4(k.double(), k, cache, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="heads"):
        fc.paged_cache_write_fp4(k[:, :1], k[:, :1], cache, torch.zeros(2, dtype=torch.int64))


def test_layouts():
    """Rows lie where the stride array says, those of axes of one element too."""
    for shape in ((5, 16, 2, 64), (1, 16, 2, 128), (5, 1, 1, 256), (1, 1, 3, 64), (1, 1, 1, 64), (4, 3, 1, 128)):
        for heads_first in (False, True):
            cache = fc.fp4_cache(*shape, "cpu", heads_first)
            sizes, steps, _ = fc._fp4(cache)
            assert sizes == shape
            for x, d in ((cache.k, 1), (cache.v, 1), (cache.k_scale, 16), (cache.v_scale, 16)):
                x.copy_(torch.randint(256, x.shape))
                assert torch.equal(read_by(x, [s // d for s in steps]), x)
            page_rows, left = divmod(steps[0], steps[1])
            assert left == 0 and page_rows >= shape[1] and steps[2] >= 0
    both = torch.zeros(5, 2, 16, 2, 32, dtype=torch.uint8), torch.zeros(5, 2, 16, 2, 2, dtype=torch.uint8)
    mixed = tuple(x[:, i] for x in both for i in range(2))  # keys and values page by page
    assert list(fc._fp4(mixed)[1]) == [2 * 16 * 64, 64, 32]


def test_layouts_that_do_not_match_are_refused():
    cache = empty()
    other = empty(heads_first=True)
    for bad in ((cache.k, other.v, cache.k_scale, cache.v_scale), (cache.k, cache.v, other.k_scale, other.v_scale)):
        with pytest.raises(ValueError, match="laid out alike"):
            fc._fp4(bad)
    with pytest.raises(ValueError, match="laid out alike"):
        fc._fp4(tuple(x[:1].expand(5, -1, -1, -1) for x in cache))
    wide = torch.zeros(5, 16, 2, 40, dtype=torch.uint8)[..., :32]
    with pytest.raises(ValueError, match="laid out alike"):
        fc._fp4((wide, wide, cache.k_scale, cache.v_scale))
    with pytest.raises(ValueError, match="expected a cache"):
        fc._fp4((cache.k, cache.v[:4], cache.k_scale, cache.v_scale))
    with pytest.raises(ValueError, match="expected a cache"):
        fc._fp4((cache.k, cache.v, cache.k_scale[..., :1], cache.v_scale[..., :1]))
    with pytest.raises(ValueError, match="uint8"):
        fc._fp4((cache.k, cache.v, cache.k_scale, cache.v_scale.view(torch.int8)))
    with pytest.raises(ValueError, match="width"):
        fc._fp4(tuple(torch.zeros(5, 16, 2, n, dtype=torch.uint8) for n in (16, 16, 1, 1)))
    off = torch.zeros(5 * 16 * 2 * 32 + 8, dtype=torch.uint8)[8:].view(5, 16, 2, 32)
    with pytest.raises(ValueError, match="16 bytes"):
        fc._fp4((off, cache.v, cache.k_scale, cache.v_scale))


# ----------------------------------------------------------------------------
# The kernels' matrix results.
# ----------------------------------------------------------------------------
def test_matrix_results_are_read_late_enough(tmp_path):
    out = tmp_path / "fp4.s"
    subprocess.run([build.hipcc(), *build.HIPCC_FLAGS, f"-I{build.INCLUDE}", "--cuda-device-only", "-S",
                    f"{build.CSRC}/attn_fp4.hip", "-o", str(out)], check=True, capture_output=True)
    asm = out.read_text()
    assert "v_mfma" in asm
    found = hazards.short_reads(asm)
    assert not found, "\n".join(f"{n[-48:]}: '{p}' read by '{r}' after {w}" for n, p, r, w in found[:20])
