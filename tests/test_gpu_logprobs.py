"""GPU parity of the token log probabilities against 64-bit numpy.

Tolerance: sums of up to 2^11 f32 terms per thread and exponentials good to
2^-22 leave ln s and w / s within about 2^-19 relative of their sums' size, and
each result is a difference of terms up to ln V + |ref|:
  |x - ref| <= 4e-6 (1 + ln V + |ref|).
Ids are compared exactly (the order goes by the logits themselves).
"""
from __future__ import annotations

import numpy as np
import pytest

from doe_b200 import ops
from doe_b200._abi import DOE_DEVICE_ERR_POSITION
from oracle import kv_int4

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _near(got, ref, V):
    got, ref = got.double().cpu().numpy(), np.asarray(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    inf = np.isinf(ref)
    assert np.array_equal(got[inf], ref[inf])
    f = np.isfinite(ref)
    assert np.isfinite(got[f]).all()
    err = np.abs(got[f] - ref[f])
    assert (err <= 4e-6 * (1 + np.log(V) + np.abs(ref[f]))).all(), float(err.max())


def _check(x, tokens, k, **kw):
    """x: a CUDA tensor [rows, V]."""
    status = ops.status_word()
    r = ops.token_logprobs(x, torch.as_tensor(tokens, dtype=torch.int32, device="cuda"), top_k=k, status=status, **kw)
    lp, h, ids, top = kv_int4.logprobs(x.float().cpu().numpy(), np.asarray(tokens), k)
    assert int(status.item()) == 0
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    _near(r.logprob, lp, x.shape[1])
    _near(r.entropy, h, x.shape[1])
    _near(r.top_logprobs, top, x.shape[1])
    return r


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,k", [(1, 32, 1), (3, 33, 32), (1, 4097, 5), (2, 32000, 20), (7, 1000, 0), (300, 2049, 3),
                                      (64, 50001, 32), (1, 262144, 32)])
def test_random_rows(dtype, rows, V, k):
    g = np.random.default_rng(V + rows)
    x = torch.from_numpy((g.standard_normal((rows, V)) * 4).astype(np.float32)).to(DTYPES[dtype]).cuda()
    _check(x, g.integers(0, V, rows), k)


@pytest.mark.parametrize("V", [1, 2, 3, 7, 31])
def test_fewer_tokens_than_alternatives(V):
    g = np.random.default_rng(V)
    x = torch.from_numpy(g.standard_normal((2, V)).astype(np.float32)).cuda()
    r = ops.token_logprobs(x, torch.tensor([0, V - 1], dtype=torch.int32, device="cuda"), top_k=32)
    lp, h, ids, top = kv_int4.logprobs(x.cpu().numpy(), np.array([0, V - 1]), V)
    assert np.array_equal(r.top_ids[:, :V].cpu().numpy(), ids) and (r.top_ids[:, V:] == -1).all()
    assert (r.top_logprobs[:, V:] == -np.inf).all()
    _near(r.top_logprobs[:, :V], top, V)
    _near(r.logprob, lp, V)
    _near(r.entropy, h, V)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 3, 5])
def test_strides_and_alignment(dtype, offset):
    g = np.random.default_rng(offset)
    wide = torch.from_numpy(g.standard_normal((5, 6007)).astype(np.float32)).to(DTYPES[dtype]).cuda()
    wide[:, :offset] = 1e4  # outside the view: must not be read into it
    wide[:, offset + 5001:] = 1e4
    _check(wide[:, offset:offset + 5001], g.integers(0, 5001, 5), 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties_go_to_the_lowest_index(dtype):
    g = np.random.default_rng(1)
    x = torch.from_numpy(g.integers(-3, 4, (4, 40000)).astype(np.float32)).to(DTYPES[dtype]).cuda()
    x[1] = 2.5                      # one value everywhere
    x[2, ::2] = 0.0
    x[2, 1::2] = -0.0               # the two zeros are equal
    _check(x, [5, 6, 7, 8], 32)


@pytest.mark.parametrize("order", ["up", "down", "saw"])
def test_ordered_rows(order):
    V = 100000
    x = np.arange(V, dtype=np.float32) * 1e-3
    x = x[::-1].copy() if order == "down" else x if order == "up" else x[np.argsort(np.arange(V) % 977, kind="stable")]
    _check(torch.from_numpy(np.stack([x] * 3)).cuda(), [0, V // 2, V - 1], 32)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(dtype):
    g = np.random.default_rng(2)
    x = torch.from_numpy((g.standard_normal((6, 9001)) * 3).astype(np.float32)).to(DTYPES[dtype]).cuda()
    low = torch.finfo(DTYPES[dtype]).min
    x[0, ::2] = -np.inf
    x[1] = -np.inf                  # nothing left
    x[2] = -np.inf
    x[2, 77] = 1.0                  # one token left
    x[3, :9000] = low
    x[4] = low                      # the type's lowest value everywhere
    x[5, 100:] = -np.inf
    r = _check(x, [1, 5, 77, 9000, 3, 50], 20)
    assert r.entropy[1].item() == 0.0 and r.logprob[1].item() == -np.inf
    assert abs(r.logprob[2].item()) < 1e-6


def test_nan_and_infinity_rows():
    x = torch.randn((3, 5000), device="cuda")
    x[0, 17] = float("nan")
    x[1, 18] = float("inf")
    r = ops.token_logprobs(x, torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), top_k=4)
    assert torch.isnan(r.logprob[:2]).all() and torch.isnan(r.entropy[:2]).all() and torch.isnan(r.top_logprobs[:2]).all()
    assert 17 not in r.top_ids[0].tolist() and r.top_ids[1, 0].item() == 18
    assert torch.isfinite(r.logprob[2]) and torch.isfinite(r.top_logprobs[2]).all()


@pytest.mark.parametrize("shift", [0.0, 1e4, -3e4])
def test_large_logits(shift):
    """A common offset changes nothing but the logits' own rounding."""
    g = np.random.default_rng(3)
    x = (g.standard_normal((2, 7001)) * 3 + shift).astype(np.float32)
    _check(torch.from_numpy(x).cuda(), [1, 2], 5)


def test_peaked_rows_have_small_entropy():
    x = torch.zeros((2, 30000), device="cuda")
    x[0, 3] = 40.0
    x[1, 4] = 200.0
    r = _check(x, [3, 4], 2)
    assert r.entropy[1].item() >= -1e-6


def test_tokens_outside_the_vocabulary_and_none():
    x = torch.randn((3, 100), device="cuda")
    status = ops.status_word()
    r = ops.token_logprobs(x, torch.tensor([-1, 100, 5], dtype=torch.int32, device="cuda"), top_k=2, status=status)
    assert int(status.item()) == DOE_DEVICE_ERR_POSITION
    assert r.logprob[0].item() == r.logprob[1].item() == -np.inf and torch.isfinite(r.logprob[2])
    r = ops.token_logprobs(x, top_k=2)
    assert r.logprob is None and torch.isfinite(r.entropy).all()
    assert ops.token_logprobs(x[:0], top_k=2).top_ids.shape == (0, 2)


def test_many_rows_and_side_stream():
    x = torch.randn((70000, 40), device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    r = ops.token_logprobs(x, torch.zeros(70000, dtype=torch.int32, device="cuda"), top_k=3, stream=s)
    s.synchronize()
    want = torch.log_softmax(x.double(), -1)
    assert torch.equal(r.top_ids.long(), torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :3])
    assert bool(((r.logprob.double() - want[:, 0]).abs() < 4e-6 * (5 + want[:, 0].abs())).all())


def test_repeated_calls_agree():
    x = torch.randn((4, 128256), device="cuda").bfloat16()
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    a, b = (ops.token_logprobs(x, t, top_k=32) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refusals():
    x = torch.randn((3, 100), device="cuda")
    for bad in (x.double(), x.t(), x.cpu(), x[0]):
        with pytest.raises(ValueError):
            ops.token_logprobs(bad)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError):
        ops.token_logprobs(x, top_k=33)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1, -1])
def test_maxima_on_both_sides_of_the_exponents_two_forms(dtype, sign):
    """Largest logits just below and above 60000 in different parts of a row, some masked."""
    g = np.random.default_rng(4)
    x = g.standard_normal((4, 70001)) * 3 + sign * 59999.0
    x[1] += 3.0
    x[2, ::3] = -np.inf
    x[3, 5:] = -np.inf
    x = torch.from_numpy(x.astype(np.float32)).to(DTYPES[dtype]).cuda()
    assert torch.isfinite(x[0]).all()
    _check(x, [0, 1, 4, 3], 7)


def test_rows_past_32_bit_offsets():
    """A row stride of over 2^32 elements."""
    stride = 2 ** 32 + 24
    store = torch.empty(stride + 5000, dtype=torch.float16, device="cuda")
    x = store.as_strided((2, 5000), (stride, 1))
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x.copy_(torch.randn((2, 5000), generator=g, device="cuda") * 3)
    _check(x, [17, 4999], 6)


def _stable_ids(x, k):
    return torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :k].int()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ["plateau", "short", "holes"])
def test_ties_behind_masked_stretches(dtype, case):
    """A forbidden stretch leaves a group of threads without a maximum, so every allowed element is a
    candidate and more of them are met than the buffer holds; which ones fit is a matter of timing."""
    g = np.random.default_rng(11)
    if case == "plateau":      # one value, the first allowed tokens far from the first thread's
        x = np.zeros((4, 4096), np.float32)
        x[:, :1536] = x[:, 2048:2112] = -np.inf
        x[1, 1600:] = 1.0
        x[2, 1536:1700] = -1.0
        x[3, 1560::7] = 2.0
        rows = [x]
    elif case == "short":      # fewer groups hold an element than alternatives are asked for
        rows = [g.integers(0, n, (8, V)).astype(np.float32) for V in (1025, 1056, 1100, 1537, 2000) for n in (2, 40)]
    else:                      # a hole at the start of every split
        x = g.integers(0, 3, (2, 131072)).astype(np.float32)
        for s in range(0, 131072, 4096):
            x[:, s:s + 64] = -np.inf
        x[1] = np.where(np.isinf(x[1]), x[1], 0.5)
        rows = [x]
    for x in rows:
        x = torch.from_numpy(x).to(DTYPES[dtype]).cuda()
        for k in (20, 32):
            want = _stable_ids(x, k)
            got = [ops.token_logprobs(x, top_k=k).top_ids for _ in range(50)]
            assert all(torch.equal(i, want) for i in got)
