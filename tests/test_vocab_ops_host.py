"""What the vocabulary operators refuse, checked without a GPU: every test ends before a launch."""
import ctypes
import importlib

import numpy as np
import pytest
import torch

from helpers import pkg  # noqa: F401
from oracle import vocab_refs as ref

hip = importlib.import_module("image-captioning-through-rl_amd.hipabi")
A = 1 << 20   # an address that is aligned and never followed: the arguments are refused first


def refused(name, *args, match):
    lib = hip.load()
    assert getattr(lib, name)(*args) == -1
    assert match in lib.icrl_last_error().decode()


SAMPLE = dict(logits=A, dtype=0, ld=100, n=4, v=100, u=A, t_rows=None, t=1.0, k_rows=None, k=0, p_rows=None, p=1.0,
              m_rows=None, m=0.0, out=A, stride=1, lp=None, lps=1, work=None, nwork=0, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(logits=None), "null pointer"), (dict(u=None), "null pointer"), (dict(out=None), "null pointer"),
    (dict(n=0), "empty shape"), (dict(v=0), "empty shape"), (dict(ld=99), "ld_logits < V"), (dict(dtype=7), "dtype"),
    (dict(v=(1 << 22) + 1, ld=1 << 23), "exceeds"), (dict(t=-1.0), "temperature"), (dict(t=float("nan")), "temperature"),
    (dict(t=float("inf")), "temperature"), (dict(k=-1), "top_k"), (dict(p=-0.1), "top_p"), (dict(p=1.5), "top_p"),
    (dict(p=float("nan")), "top_p"), (dict(m=1.01), "min_p"), (dict(m=float("nan")), "min_p"),
    (dict(v=100000, ld=100000, work=A, nwork=1000), "work"), (dict(work=A + 4), "work")])
def test_sample_filtered_refuses(change, match):
    refused("icrl_sample_tokens_filtered", *dict(SAMPLE, **change).values(), match=match)


RECORD = dict(logits=A, dtype=0, ld=100, n=4, v=100, k=8, t=1.0, values=A, indices=A, lse=None, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(logits=None), "null pointer"), (dict(values=None), "null pointer"), (dict(indices=None), "null pointer"),
    (dict(n=0), "empty shape"), (dict(k=0), "k must be"), (dict(k=101), "k must be"), (dict(v=5000, ld=5000, k=1025), "k must be"),
    (dict(t=0.0), "temperature"), (dict(t=float("inf")), "temperature"), (dict(ld=10), "ld_logits"), (dict(dtype=3), "dtype")])
def test_topk_lse_refuses(change, match):
    refused("icrl_topk_lse_rows", *dict(RECORD, **change).values(), match=match)


LOSS = dict(logits=A, dtype=1, ld=100, n=4, v=100, tv=A, ti=A, k=8, lse=None, t=1.0, w=None, loss=A, stats=None, d=None, ldd=0,
            stream=None)
GRAD = dict(logits=A, dtype=1, ld=100, n=4, v=100, tv=A, ti=A, k=8, t=1.0, stats=A, w=None, d=A, ldd=100, stream=None)
SHARED = [(dict(logits=None), "null pointer"), (dict(tv=None), "null pointer"), (dict(ti=None), "null pointer"),
          (dict(n=-1), "empty shape"), (dict(k=0), "k must be"), (dict(k=101), "k must be"), (dict(ld=99), "ld_logits"),
          (dict(t=0.0), "temperature"), (dict(t=float("nan")), "temperature"), (dict(dtype=-1), "dtype"),
          (dict(v=(1 << 18) + 1, ld=1 << 20, ldd=1 << 20), "exceeds"), (dict(stats=A + 4), "8-byte")]


@pytest.mark.parametrize("change,match", SHARED + [(dict(loss=None), "null pointer"), (dict(d=A, ldd=99), "ld_dlogits")])
def test_distill_loss_refuses(change, match):
    refused("icrl_distill_loss", *dict(LOSS, **change).values(), match=match)


@pytest.mark.parametrize("change,match", SHARED + [(dict(stats=None), "null pointer"), (dict(d=None), "null pointer"),
                                                   (dict(ldd=99), "ld_dlogits")])
def test_distill_grad_refuses(change, match):
    refused("icrl_distill_grad", *dict(GRAD, **change).values(), match=match)


# bf16, four rows of 100: one entry further, a row further, other strides from the same place, halves that overlap
@pytest.mark.parametrize("ld,d,ldd", [(100, A + 2, 100), (100, A - 2, 100), (100, A + 200, 100), (100, A, 128), (150, A + 120, 150),
                                      (250, A + 302, 250), (120, A + 120 * 2 * 3 + 198, 200)])
def test_distill_refuses_gradients_that_overlap_the_logits(ld, d, ldd):
    refused("icrl_distill_loss", *dict(LOSS, ld=ld, d=d, ldd=ldd).values(), match="overlaps")
    refused("icrl_distill_grad", *dict(GRAD, ld=ld, d=d, ldd=ldd).values(), match="overlaps")


CUT = dict(x=A, dtype=0, ld=64, rows=4, k=64, pieces=A, scales=A, stream=None)
GEMM = dict(ap=A, as_=A, bp=A, bs=A, c=A, dtype=0, ldc=100, m=4, n=100, k=64, bias=None, stream=None)


@pytest.mark.parametrize("change,match", [(dict(x=None), "null pointer"), (dict(rows=0), "empty shape"), (dict(ld=63), "row stride"),
                                          (dict(pieces=A + 8), "aligned"), (dict(scales=A + 2), "aligned"), (dict(dtype=9), "dtype")])
def test_cut_fp8_refuses(change, match):
    refused("icrl_cut_fp8", *dict(CUT, **change).values(), match=match)


@pytest.mark.parametrize("change,match", [(dict(ap=None), "null operand"), (dict(bs=None), "null operand"), (dict(k=0), "empty shape"),
                                          (dict(ldc=99), "ldc"), (dict(bp=A + 4), "aligned"), (dict(dtype=4), "dtype")])
def test_gemm_fp8_refuses(change, match):
    refused("icrl_gemm_fp8", *dict(GEMM, **change).values(), match=match)


def test_fp8_buffer_sizes():
    lib = hip.load()
    assert lib.icrl_fp8_piece_bytes(1, 1) == 32 * 128 and lib.icrl_fp8_piece_bytes(33, 129) == 64 * 256
    assert lib.icrl_fp8_scale_bytes(1, 1) == 32 * 4 and lib.icrl_fp8_scale_bytes(33, 513) == 64 * 8
    assert lib.icrl_fp8_piece_bytes(0, 5) == 0 and lib.icrl_fp8_scale_bytes(5, 0) == 0
    assert lib.icrl_fp8_piece_bytes(1 << 20, 1 << 14) == 1 << 34   # past 32 bits
    for rows, k in ((1, 1), (31, 128), (32, 129), (33, 512), (10000, 513), (1 << 20, 1 << 14)):
        assert hip._fp8_bytes(rows, k) == (lib.icrl_fp8_piece_bytes(rows, k), lib.icrl_fp8_scale_bytes(rows, k))


def test_bindings_refuse_host_tensors_and_wrong_types():
    x, u, out = torch.zeros(2, 10), torch.zeros(2, dtype=torch.float64), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(AssertionError):
        hip.sample_tokens_filtered(x, out, 1, u)
    with pytest.raises(AssertionError):
        hip._row_stride(torch.zeros(4, 8).t())
    with pytest.raises(AssertionError):
        hip._row_stride(torch.zeros(8).expand(4, 8))   # rows on top of each other
    assert hip._row_stride(torch.zeros(4, 20)[:, :8]) == 20 and hip._row_stride(torch.zeros(8).expand(1, 8)) == 8
    with pytest.raises(AssertionError):
        hip._dtype_code(torch.zeros(1, dtype=torch.float64))
    with pytest.raises(AssertionError):
        hip._vector(torch.zeros(3), 4, torch.float32, "row_weight")
    assert hip._holds(torch.zeros(11)[1:], 4, 3) and not hip._holds(torch.zeros(10)[1:], 4, 3)


# ------------------------------------------------------------------ the references themselves
def test_reference_gradient_against_differences():
    rs = np.random.RandomState(0)
    x, t = rs.standard_normal(40) * 2, rs.standard_normal(40) * 2
    idx = np.argsort(-t)[:6]
    temp = 1.7
    lse = np.log(np.exp(t / temp).sum())
    for given in (lse, None):
        _, grad, _ = ref.distill(x, t[idx], idx, given, temp, 0.6)
        for i in range(40):
            h = np.zeros(40)
            h[i] = 1e-5
            up, down = (ref.distill(x + s * h, t[idx], idx, given, temp, 0.6)[0] for s in (1, -1))
            assert abs((up - down) / 2e-5 - grad[i]) < 1e-9


def test_reference_filters_agree_with_the_unfiltered_draw():
    rs = np.random.RandomState(1)
    x = rs.standard_normal(50) * 2
    p = np.exp(x - x.max())
    cdf = np.cumsum(p / p.sum())
    for u in rs.random_sample(30):
        assert ref.sample_filtered(x, u)[0] == (cdf <= u).sum()
    kept = {ref.sample_filtered(x, u, top_k=3)[0] for u in np.linspace(0, 0.999, 200)}
    assert kept == set(np.argsort(-x)[:3].tolist())


def test_reference_eight_bit_values_against_torch():
    x = (np.random.RandomState(2).standard_normal((6, 300)) * np.exp2(np.random.RandomState(3).randint(-20, 20, (6, 1)))).astype(np.float32)
    x[2, :128] = 0
    values, exps = ref.fp8_values(x)
    scale = np.exp2(exps.astype(np.float64)).repeat(128, axis=1)[:, :300]
    codes = torch.from_numpy((x / scale).astype(np.float32)).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(values, codes * scale)
    assert (np.abs(x).reshape(6, -1)[:, :128].max(1) <= 448 * 2.0 ** exps[:, 0]).all()
