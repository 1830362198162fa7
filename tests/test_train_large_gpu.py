"""The operators around a layer's products, dropout and the 8-bit products on tensors of more than 2^31 elements or 2^32 bytes, on a real MI355X:
rows on both sides of those marks against the same rows alone."""
import pytest
import torch

from grouped_mm_bf16_amd import dropout, int8, moe_train
from oracle import operators_oracle as plain, training_oracle as oracle

pytestmark = pytest.mark.gpu
BF, DEV = torch.bfloat16, "cuda"


def randn(*shape, seed=0):
    return torch.randn(*shape, device=DEV, dtype=BF, generator=torch.Generator(device=DEV).manual_seed(seed))


def bytes_(*shape, seed=0):
    return torch.randint(-127, 128, shape, device=DEV, dtype=torch.int8, generator=torch.Generator(device=DEV).manual_seed(seed))


def pieces(rows, width, size):
    """Rows at the start, around 2^31 and 2^32 elements and bytes, and at the end."""
    marks = {0, rows - 8} | {mark // (width * s) - 4 for mark in (2 ** 31, 2 ** 32) for s in (1, size)}
    return [slice(m, m + 8) for m in sorted(marks) if 0 <= m <= rows - 8]


def test_activation():
    h, grad = randn(140000, 16400).requires_grad_(), randn(140000, 8200, seed=1)
    out = moe_train.gated(h)
    dh, = torch.autograd.grad(out, h, grad)
    for s in pieces(140000, 16400, 2) + pieces(140000, 8200, 2):
        part = h.detach()[s].clone().requires_grad_()
        want = moe_train.gated(part)
        assert torch.equal(out[s], want) and torch.equal(dh[s], torch.autograd.grad(want, part, grad[s])[0])


def test_sorted_rows_and_sums():
    T, k, H = 40000, 4, 16400
    x, y, grad = randn(T, H), randn(T * k, H, seed=1).requires_grad_(), randn(T, H, seed=2)
    r = moe_train.route(randn(T, 16, seed=3), k)
    r = r._replace(slot_weight=r.slot_weight.clone().requires_grad_())
    rows = moe_train.sort_rows(x, r)
    back = r.row_token.long()
    for s in pieces(T * k, H, 2):
        assert torch.equal(rows[s], x[back[s]])
    out = moe_train.combine_rows(y, r, k)
    dy, dw = torch.autograd.grad(out, (y, r.slot_weight), grad)
    at = r.token_rows.reshape(T, k)
    for s in pieces(T * k, H, 2):
        tokens = back[s].unique()
        mine = at[tokens].reshape(-1).long()
        alone = r._replace(token_rows=torch.arange(mine.numel(), dtype=torch.int32, device=DEV),
                           slot_weight=r.slot_weight.detach().reshape(T, k)[tokens].reshape(-1).requires_grad_())
        part = y.detach()[mine].requires_grad_()
        want = moe_train.combine_rows(part, alone, k)
        gy, gw = torch.autograd.grad(want, (part, alone.slot_weight), grad[tokens])
        assert torch.equal(out[tokens], want) and torch.equal(dy[mine], gy) and torch.equal(dw.reshape(T, k)[tokens].reshape(-1), gw)


@pytest.mark.parametrize("width,pad", [(16384, 0), (16390, 0), (16390, 2)])
def test_dropout(width, pad):
    rows, p = 270000, 0.3
    x = randn(rows, width + pad)[:, :width]
    rng = torch.tensor([9, 2 ** 40 + 1], device=DEV)
    out = dropout.dropout(x, p, rng, site=3)
    limit = round(p * 65536)
    for s in pieces(rows, width, 2):
        first = s.start * width // 8
        skip = s.start * width - 8 * first
        bits = oracle.dropout_bits(skip + width, 9, 2 ** 40 + 1, 3, first)[skip:]
        kept = torch.from_numpy(bits >= limit)
        want = torch.where(kept, plain.f64(x[s.start]) * (65536 / (65536 - limit)), torch.zeros((), dtype=torch.float64))
        assert ((plain.f64(out[s.start]) - want).abs() <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -14)).all()


def test_rounding_of_rows():
    x = randn(140000, 16400)
    q, scale = int8.quantize_rows(x)
    for s in pieces(140000, 16400, 2):
        want = int8.quantize_rows(x[s])
        assert torch.equal(q[s], want.values) and torch.equal(scale[s], want.scale)


def test_products_of_many_rows():
    a = int8.Rows(bytes_(300000, 16384), torch.rand(300000, device=DEV) + 0.5)
    b = int8.Columns(bytes_(72, 16384, seed=1).t(), torch.rand(72, device=DEV) + 0.5)
    out = int8.int8_mm(a, b)
    for s in pieces(300000, 16384, 1):
        assert torch.equal(out[s], int8.int8_mm(int8.Rows(a.values[s], a.scale[s]), b))


def test_products_with_a_large_result():
    a = int8.Rows(bytes_(70000, 128), torch.rand(70000, device=DEV) + 0.5)
    b = int8.Columns(bytes_(33000, 128, seed=1).t(), torch.rand(33000, device=DEV) + 0.5)
    offs = torch.tensor([1000, 31111, 64999, 70000], dtype=torch.int32, device=DEV)
    want = [int8.int8_mm(int8.Rows(a.values[s], a.scale[s]), b) for s in pieces(70000, 33000, 2)]
    for out in (int8.int8_mm(a, b), int8.grouped_int8_mm(a, int8.Columns(b.values.expand(4, -1, -1), b.scale.expand(4, -1).contiguous()), offs)):
        for s, w in zip(pieces(70000, 33000, 2), want):
            assert torch.equal(out[s], w)


@pytest.mark.parametrize("M", [3, 40, 300])
def test_products_with_large_weights(M):
    """One matrix past 2 GiB, and many that are together."""
    a = int8.Rows(bytes_(M, 16384), torch.rand(M, device=DEV) + 0.5)
    b = int8.Columns(bytes_(140000, 16384, seed=1).t(), torch.rand(140000, device=DEV) + 0.5)
    out = int8.int8_mm(a, b)
    for s in pieces(140000, 16384, 1):
        assert torch.equal(out[:, s], int8.int8_mm(a, int8.Columns(b.values[:, s], b.scale[s])))
    many = int8.Columns(b.values.t().reshape(70, 2000, 16384).transpose(1, 2), b.scale.reshape(70, 2000))
    offs = torch.full((70,), M, dtype=torch.int32, device=DEV)
    offs[:68] = M // 3
    offs[:40] = 0
    got = int8.grouped_int8_mm(a, many, offs)
    for g, s in ((40, slice(0, M // 3)), (68, slice(M // 3, M))):
        if s.stop > s.start:
            assert torch.equal(got[s], int8.int8_mm(int8.Rows(a.values[s], a.scale[s]), int8.Columns(many.values[g], many.scale[g])))
