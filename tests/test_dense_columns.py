"""Outputs that stand beside their inputs in one buffer: columns of the same rows, which share no element."""
import itertools

import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import dense


def _touch(a, b):
    """Whether two tensors on one buffer share a byte, element by element."""
    def spans(t):
        lo, size = t.data_ptr(), t.element_size()
        return {lo + sum(i * s for i, s in zip(idx, t.stride())) * size + k for idx in itertools.product(*map(range, t.shape)) for k in range(size)}
    return bool(spans(a) & spans(b))


def test_overlap_of_columns_is_by_element():
    buf = torch.zeros(400)
    rows = buf[:240].view(10, 24)
    half = rows.view(torch.bfloat16)                     # the same rows, 48 columns
    parts = [rows[:, i:j] for i, j in ((0, 8), (8, 16), (7, 9), (16, 24), (0, 24), (23, 24))]
    parts += [rows[2:5, 4:8], rows[9:, 4:8], rows[:1, :], rows[3:4, 20:], half[:, 16:32], half[:, :17], half[1:, 47:], rows[5, 3:9], rows[5, 20:], buf[100:130],
              buf[230:260], rows[::2, :4], rows[1::2, 4:]]
    for a, b in itertools.product(parts, parts):
        got = dense._overlap(a, b)
        assert got or not _touch(a, b)                   # never missed
        one = a.dim() == 1 or b.dim() == 1 or 1 in (a.shape[0], b.shape[0])
        if not one and a.stride(0) * a.element_size() == b.stride(0) * b.element_size():
            assert got == _touch(a, b), (a.shape, a.storage_offset(), b.shape, b.storage_offset())
    assert not dense._overlap(rows[:, :8], rows[:, 8:]) and not dense._overlap(half[:, 16:], rows[:, :8]) and dense._overlap(half[:, 15:], rows[:, :8])


def _gen(seed):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 9, 300, 700])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_product_into_the_columns_beside_its_tokens(T, dtype):
    g = _gen(T)
    f32 = dtype is torch.float32
    for K, N in ((200, 96), (201, 97), (512, 640)):
        w = okc.quantize_rows(torch.randn((N, K), generator=g, device="cuda"))
        both = okc.quantize_rows(torch.randn((2 * N, K), generator=g, device="cuda"))
        for fn, weight in ((okc.int8_linear, w), (okc.int8_gated, both)):
            for lo in (0, N):        # tokens in front of the result, and behind it
                store = torch.randn((T, N + K + 3), generator=g, device="cuda").to(dtype)
                x, out = store[:, lo:lo + K], store[:, (K if lo == 0 else 0):][:, :N]
                before, want = store.clone(), fn(x.clone(), weight, out_f32=f32)
                assert fn(x, weight, out_f32=f32, out=out) is out and torch.equal(out, want)
                out.copy_(before[:, (K if lo == 0 else 0):][:, :N])
                assert torch.equal(store, before)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 9, 300, 700])
@pytest.mark.parametrize("H", [200, 201])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_norm_of_columns_of_one_buffer_in_place(T, H, dtype):
    """Stream, block and gate side by side in one buffer, the stream updated in place."""
    g = _gen(T + H)
    store = torch.randn((T, 2 * H + 1), generator=g, device="cuda").to(dtype)
    gain = torch.ones(H, device="cuda")
    for order in ((0, H), (H, 0)):
        r, y, gate = store[:, order[0]:order[0] + H], store[:, order[1]:order[1] + H], store[:, 2 * H:]
        before = store.clone()
        # out of place, from rows of the same alignment: the order of a row's sum goes by it
        want, x = okc.block_norm(before[:, order[0]:order[0] + H], before[:, order[1]:order[1] + H], post_gain=gain, gate=before[:, 2 * H:], pre_gain=gain, out="f32",
                                 residual_out=torch.empty_like(store)[:, order[0]:order[0] + H])
        r2, x2 = okc.block_norm(r, y, post_gain=gain, gate=gate, pre_gain=gain, out="f32", residual_out=r)
        assert r2 is r and torch.equal(r, want) and torch.equal(x, x2)
        r.copy_(before[:, order[0]:order[0] + H])
        assert torch.equal(store, before)
