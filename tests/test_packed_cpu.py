"""Packed batches without a GPU: what is refused before any device call, and the 64-bit definitions
that the GPU tests go by against an independent restatement."""
import ctypes as C

import numpy as np
import torch

from tests import numpy_ref
from tests import packed_ref as ref


def test_null_handles_are_refused():
    from tinylama_b200 import _lib
    L = _lib.lib
    x = C.c_void_p(256)
    k, v = C.c_void_p(), C.c_void_p()
    calls = [
        L.tl_kv_device(None, 0, 0, C.byref(k), C.byref(v)),
        L.tl_packed_reserve(None, 1, 1),
        L.tl_qk_norm_rope_append(None, 0, 0, 1, 1, x, x, 0, 0, x, 64, x, 64, x, 64, None, None, 1e-5, None, x, None),
        L.tl_prefill_packed(None, 0, 0, 1, 1, x, x, None, 0, 0, 0, x, x, None),
        L.tl_decode_shared(None, 0, 0, 1, x, None, None, 0, 0, 0, x, x, None),
    ]
    assert calls == [_lib.TL_ERR_INVALID] * len(calls)
    assert b"NULL" in L.tl_last_error()


def test_attention_definition_matches_the_reference_restatement():
    rng = np.random.default_rng(0)
    H, K, D, n, first = 4, 2, 64, 5, 3
    q, k, v = (rng.standard_normal((x * D, m)) for x, m in ((H, n), (K, n + first), (K, n + first)))
    want = numpy_ref.attention(q, k, v, H, K, D, first + np.arange(n), n + first)
    heads = [torch.from_numpy(x.reshape(-1, D, x.shape[1])) for x in (q, k, v)]
    out, spread, _ = ref.attention(heads[0].permute(2, 0, 1), heads[1].transpose(1, 2), heads[2].transpose(1, 2), first)
    assert np.allclose(out.permute(1, 2, 0).reshape(H * D, n).numpy(), want, atol=1e-12)
    assert (spread >= out.abs() - 1e-12).all()


def test_rows_without_keys_are_zero():
    out, _, _ = ref.attention(torch.ones(2, 2, 4), torch.ones(1, 0, 4), torch.ones(1, 0, 4), -1)
    assert (out == 0).all()
    out, _, _ = ref.attention(torch.ones(1, 2, 4), torch.ones(1, 3, 4), torch.full((1, 3, 4), 7.0), -1)
    assert (out == 0).all()


def test_rotation_definition_matches_the_reference_restatement():
    rng = np.random.default_rng(1)
    H, D, rd, n = 3, 64, 32, 6
    x = rng.standard_normal((H * D, n)).astype(np.float32)
    pos = np.array([0, 1, 5, 100, 7, 2])
    i = np.arange(rd // 2)
    theta = np.power(np.float32(1) / np.float32(10000.0), (2 * i).astype(np.float32) / np.float32(rd))
    want = numpy_ref.rope_cols(x, H, D, rd, 10000.0, pos)
    got, size = ref.norm_rope(torch.from_numpy(x.reshape(H, D, n)).permute(2, 0, 1), None, 0.0, torch.from_numpy(pos),
                              torch.from_numpy(theta), rd)
    # the definition's angle is rounded to float32, the restatement's is not: up to 100 * 2^-24
    assert np.allclose(got.permute(1, 2, 0).reshape(H * D, n).numpy(), want, atol=100 * 2.0 ** -24 * 4)
    assert (size >= got.abs() - 1e-12).all()


def test_norm_definition():
    x = torch.tensor([[[3.0, 4.0]]], dtype=torch.float32)
    y, _ = ref.norm_rope(x, torch.tensor([2.0, 1.0]), 0.0, torch.zeros(1), torch.zeros(0), 0)
    assert torch.allclose(y, torch.tensor([[[6.0, 4.0]]], dtype=torch.float64) / np.sqrt(12.5))


def test_the_rms_limit_sees_a_lost_part():
    """Attention in 64 bits from operands that kept two bf16 parts of three is outside the limit, whichever
    operand it is; the same in 32 bits throughout is inside."""
    g = torch.Generator().manual_seed(3)
    n, H, K, D = 96, 4, 2, 64
    q = torch.randn(n, H, D, generator=g) * 1.5
    k, v = (torch.randn(K, n, D, generator=g) for _ in range(2))
    want, _, _ = ref.attention(q, k, v, 0)
    for lost in ((ref.two_parts(q), k, v), (q, ref.two_parts(k), v), (q, k, ref.two_parts(v))):
        assert ref.rms_error(ref.attention(*lost, 0)[0], want) > 2 * ref.RMS32
    s = torch.einsum("nhd,hmd->nhm", q, k.repeat_interleave(H // K, 0)) / D ** 0.5
    s = s.masked_fill((torch.arange(n)[None] > torch.arange(n)[:, None])[:, None], -float("inf"))
    got = torch.einsum("nhm,hmd->nhd", torch.softmax(s, -1), v.repeat_interleave(H // K, 0))
    assert ref.rms_error(got, want) < ref.RMS32 / 2
