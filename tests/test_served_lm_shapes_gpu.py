"""
The operators of a served language model at sizes where another form of their kernels runs: many requests (several key heads in a tile), every number of
heads per key head, many and few rows of logits, rows shared by CTAs, tiles of many tokens. Against 64 bits, with the tolerances derived beside the plain tests.
"""

import pytest
import torch

import test_norm_rope
import test_paged
import test_token_log_probs

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])


@TYPES
@pytest.mark.parametrize("n,h,hk,d,page", [(100, 8, 8, 64, 16), (60, 40, 8, 96, 8), (120, 32, 4, 128, 1), (80, 64, 4, 64, 7), (50, 128, 4, 24, 16), (90, 12, 12, 64, 64), (170, 8, 4, 256, 16),
                                           (40, 14, 14, 32, 16), (300, 6, 1, 80, 3), (75, 6, 2, 128, 16), (38, 24, 8, 48, 100)])
def test_attention_of_many_requests(n, h, hk, d, page, dtype):
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 40, (n,), generator=g)
    lens[torch.randperm(n, generator=g)[:3]] = torch.tensor([300, 129, 513])
    test_paged._attend(n, h, hk, d, page, lens.tolist(), dtype, seed=n)
    test_paged._attend(n, h, hk, d, page, (lens % 3).tolist(), dtype, layout="tokens", seed=n + 1)


@TYPES
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 9, 17])
def test_attention_heads_of_a_key_head(group, dtype):
    for d in (64, 128, 256):
        test_paged._attend(3, 2 * group, 2, d, 16, [2100, 0, 77], dtype, seed=group + d)


@TYPES
@pytest.mark.parametrize("rows,v,top", [(1200, 80, 8), (1500, 1001, 20), (1184, 257, 32), (200, 10001, 24), (400, 9000, 13), (500, 8200, 28), (600, 1001, 24), (148, 20000, 12), (10, 20011, 24),
                                        (10, 20011, 32), (297, 16384, 1), (1183, 8191, 3)])
def test_log_probs_by_rows(rows, v, top, dtype):
    x, t = test_token_log_probs._rows(rows, v, dtype)
    test_token_log_probs._check(x, t, top)
    x[:, v // 3:] = torch.finfo(dtype).min  # masked labels: many equal ones
    x[0] = 0.0
    t = t % (v // 3)
    test_token_log_probs._check(x, t, top, entropy=False)


@TYPES
@pytest.mark.parametrize("rows,v,top,pad", [(25, 40011, 3, 5), (4, 128000, 8, 0), (180, 9001, 32, 0), (700, 513, 0, 0), (2400, 333, 4, 1), (60, 8192, 5, 0)])
def test_log_probs_gradient_by_rows(rows, v, top, pad, dtype):
    test_token_log_probs.test_gradient(dtype, rows, v, top, pad)


ROTATED = [(300, 32, 8, 128, 128), (702, 16, 2, 128, 64), (2600, 4, 4, 32, 16), (5000, 5, 3, 64, 64), (8191, 3, 2, 128, 32), (19, 40, 24, 64, 64), (1, 300, 4, 16, 16), (4700, 1, 1, 64, 64),
           (1300, 24, 0, 256, 128), (25001, 2, 1, 64, 64)]


@TYPES
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotation_by_tokens(interleaved, dtype):
    for case in ROTATED:
        test_norm_rope._forward("cuda", dtype, *case, interleaved, True)
        test_norm_rope._forward("cuda", dtype, *case, interleaved, False, fused=False)


@TYPES
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("norm", [True, False])
def test_rotation_gradient_by_tokens(interleaved, norm, dtype, monkeypatch):
    monkeypatch.setattr(test_norm_rope, "CASES", ROTATED)
    test_norm_rope.test_gradient(dtype, interleaved, norm)


@TYPES
@pytest.mark.parametrize("n,hq,hk", [(300, 32, 8), (700, 5, 3), (2600, 4, 4), (30, 40, 40)])
def test_rotation_to_cache_by_tokens(n, hq, hk, dtype):
    test_norm_rope.test_to_cache(dtype, n, hq, hk, 64, 64, 16, "heads")
