"""Decode attention over the 8-bit cache where scores, K scales or queries are very large or very small: every form of
it, against the 64-bit forms of kv8_ref."""
import numpy as np
import pytest

import kv8_ref
from test_gpu_kv8 import Cache, check, dev, run_decode

pytestmark = pytest.mark.gpu

# rows, own keys, prefix, kv heads, launches: one launch; split over the GPU; behind a short prefix; behind a long one
# with own keys in one launch, and split
FORMS = [(3, 300, 0, 2, 1), (3, 80001, 0, 1, 2), (3, 50, 200, 2, 1), (130, 40, 1000, 8, 5), (130, 1100, 900, 8, 6)]


def signed_keys(c, pattern, positive, k_scale):
    """K codes pattern[kv head] or their negative, all of one scale.  Every third key is a positive one where
    `positive`, the first one among them.  Returns the signs."""
    import torch
    sign = np.where(positive & (np.arange(c.tokens) % 3 == 0), 1, -1).astype(np.int8)
    c.k[:] = dev(sign[None, None, :, None] * pattern[None, :, None, :])
    c.ks[:] = k_scale
    torch.cuda.synchronize()
    return sign


def check_signed_keys(ctx, B, n, P, n_kv, launches, hd, group, k_scale, sizes):
    """Keys with one and the same score, and keys with its negative, too far below for anything but the clamped
    weight w(-87.3): the answer (sum v + w sum v') / (n + w n') holds whatever the scores' size and rounding.  The
    tolerance is kv8_ref.attend's without its term for the scores."""
    rs = np.random.RandomState(hd + group)
    pattern = rs.randint(-127, 128, (n_kv, hd)).astype(np.int8)
    pattern[:, 0] = 127
    lens = rs.randint(1, n + 1, B)
    lens[:3] = n, 1, 0 if P else 2
    low = float(kv8_ref.weight(np.array(-87.3)))
    c = Cache(ctx, B, n, n_kv, hd).fill(rs, lens)
    p = Cache(ctx, 1, max(P, 1), n_kv, hd).fill(rs, [P])
    for positive_own in (False, True) if P else (True,):
        # largest scores on one side only: two forms of the products need not agree to the last bit
        sides = [(c, signed_keys(c, pattern, positive_own, k_scale))]
        if P:
            sides.insert(0, (p, signed_keys(p, pattern, not positive_own, k_scale)))
        arrays = [(x.arrays(), s) for x, s in sides]
        for size in sizes:
            q = pattern.repeat(group, 0)[None] / 127.0 * size * (1 + rs.rand(B, n_kv * group, 1))
            before = ctx.launch_count()
            got = run_decode(ctx, c, q.astype(np.float32), None, lens, n, prefix=p if P else None, prefix_len=P)
            assert ctx.launch_count() == before + launches
            for b in (0, 1, 2, B - 1):
                # (arrays, slot, keys, signs) of the row's parts
                parts = [(a, 0 if x is p else b, P if x is p else lens[b], s) for (x, _), (a, s) in zip(sides, arrays)]
                for g in range(0, n_kv, 3):
                    codes = np.concatenate([a[2][s, g, :m] for a, s, m, _ in parts]).astype(np.float64)
                    scale = np.concatenate([a[3][s, g, :m] for a, s, m, _ in parts]).astype(np.float64)
                    sign = np.concatenate([sg[:m] for _, _, m, sg in parts])
                    # without a positive key in sight the negative ones are the largest
                    w = np.where((sign > 0) | (sign.max() < 0), 1.0, low)
                    v, total = codes * scale[:, None], w.sum()
                    rel = 2 * (8 + 64 + len(w) / 64) * 2.0 ** -24
                    tol = rel * (w @ np.abs(v)) / total + 2.0 ** -24 * scale.max() * np.abs(codes).sum(0) / total
                    h = slice(g * group, (g + 1) * group)
                    check(got[b, h], np.broadcast_to(w @ v / total, (group, hd)),
                          np.broadcast_to(tol, (group, hd)))
    assert ctx.device_status() == 0


@pytest.mark.parametrize("group", [1, 4, 8, 16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("B,n,P,n_kv,launches", FORMS)
def test_the_largest_score_has_weight_one(ctx, B, n, P, n_kv, launches, hd, group):
    check_signed_keys(ctx, B, n, P, n_kv, launches, hd, group, 0.5, (1.0, 1e2, 1e4, 1e6, 1e9))


@pytest.mark.parametrize("hd,group", [(64, 8), (64, 16), (128, 4)])
@pytest.mark.parametrize("B,n,P,n_kv,launches", FORMS)
@pytest.mark.parametrize("k_scale,sizes", [(1e30, (1.0, 1e-29)), (2e36, (1e-3, 1e-29)),
                                           (1e-38, (1e38,))])
def test_k_scales_at_both_ends(ctx, B, n, P, n_kv, launches, hd, group, k_scale, sizes):
    """Scores in fp32's range (up to 1e36) from K scales up to the largest that a finite row can have."""
    check_signed_keys(ctx, B, n, P, n_kv, launches, hd, group, k_scale, sizes)


@pytest.mark.parametrize("B,n,P,n_kv,launches", FORMS)
@pytest.mark.parametrize("hd", [64, 128])
def test_large_k_scales_with_moderate_scores(ctx, B, n, P, n_kv, launches, hd):
    rs = np.random.RandomState(B + hd)
    n_heads = 2 * n_kv
    lens = rs.randint(n // 2, n + 1, B)
    c = Cache(ctx, B, n, n_kv, hd).fill(rs, lens)
    p = Cache(ctx, 1, max(P, 1), n_kv, hd).fill(rs, [P])
    for x in (c, p):
        x.ks *= 1e30
    q = (rs.randn(B, n_heads, hd) * 1e-29).astype(np.float32)
    got = run_decode(ctx, c, q, None, lens, n, prefix=p if P else None, prefix_len=P)
    a, pa = c.arrays(), p.arrays()
    some = [0, 1, B - 1]
    keys = [([(pa, 0, P)] if P else []) + [(a, b, lens[b])] for b in some]
    check(got[some], *kv8_ref.attend_rows(q[some], n_kv, keys))
    assert np.isfinite(got).all()


@pytest.mark.parametrize("B,n,P,n_kv,launches", FORMS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [1e31, 1e33, 1e36])
def test_tiny_queries_and_large_keys(ctx, B, n, P, n_kv, launches, hd, size):
    """Queries down to 2^-120 keep their digits."""
    rs = np.random.RandomState(B + hd)
    n_heads = 2 * n_kv
    lens = rs.randint(n // 2, n + 1, B)
    some = [0, 1, B - 1]
    c = Cache(ctx, B, n, n_kv, hd).fill(rs, [m if b in some else 0 for b, m in enumerate(lens)])
    p = Cache(ctx, 1, max(P, 1), n_kv, hd).fill(rs, [P])
    for x in (c, p):
        x.ks *= size
    q = (rs.randn(B, n_heads, hd) / size).astype(np.float32)
    before = ctx.launch_count()
    got = run_decode(ctx, c, q, None, lens, n, prefix=p if P else None, prefix_len=P)
    assert ctx.launch_count() == before + launches
    a, pa = c.arrays(), p.arrays()
    keys = [([(pa, 0, P)] if P else []) + [(a, b, lens[b])] for b in some]
    check(got[some], *kv8_ref.attend_rows(q[some], n_kv, keys))
