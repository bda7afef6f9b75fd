"""The 8-bit KV cache on the GPU: quantising writes, read-back and decode attention with and without a shared
prefix, against the 64-bit forms of kv8_ref (whose attend() derives the tolerances)."""
import numpy as np
import pytest

import kv8_ref

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -24  # half a step of fp32


def dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Cache:
    """Device arrays of a cache (codes 55 and scales NaN where nothing is written) and its handle."""

    def __init__(self, ctx, slots, tokens, n_kv, hd):
        import torch

        import smallmind_b200 as sm
        self.k, self.v = (torch.full((slots, n_kv, tokens, hd), 55, dtype=torch.int8, device="cuda") for _ in "kv")
        self.ks, self.vs = (torch.full((slots, n_kv, tokens), float("nan"), device="cuda") for _ in "kv")
        self.n_kv, self.hd, self.tokens, self.slots = n_kv, hd, tokens, slots
        self.h = sm.KV8Cache(ctx, self.k.data_ptr(), self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(), slots,
                             tokens, n_kv, hd)

    def fill(self, rs, lens):
        """Positions [0, lens[slot]) of each slot: codes and scales of normal values."""
        import torch
        for s, n in enumerate(lens):
            for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
                x = rs.randn(self.n_kv, n, self.hd).astype(np.float32)
                x[..., ::21] *= 4
                if n:
                    c, f = kv8_ref.quantize(x)
                    codes[s, :, :n], scales[s, :, :n] = dev(c), dev(f)
        torch.cuda.synchronize()
        return self

    def arrays(self):
        return tuple(t.cpu().numpy() for t in (self.k, self.ks, self.v, self.vs))


def check(got, want, tol):
    """Values of rows that are left alone (want NaN) are checked by the caller."""
    live = ~np.isnan(want)
    err = np.abs(got.astype(np.float64) - want)[live]
    over = err - tol[live]
    assert not np.isnan(got[live]).any()
    assert over.max(initial=-1) <= 0, (over.max(), err.max(), np.argmax(over))


# ---------------------------------------------------------------- write and read
@pytest.mark.parametrize("n_kv,hd", [(1, 64), (3, 64), (4, 64), (8, 128), (2, 128)])
@pytest.mark.parametrize("n", [1, 2, 7, 130])
def test_write_is_exact_and_touches_nothing_else(ctx, n_kv, hd, n):
    import torch
    rs = np.random.RandomState(n * 10 + n_kv)
    slots, tokens = 3, n + 5
    c = Cache(ctx, slots, tokens, n_kv, hd)
    stride = (2 * n_kv + 2) * hd + 8
    rows = (rs.randn(n, stride) * 10.0 ** rs.randint(-3, 3, (n, 1))).astype(np.float32)
    rows[0, :hd] = 0  # a head of zeros
    seq = rs.randint(0, slots, n).astype(np.int32)
    pos = rs.permutation(tokens)[:n].astype(np.int32)
    before = c.arrays()
    d, ds, dp = dev(rows), dev(seq), dev(pos)
    torch.cuda.synchronize()
    at_v = (n_kv + 1) * hd
    c.h.write_device(d.data_ptr(), d.data_ptr() + 4 * at_v, ds.data_ptr(), dp.data_ptr(), n, row_stride=stride)
    ctx.sync()
    after = c.arrays()
    want = [a.copy() for a in before]
    for first, i in ((0, 0), (at_v, 2)):
        x = rows[:, first:first + n_kv * hd].reshape(n, n_kv, hd)
        codes, scale = kv8_ref.quantize(x)
        want[i][seq, :, pos], want[i + 1][seq, :, pos] = codes, scale
    for a, w in zip(after, want):
        assert np.array_equal(a, w, equal_nan=a.dtype == np.float32)


def test_write_rounds_exactly_next_to_the_borders(ctx):
    """Values one ulp around (and, where fp32 has them, on) the borders between codes, at scales from the
    subnormal range to the largest; the wanted codes come from exact rational arithmetic."""
    import torch
    from fractions import Fraction
    rs = np.random.RandomState(7)
    n, n_kv, hd = 64, 2, 64
    x = np.empty((n, n_kv, hd), np.float32)
    for r in range(n):
        for g in range(n_kv):
            peak = np.float32(rs.rand() + 0.5) * np.float32(2.0) ** np.float32([-149, -140, -126, -100, -20, 0, 3, 120][r % 8])
            s = np.float32(np.float64(peak) / 127.0)
            half = (rs.randint(-127, 127, hd) + 0.5) * np.float64(s)
            x[r, g] = np.clip(half, -np.float64(peak), np.float64(peak)).astype(np.float32)
            x[r, g, 0::3] = np.nextafter(x[r, g, 0::3], np.float32(np.inf))
            x[r, g, 1::3] = np.nextafter(x[r, g, 1::3], np.float32(-np.inf))
            x[r, g] = np.clip(x[r, g], -peak, peak)
            x[r, g, 5] = peak
    c = Cache(ctx, 1, n, n_kv, hd)
    d, ds, dp = dev(x), dev(np.zeros(n, np.int32)), dev(np.arange(n, dtype=np.int32))
    torch.cuda.synchronize()
    c.h.write_device(d.data_ptr(), d.data_ptr(), ds.data_ptr(), dp.data_ptr(), n)
    ctx.sync()
    codes, scale = c.arrays()[:2]
    want, want_scale = kv8_ref.quantize(x)
    assert np.array_equal(scale[0].T, want_scale)
    assert np.array_equal(codes[0].transpose(1, 0, 2), want)
    for r in range(0, n, 5):
        for g in range(n_kv):
            s = Fraction(float(want_scale[r, g]))
            for i in range(hd):
                exact = 0 if s == 0 else max(-127, min(127, round(Fraction(float(x[r, g, i])) / s)))
                assert codes[0, g, r, i] == exact


def test_write_of_non_finite_heads_reads_back_as_nan(ctx):
    import torch
    n_kv, hd = 2, 64
    x = np.random.RandomState(0).randn(3, n_kv, hd).astype(np.float32)
    x[0, 1, 3], x[1, 0, 63], x[2, 1, 0] = np.inf, np.nan, -np.inf
    c = Cache(ctx, 1, 4, n_kv, hd)
    d, ds, dp = dev(x), dev(np.zeros(3, np.int32)), dev(np.arange(3, dtype=np.int32))
    out = torch.zeros(2, 3, n_kv, hd, device="cuda")
    torch.cuda.synchronize()
    c.h.write_device(d.data_ptr(), d.data_ptr(), ds.data_ptr(), dp.data_ptr(), 3)
    c.h.read_device(ds.data_ptr(), dp.data_ptr(), 3, out[0].data_ptr(), out[1].data_ptr())
    ctx.sync()
    got = out.cpu().numpy()
    bad = ~np.isfinite(x).all(-1)
    assert np.isnan(got[:, bad]).all() and np.isfinite(got[:, ~bad]).all()
    assert not c.arrays()[0][0, 1, 0].any()


@pytest.mark.parametrize("offset,stride_extra", [(0, 0), (1, 0), (0, 3), (2, 2), (4, 4)])
def test_rows_of_any_alignment(ctx, offset, stride_extra):
    """fp32 rows that start on any 4-byte boundary, with any stride."""
    import torch
    rs = np.random.RandomState(3)
    n, n_kv, hd = 9, 3, 128
    w = n_kv * hd
    stride = w + stride_extra
    flat = rs.randn(offset + n * stride + 8).astype(np.float32)
    c = Cache(ctx, 2, 16, n_kv, hd)
    seq, pos = rs.randint(0, 2, n).astype(np.int32), rs.permutation(16)[:n].astype(np.int32)
    d, ds, dp = dev(flat), dev(seq), dev(pos)
    out = torch.full((flat.size,), 7.0, device="cuda")
    torch.cuda.synchronize()
    c.h.write_device(d.data_ptr() + 4 * offset, d.data_ptr() + 4 * offset, ds.data_ptr(), dp.data_ptr(), n,
                     row_stride=stride)
    c.h.read_device(ds.data_ptr(), dp.data_ptr(), n, None, out.data_ptr() + 4 * offset, row_stride=stride)
    ctx.sync()
    got = out.cpu().numpy()
    want = np.full_like(got, 7.0)
    for r in range(n):
        at = offset + r * stride
        codes, scale = kv8_ref.quantize(flat[at:at + w].reshape(n_kv, hd))
        want[at:at + w] = (codes.astype(np.float32) * scale[:, None]).reshape(-1)
    assert np.array_equal(got, want)


def test_padding_and_out_of_range_rows_are_left_alone():
    """Rows with a negative id are skipped silently, rows outside the cache with an error status."""
    import torch

    import smallmind_b200 as sm
    ctx = sm.CudaContext(0)
    n_kv, hd = 2, 64
    c = Cache(ctx, 3, 8, n_kv, hd)
    rs = np.random.RandomState(1)
    x = dev(rs.randn(6, n_kv, hd).astype(np.float32))
    out = torch.full((2, 6, n_kv, hd), 3.0, device="cuda")
    before = c.arrays()
    ds, dp = dev(np.full(6, -1, np.int32)), dev(np.array([0, 99, -5, 1, 2, 3], np.int32))
    torch.cuda.synchronize()
    c.h.write_device(x.data_ptr(), x.data_ptr(), ds.data_ptr(), dp.data_ptr(), 6)
    c.h.read_device(ds.data_ptr(), dp.data_ptr(), 6, out[0].data_ptr(), out[1].data_ptr())
    assert ctx.device_status() == 0
    assert (out == 3.0).all()
    bad_s, bad_p = dev(np.array([3, 0, 1, 2, 2 ** 31 - 1, 0], np.int32)), dev(np.array([0, 8, -1, 1, 0, 2 ** 31 - 1], np.int32))
    torch.cuda.synchronize()
    c.h.write_device(x.data_ptr(), x.data_ptr(), bad_s.data_ptr(), bad_p.data_ptr(), 6)
    assert ctx.device_status() == -2
    after = c.arrays()
    for a, b in zip(after, before):
        a[2, :, 1] = b[2, :, 1]  # the one row in range
        assert np.array_equal(a, b, equal_nan=a.dtype == np.float32)
    c.h.read_device(bad_s.data_ptr(), bad_p.data_ptr(), 6, out[0].data_ptr(), out[1].data_ptr())
    ctx.sync()
    assert (out[:, [0, 1, 2, 4, 5]] == 3.0).all() and not (out[:, 3] == 3.0).any()
    ctx.close()


def test_empty_calls_do_nothing(ctx):
    c = Cache(ctx, 1, 8, 2, 64)
    n = ctx.launch_count()
    c.h.write_device(0, 0, 0, 0, 0)
    c.h.read_device(0, 0, 0, None, None)
    c.h.attention_decode_device(0, None, 0, 0, 4, 0)
    c.h.attention_shared_device(0, c.h, 0, 3, None, 0, 0, 4, 0)
    assert ctx.launch_count() == n


# ---------------------------------------------------------------- attention
def run_decode(ctx, c, q, seq, lens, max_len, prefix=None, prefix_seq=0, prefix_len=0, q_stride=None):
    """q [B, n_heads, hd] (or rows of q_stride floats); returns out [B, n_heads, hd], 5.0 where nothing was written."""
    import torch
    B, n_heads = q.shape[0], q.shape[1]
    dq, dl = dev(q), dev(np.asarray(lens, np.int32))
    if q_stride is not None:
        wide = torch.full((B * q_stride + 1,), float("nan"), device="cuda")
        for b in range(B):
            wide[1 + b * q_stride:1 + b * q_stride + n_heads * c.hd] = dq[b].reshape(-1)
        dq = wide[1:]
    ds = None if seq is None else dev(np.asarray(seq, np.int32))
    out = torch.full((B, n_heads, c.hd), 5.0, device="cuda")
    torch.cuda.synchronize()
    sp = None if ds is None else ds.data_ptr()
    if prefix is None:
        c.h.attention_decode_device(dq.data_ptr(), sp, dl.data_ptr(), B, n_heads, out.data_ptr(), max_len=max_len,
                                    q_stride=q_stride)
    else:
        c.h.attention_shared_device(dq.data_ptr(), prefix.h, prefix_seq, prefix_len, sp, dl.data_ptr(), B, n_heads,
                                    out.data_ptr(), max_len=max_len, q_stride=q_stride)
    ctx.sync()
    return out.cpu().numpy()


@pytest.mark.parametrize("n_heads,n_kv", [(1, 1), (2, 1), (3, 1), (4, 2), (9, 3), (10, 2), (7, 1), (8, 1), (32, 4),
                                          (9, 1), (16, 1), (24, 2), (8, 8)])
@pytest.mark.parametrize("hd", [64, 128])
def test_decode_groups_and_short_lengths(ctx, n_heads, n_kv, hd):
    rs = np.random.RandomState(n_heads * 7 + n_kv)
    lens = [1, 0, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100]
    c = Cache(ctx, len(lens), 100, n_kv, hd).fill(rs, lens)
    q = rs.randn(len(lens), n_heads, hd).astype(np.float32)
    want, tol = kv8_ref.attend_rows(q, n_kv, [[(c.arrays(), b, n)] for b, n in enumerate(lens)])
    got = run_decode(ctx, c, q, None, lens, 100)
    check(got, want, tol)
    assert not got[1].any()


@pytest.mark.parametrize("lens,n_heads,n_kv,hd", [
    ([1000], 32, 4, 64), ([5001], 9, 3, 64), ([777, 3, 2048, 1], 32, 4, 64), ([20000], 16, 1, 128),
    ([4097, 1], 32, 8, 128), ([300] * 40, 8, 2, 64), ([1 + 61 * i % 500 for i in range(90)], 12, 4, 128)])
def test_decode_long_and_batched(ctx, lens, n_heads, n_kv, hd):
    rs = np.random.RandomState(len(lens) + n_heads)
    c = Cache(ctx, len(lens) + 1, max(lens) + 3, n_kv, hd)
    seq = rs.permutation(len(lens) + 1)[:len(lens)].astype(np.int32)
    held = np.zeros(len(lens) + 1, int)
    held[seq] = lens
    c.fill(rs, held)
    q = (rs.randn(len(lens), n_heads, hd) * 2).astype(np.float32)
    a = c.arrays()
    want, tol = kv8_ref.attend_rows(q, n_kv, [[(a, s, n)] for s, n in zip(seq, lens)])
    got = run_decode(ctx, c, q, seq, lens, max(lens))
    check(got, want, tol)
    assert np.array_equal(got, run_decode(ctx, c, q, seq, lens, max(lens)))  # no order of sums is left to chance
    check(run_decode(ctx, c, q, seq, lens, max(lens) + 3), want, tol)  # a bound above the lengths


def test_decode_padding_rows_strided_q_and_one_slot_for_two_rows(ctx):
    rs = np.random.RandomState(11)
    c = Cache(ctx, 4, 50, 2, 64).fill(rs, [50, 20, 0, 33])
    q = rs.randn(6, 8, 64).astype(np.float32)
    seq, lens = [1, -1, 3, 3, -7, 0], [20, 999, 33, 12, -4, 50]
    a = c.arrays()
    keys = [None if s < 0 else [(a, s, n)] for s, n in zip(seq, lens)]
    want, tol = kv8_ref.attend_rows(q, 2, keys)
    for stride in (None, 8 * 64 + 3):
        got = run_decode(ctx, c, q, seq, lens, 50, q_stride=stride)
        check(got, want, tol)
        assert (got[[1, 4]] == 5.0).all()
    want, tol = kv8_ref.attend_rows(q, 2, [k if k is None else [(a, 0, 7)] + k for k in keys])
    got = run_decode(ctx, c, q, seq, lens, 50, prefix=c, prefix_seq=0, prefix_len=7)
    check(got, want, tol)
    assert (got[[1, 4]] == 5.0).all()
    assert ctx.device_status() == 0


def test_bad_slots_and_lengths_set_the_status():
    import smallmind_b200 as sm
    rs = np.random.RandomState(5)
    q = rs.randn(4, 4, 64).astype(np.float32)
    for bad_seq, bad_len in ((4, 3), (2 ** 31 - 1, 3), (1, 11), (1, -1), (1, 2 ** 31 - 1)):
        for shared in (False, True):
            ctx = sm.CudaContext(0)
            c = Cache(ctx, 4, 12, 2, 64).fill(rs, [12, 12, 12, 12])
            a = c.arrays()
            lens, seq = [10, bad_len, 0, 5], [0, bad_seq, 2, 3]
            more = dict(prefix=c, prefix_seq=3, prefix_len=12) if shared else {}
            got = run_decode(ctx, c, q, seq, lens, 10, **more)
            head = [(a, 3, 12 if shared else 0)]
            want, tol = kv8_ref.attend_rows(q, 2, [head + [(a, 0, 10)], None, head, head + [(a, 3, 5)]])
            check(got, want, tol)
            assert (got[1] == 5.0).all()
            assert ctx.device_status() == -2
            ctx.close()


def test_extreme_values(ctx):
    """Scores far apart (the clamped weight), equal scores, zero q, zero keys, scales of very different size."""
    rs = np.random.RandomState(2)
    n_kv, hd, n = 2, 64, 70
    c = Cache(ctx, 1, n, n_kv, hd).fill(rs, [n])
    q = rs.randn(1, 8, hd).astype(np.float32)
    q[0, 1] *= 100  # differences of scores in the hundreds: most weights at the clamp
    q[0, 2] = 0
    q[0, 3] *= 1e-20
    q[0, 5] *= 1e4
    q[0, 6, 1:] = 0
    c.ks[0, 1, ::7] = 0
    c.vs[0, 0, 5] *= 1000
    c.vs[0, 1] *= 1e-6
    c.k[0, 0, 40:] = 0
    want, tol = kv8_ref.attend_rows(q, n_kv, [[(c.arrays(), 0, n)]])
    check(run_decode(ctx, c, q, None, [n], n), want, tol)
    want2, tol2 = kv8_ref.attend_rows(q, n_kv, [[(c.arrays(), 0, 60), (c.arrays(), 0, n)]])
    check(run_decode(ctx, c, q, None, [n], n, prefix=c, prefix_len=60), want2, tol2)


def test_nan_reaches_exactly_the_outputs_that_depend_on_it(ctx):
    rs = np.random.RandomState(4)
    n_kv, hd = 2, 64
    c = Cache(ctx, 3, 90, n_kv, hd).fill(rs, [90, 80, 80])
    q = rs.randn(3, 8, hd).astype(np.float32)
    q[2, 5, 9] = np.nan
    c.ks[0, 1, 17] = float("nan")
    c.vs[1, 0, 3] = float("nan")
    c.ks[1, 1, 80:] = float("nan")  # behind the length: not seen
    got = run_decode(ctx, c, q, None, [90, 80, 80], 90)
    nan = np.isnan(got).all(-1)
    assert np.array_equal(nan, np.isnan(got).any(-1))
    want = np.zeros((3, 8), bool)
    want[0, 4:], want[1, :4], want[2, 5] = True, True, True
    assert np.array_equal(nan, want)
    # through a shared prefix: every sequence sees it
    p = Cache(ctx, 1, 40, n_kv, hd).fill(rs, [40])
    p.ks[0, 0, 39] = float("nan")
    got = run_decode(ctx, c, q, None, [10, 0, 2], 90, prefix=p, prefix_len=40)
    assert np.isnan(got[:, :4]).all() and np.isfinite(got[:2, 4:]).all()
    assert np.isnan(got[2, 5]).all() and np.isfinite(got[2, [4, 6, 7]]).all()
    got = run_decode(ctx, c, q, None, [10, 0, 2], 90, prefix=p, prefix_len=39)
    assert np.isfinite(got[:2]).all()


@pytest.mark.parametrize("n_heads,n_kv,hd", [(9, 3, 64), (32, 4, 64), (8, 8, 64), (16, 1, 64), (32, 8, 128),
                                             (16, 1, 128), (3, 3, 128), (5, 1, 128)])
@pytest.mark.parametrize("B,prefix_len", [(1, 1), (2, 0), (3, 129), (17, 128), (33, 500), (64, 1027)])
def test_shared_prefix(ctx, n_heads, n_kv, hd, B, prefix_len):
    rs = np.random.RandomState(B + prefix_len + n_heads)
    lens = rs.randint(0, 70, B)
    lens[0] = 0
    p = Cache(ctx, 2, max(1, prefix_len) + 9, n_kv, hd).fill(rs, [0, prefix_len])
    c = Cache(ctx, B, 70, n_kv, hd).fill(rs, lens)
    q = rs.randn(B, n_heads, hd).astype(np.float32)
    a, pa = c.arrays(), p.arrays()
    want, tol = kv8_ref.attend_rows(q, n_kv, [[(pa, 1, prefix_len), (a, b, n)] for b, n in enumerate(lens)])
    got = run_decode(ctx, c, q, None, lens, 70, prefix=p, prefix_seq=1, prefix_len=prefix_len)
    check(got, want, tol)
    if prefix_len == 0:
        assert not got[0].any()


@pytest.mark.parametrize("n_heads,n_kv,hd,B,prefix_len,longest", [
    (32, 4, 64, 64, 3001, 90), (9, 3, 64, 90, 2705, 33), (8, 8, 64, 40, 2688, 0), (32, 8, 128, 17, 3100, 700),
    (16, 1, 128, 130, 2817, 40), (7, 1, 64, 260, 6500, 5), (12, 4, 128, 150, 1500, 1), (2, 2, 128, 300, 700, 64)])
def test_long_shared_prefix(ctx, n_heads, n_kv, hd, B, prefix_len, longest):
    """Batches times prefixes beyond what a cluster per row reads: the matrix form."""
    rs = np.random.RandomState(B + prefix_len)
    lens = rs.randint(0, longest + 1, B)
    lens[0], lens[-1] = 0, longest
    seq = rs.permutation(B + 2)[:B]
    seq[B // 2] = -1
    held = np.zeros(B + 2, int)
    held[seq[seq >= 0]] = lens[seq >= 0]
    p = Cache(ctx, 1, prefix_len, n_kv, hd).fill(rs, [prefix_len])
    c = Cache(ctx, B + 2, max(1, longest), n_kv, hd).fill(rs, held)
    q = (rs.randn(B, n_heads, hd) * np.exp(rs.randn(B, n_heads, 1))).astype(np.float32)
    q[1, 0] = 0
    a, pa = c.arrays(), p.arrays()
    keys = [None if s < 0 else [(pa, 0, prefix_len), (a, s, n)] for s, n in zip(seq, lens)]
    want, tol = kv8_ref.attend_rows(q, n_kv, keys)
    got = run_decode(ctx, c, q, seq, lens, longest, prefix=p, prefix_len=prefix_len, q_stride=n_heads * hd + 1)
    check(got, want, tol)
    assert (got[B // 2] == 5.0).all()
    assert np.array_equal(got, run_decode(ctx, c, q, seq, lens, longest, prefix=p, prefix_len=prefix_len))
    assert ctx.device_status() == 0


def test_long_shared_prefix_nan_and_bad_rows():
    """NaNs of q and of the scales reach what depends on them, bad rows set the status, in the matrix form too."""
    import smallmind_b200 as sm
    ctx = sm.CudaContext(0)
    rs = np.random.RandomState(77)
    n_heads, n_kv, hd, B, P = 32, 4, 64, 70, 2900
    lens = np.full(B, 9)
    p = Cache(ctx, 1, P + 40, n_kv, hd).fill(rs, [P])
    c = Cache(ctx, B, 9, n_kv, hd).fill(rs, lens)
    q = rs.randn(B, n_heads, hd).astype(np.float32)
    q[3, 9, 5], q[4, 1, 0] = np.nan, np.inf
    seq = np.arange(B)
    seq[5], seq[6] = B, -1
    lens[7], lens[8] = 10, -1
    p.ks[0, 3, P - 1] = float("nan")
    c.vs[10, 0, 8] = float("nan")
    got = run_decode(ctx, c, q, seq, lens, 9, prefix=p, prefix_len=P)
    assert (got[[5, 6, 7, 8]] == 5.0).all()
    nan = np.isnan(got).all(-1)
    assert np.array_equal(nan, np.isnan(got).any(-1))
    want = np.zeros((B, n_heads), bool)
    want[:, 24:], want[3, 9], want[4, 1], want[10, :8] = True, True, True, True
    want[[5, 6, 7, 8]] = False
    assert np.array_equal(nan, want)
    assert ctx.device_status() == -2
    ctx.close()


def test_shared_equals_decode_over_a_copied_prefix(ctx):
    """The shared form against the plain decode call over slots that hold the prefix and the own keys in a row."""
    import torch
    rs = np.random.RandomState(21)
    n_heads, n_kv, hd, B, P = 32, 4, 64, 24, 2100
    lens = rs.randint(1, 300, B)
    p = Cache(ctx, 1, P, n_kv, hd).fill(rs, [P])
    c = Cache(ctx, B, 300, n_kv, hd).fill(rs, lens)
    both = Cache(ctx, B, P + 300, n_kv, hd)
    for whole, pre, own in ((both.k, p.k, c.k), (both.v, p.v, c.v), (both.ks, p.ks, c.ks), (both.vs, p.vs, c.vs)):
        whole[:, :, :P], whole[:, :, P:] = pre, own
    torch.cuda.synchronize()
    q = rs.randn(B, n_heads, hd).astype(np.float32)
    one = run_decode(ctx, c, q, None, lens, 300, prefix=p, prefix_len=P)
    two = run_decode(ctx, both, q, None, lens + P, P + 300)
    rows = kv8_ref.attend_rows(q[:2], n_kv, [[(both.arrays(), b, P + lens[b])] for b in range(2)])
    check(one[:2], *rows)
    check(two[:2], *rows)
    assert np.abs(one - two).max() <= 2 * rows[1].max() + 1e-6


def test_offsets_past_32_bits(ctx):
    """Slots and positions whose code offsets exceed 2^31 (a cache of 2.7 G codes)."""
    import torch
    n_kv, hd, tokens, slots = 8, 128, 131072, 20
    c = Cache(ctx, 1, 1, n_kv, hd)
    import smallmind_b200 as sm
    k, v = (torch.zeros(slots, n_kv, tokens, hd, dtype=torch.int8, device="cuda") for _ in "kv")
    ks, vs = (torch.zeros(slots, n_kv, tokens, device="cuda") for _ in "kv")
    c.k, c.v, c.ks, c.vs, c.tokens, c.slots = k, v, ks, vs, tokens, slots
    c.h = sm.KV8Cache(ctx, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), slots, tokens, n_kv, hd)
    rs = np.random.RandomState(0)
    x = rs.randn(2, 3, n_kv, hd).astype(np.float32)
    d, ds = dev(x), dev(np.full(3, slots - 1, np.int32))
    dp = dev(np.array([tokens - 1, 0, tokens - 2], np.int32))
    out = torch.empty(2, 3, n_kv, hd, device="cuda")
    torch.cuda.synchronize()
    c.h.write_device(d[0].data_ptr(), d[1].data_ptr(), ds.data_ptr(), dp.data_ptr(), 3)
    c.h.read_device(ds.data_ptr(), dp.data_ptr(), 3, out[0].data_ptr(), out[1].data_ptr())
    ctx.sync()
    codes, scale = kv8_ref.quantize(x)
    assert np.array_equal(out.cpu().numpy(), codes.astype(np.float32) * scale[..., None])
    got = torch.stack([k[slots - 1, :, [tokens - 1, 0, tokens - 2]], v[slots - 1, :, [tokens - 1, 0, tokens - 2]]])
    assert np.array_equal(got.cpu().numpy().transpose(0, 2, 1, 3), codes)
    # attention over a last slot whose other keys are zero (score 0, value 0)
    q = rs.randn(1, 32, hd).astype(np.float32)
    got = run_decode(ctx, c, q, [slots - 1], [tokens], tokens)
    order = [1, 2, 0]  # positions 0, tokens - 2, tokens - 1
    kk, vv = (codes[i].astype(np.float64) * scale[i][..., None] for i in (0, 1))
    zeros = np.zeros((n_kv, tokens, hd))
    for g in range(n_kv):
        kg, vg = zeros[g].copy(), zeros[g].copy()
        for at, r in zip((0, tokens - 2, tokens - 1), order):
            kg[at], vg[at] = kk[r, g], vv[r, g]
        want, tol = kv8_ref.attend(q[0, g * 4:g * 4 + 4], kg, vg)
        check(got[0, g * 4:g * 4 + 4], want, tol)


def test_runs_on_the_callers_stream_and_in_graphs():
    """Two captured graphs of the same calls and an eager call on another context, at once; replays follow
    the device-side lengths."""
    import torch

    import smallmind_b200 as sm
    rs = np.random.RandomState(8)
    n_heads, n_kv, hd, B, P, T = 32, 4, 64, 5, 300, 600
    other = sm.CudaContext(0)
    graphs = []
    for i in range(2):
        ctx = sm.CudaContext(0)
        s = torch.cuda.Stream()
        ctx.set_stream(s.cuda_stream)
        c = Cache(ctx, B, T, n_kv, hd).fill(rs, [T] * B)
        p = Cache(ctx, 1, P, n_kv, hd).fill(rs, [P])
        q = rs.randn(B, n_heads, hd).astype(np.float32)
        new = rs.randn(2, B, n_kv, hd).astype(np.float32)
        t = dict(q=dev(q), new=dev(new), seq=dev(np.arange(B, dtype=np.int32)), pos=dev(np.full(B, 9, np.int32)),
                 lens=dev(np.full(B, 10, np.int32)), out=torch.zeros(2, B, n_heads, hd, device="cuda"))
        torch.cuda.synchronize()

        def step(c=c, p=p, t=t):
            c.h.write_device(t["new"][0].data_ptr(), t["new"][1].data_ptr(), t["seq"].data_ptr(), t["pos"].data_ptr(), B)
            c.h.attention_decode_device(t["q"].data_ptr(), t["seq"].data_ptr(), t["lens"].data_ptr(), B, n_heads,
                                        t["out"][0].data_ptr(), max_len=T)
            c.h.attention_shared_device(t["q"].data_ptr(), p.h, 0, P, t["seq"].data_ptr(), t["lens"].data_ptr(), B,
                                        n_heads, t["out"][1].data_ptr(), max_len=T)

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
        graphs.append((ctx, s, c, p, q, new, t, g))
    co = Cache(other, 1, 400, n_kv, hd).fill(rs, [400])
    qo = rs.randn(1, n_heads, hd).astype(np.float32)
    for n in (10, 1, 555):
        for ctx, s, c, p, q, new, t, g in graphs:
            t["pos"].fill_(n - 1)
            t["lens"].fill_(n)
        torch.cuda.synchronize()
        for _ in range(3):
            for ctx, s, c, p, q, new, t, g in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        want, tol = kv8_ref.attend_rows(qo, n_kv, [[(co.arrays(), 0, 400)]])
        check(run_decode(other, co, qo, None, [400], 400), want, tol)
        torch.cuda.synchronize()
        for ctx, s, c, p, q, new, t, g in graphs:
            a, pa, got = c.arrays(), p.arrays(), t["out"].cpu().numpy()
            codes, scale = kv8_ref.quantize(new)
            assert np.array_equal(a[0][:, :, n - 1], codes[0]) and np.array_equal(a[3][:, :, n - 1], scale[1])
            check(got[0], *kv8_ref.attend_rows(q, n_kv, [[(a, b, n)] for b in range(B)]))
            check(got[1], *kv8_ref.attend_rows(q, n_kv, [[(pa, 0, P), (a, b, n)] for b in range(B)]))
    for entry in graphs:
        entry[-1].reset()
    torch.cuda.synchronize()
    for entry in graphs:
        entry[0].close()
    other.close()


def test_generation_over_the_8_bit_cache(ctx, O):
    """The operators together, as a decoder layer uses them: a prompt's K / V written once as a shared prefix,
    three sequences that continue it token by token (write, then attend), and a second prompt chunk of one of
    them that reads its cached keys back for the framework's prefill attention."""
    import torch

    import smallmind_b200 as sm
    n_heads, n_kv, hd, P, B, steps = 8, 2, 64, 150, 3, 12
    rs = np.random.RandomState(6)
    prompt_k, prompt_v = (rs.randn(P, n_kv * hd).astype(np.float32) for _ in "kv")
    p = Cache(ctx, 1, P, n_kv, hd)
    c = Cache(ctx, B + 1, 40, n_kv, hd)
    dk, dv = dev(prompt_k), dev(prompt_v)
    zeros, pos = dev(np.zeros(P, np.int32)), dev(np.arange(P, dtype=np.int32))
    torch.cuda.synchronize()
    p.h.write_device(dk.data_ptr(), dv.data_ptr(), zeros.data_ptr(), pos.data_ptr(), P)
    ctx.sync()
    held = [[], []]
    for x, h in ((prompt_k, held[0]), (prompt_v, held[1])):
        codes, scale = kv8_ref.quantize(x.reshape(P, n_kv, hd))
        h.append(codes.astype(np.float64) * scale[..., None].astype(np.float64))
    seqs = np.array([2, 0, 3], np.int32)
    own = [[[], []] for _ in range(B)]
    ds = dev(seqs)
    for t in range(steps):
        qkv = rs.randn(B, (n_heads + 2 * n_kv) * hd).astype(np.float32)
        d, dpos, dlen = dev(qkv), dev(np.full(B, t, np.int32)), dev(np.full(B, t + 1, np.int32))
        out = torch.empty(B, n_heads, hd, device="cuda")
        torch.cuda.synchronize()
        at = d.data_ptr() + 4 * n_heads * hd
        w = (n_heads + 2 * n_kv) * hd
        c.h.write_device(at, at + 4 * n_kv * hd, ds.data_ptr(), dpos.data_ptr(), B, row_stride=w)
        c.h.attention_shared_device(d.data_ptr(), p.h, 0, P, ds.data_ptr(), dlen.data_ptr(), B, n_heads,
                                    out.data_ptr(), max_len=t + 1, q_stride=w)
        ctx.sync()
        got = out.cpu().numpy()
        for b in range(B):
            for i in range(2):
                first = (n_heads + i * n_kv) * hd
                codes, scale = kv8_ref.quantize(qkv[b, first:first + n_kv * hd].reshape(n_kv, hd))
                own[b][i].append(codes.astype(np.float64) * scale[:, None].astype(np.float64))
            for g in range(n_kv):
                k, v = (np.concatenate([held[i][0][:, g], np.stack(own[b][i])[:, g]]) for i in range(2))
                h = slice(g * 4, g * 4 + 4)
                want, tol = kv8_ref.attend(qkv[b, :n_heads * hd].reshape(n_heads, hd)[h], k, v)
                check(got[b, h], want, tol)
    # sequence 1 (slot 0) takes a second prompt chunk: its cached tokens are read back in front of it
    T = 20
    k_all, v_all = (torch.empty(steps + T, n_kv * hd, device="cuda") for _ in "kv")
    chunk = rs.randn(2, T, n_kv * hd).astype(np.float32)
    k_all[steps:], v_all[steps:] = dev(chunk[0]), dev(chunk[1])
    slot, first = dev(np.zeros(steps, np.int32)), dev(np.arange(steps, dtype=np.int32))
    torch.cuda.synchronize()
    c.h.read_device(slot.data_ptr(), first.data_ptr(), steps, k_all.data_ptr(), v_all.data_ptr())
    ctx.sync()
    k_host, v_host = k_all.cpu().numpy(), v_all.cpu().numpy()
    assert np.array_equal(k_host[:steps].reshape(steps, n_kv, hd), np.stack(own[1][0]).astype(np.float32))
    q = rs.randn(T, n_heads * hd).astype(np.float32)
    out = sm.attention(ctx, q, k_host, v_host, T, steps + T, n_heads, n_kv, hd)
    ref = O.attention(q, k_host, v_host, T, steps + T, n_heads, n_kv, hd)
    from conftest import rel_err
    assert rel_err(out, ref) < 1e-4
