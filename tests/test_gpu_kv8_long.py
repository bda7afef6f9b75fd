"""The forms of the 8-bit cache's decode attention that long sequences, large batches and long prefixes reach,
against the 64-bit forms of kv8_ref (whose attend() derives the tolerances)."""
import numpy as np
import pytest

import kv8_ref
from test_gpu_kv8 import Cache, check, dev, run_decode

pytestmark = pytest.mark.gpu


# 4, 8 and 16 heads a kv head and sizes between, odd lengths; more codes than a cluster reads
@pytest.mark.parametrize("n_heads", [1, 4, 7, 8, 11, 16])
@pytest.mark.parametrize("hd,longest", [(64, 80001), (128, 41003)])
def test_a_few_very_long_sequences(hd, longest, n_heads):
    """A sequence split over the GPU: chunks that end inside a block, sequences that end in the first chunk, at
    a chunk's border and with nothing, padding and bad rows, a NaN in the last key's scale."""
    import smallmind_b200 as sm
    ctx = sm.CudaContext(0)
    rs = np.random.RandomState(n_heads)
    lens = np.array([longest, 1, 0, 4096, 4097, 30, longest + 1, 33])
    seq = np.array([0, 1, 2, 1, 2, -1, 0, 9])
    c = Cache(ctx, 3, longest, 1, hd).fill(rs, [longest, 4096, 4097])
    q = (rs.randn(8, n_heads, hd) * np.exp(rs.randn(8, n_heads, 1))).astype(np.float32)
    a = c.arrays()
    rows = [None if b in (5, 6, 7) else [(a, s, n)] for b, (s, n) in enumerate(zip(seq, lens))]
    want, tol = kv8_ref.attend_rows(q, 1, rows)
    got = run_decode(ctx, c, q, seq, lens, longest, q_stride=n_heads * hd + 3)
    check(got, want, tol)
    assert (got[5:] == 5.0).all() and not got[2].any()
    assert np.array_equal(got, run_decode(ctx, c, q, seq, lens, longest))
    assert ctx.device_status() == -2
    c.vs[0, 0, longest - 1] = float("nan")
    c.ks[2, 0, 4096] = float("nan")
    nan = np.isnan(run_decode(ctx, c, q, seq, lens, longest)).all((1, 2))
    assert np.array_equal(nan, np.isin(np.arange(8), (0, 4)))
    ctx.close()


@pytest.mark.parametrize("n_heads,n_kv,hd,B,longest", [
    (16, 8, 128, 72, 513), (16, 8, 128, 72, 512), (32, 4, 64, 200, 1025), (32, 4, 64, 200, 1024), (16, 1, 128, 300, 700),
    (5, 5, 64, 160, 1100)])
def test_large_batches_on_both_sides_of_the_split(ctx, n_heads, n_kv, hd, B, longest):
    rs = np.random.RandomState(B)
    lens = rs.randint(0, longest + 1, B)
    lens[:3] = longest, 0, longest - 1
    seq = rs.permutation(B)
    held = np.zeros(B, int)
    held[seq] = lens
    seq[4] = -1
    c = Cache(ctx, B, longest, n_kv, hd).fill(rs, held)
    q = rs.randn(B, n_heads, hd).astype(np.float32)
    a = c.arrays()
    keys = [None if s < 0 else [(a, s, n)] for s, n in zip(seq, lens)]
    got = run_decode(ctx, c, q, seq, lens, longest)
    check(got, *kv8_ref.attend_rows(q, n_kv, keys))
    assert (got[4] == 5.0).all() and not got[1].any()
    assert ctx.device_status() == 0


@pytest.mark.parametrize("n_heads,n_kv,hd,B,longest", [
    (16, 2, 128, 160, 600), (16, 1, 128, 600, 1000), (32, 4, 128, 150, 1100), (16, 1, 64, 900, 1500),
    (12, 4, 64, 400, 1200), (16, 1, 64, 320, 200), (7, 7, 128, 90, 100), (4, 4, 64, 120, 4097), (4, 4, 64, 120, 4000)])
def test_many_rows(ctx, n_heads, n_kv, hd, B, longest):
    """More sequences than fit the GPU at once, at every group size of both forms."""
    rs = np.random.RandomState(B + longest)
    lens = rs.randint(0, longest + 1, B)
    lens[:3] = longest, 0, longest - 1
    seq = rs.permutation(B)
    held = np.zeros(B, int)
    held[seq] = lens
    seq[4] = -1
    c = Cache(ctx, B, longest, n_kv, hd).fill(rs, held)
    c.vs[seq[2], n_kv - 1, lens[2]:] = float("inf")  # behind the length: not seen
    q = (rs.randn(B, n_heads, hd) * np.exp(rs.randn(B, n_heads, 1))).astype(np.float32)
    a = c.arrays()
    some = np.unique(np.r_[:6, B - 2:B, rs.randint(0, B, 24)])
    keys = [None if seq[b] < 0 else [(a, seq[b], lens[b])] for b in some]
    got = run_decode(ctx, c, q, seq, lens, longest, q_stride=n_heads * hd + 1)
    check(got[some], *kv8_ref.attend_rows(q[some], n_kv, keys))
    assert (got[4] == 5.0).all() and not got[1].any() and np.isfinite(got).all()
    assert np.array_equal(got, run_decode(ctx, c, q, seq, lens, longest))
    assert ctx.device_status() == 0


@pytest.mark.parametrize("n_heads,n_kv,hd,B,prefix_len,longest", [
    (32, 8, 128, 64, 1500, 1100), (16, 2, 64, 180, 1301, 1600), (16, 1, 64, 330, 900, 1300), (4, 4, 128, 140, 640, 800)])
def test_long_own_keys_behind_a_shared_prefix(ctx, n_heads, n_kv, hd, B, prefix_len, longest):
    """Own keys beyond one launch a row, behind a prefix in the matrix form."""
    rs = np.random.RandomState(B + 1)
    lens = rs.randint(0, longest + 1, B)
    lens[:3] = longest, 0, longest - 1
    seq = rs.permutation(B)
    held = np.zeros(B, int)
    held[seq] = lens
    seq[4] = -1
    p = Cache(ctx, 2, prefix_len, n_kv, hd).fill(rs, [0, prefix_len])
    c = Cache(ctx, B, longest, n_kv, hd).fill(rs, held)
    q = (rs.randn(B, n_heads, hd) * np.exp(rs.randn(B, n_heads, 1))).astype(np.float32)
    a, pa = c.arrays(), p.arrays()
    some = np.unique(np.r_[:6, B - 2:B, rs.randint(0, B, 12)])
    keys = [None if seq[b] < 0 else [(pa, 1, prefix_len), (a, seq[b], lens[b])] for b in some]
    got = run_decode(ctx, c, q, seq, lens, longest, prefix=p, prefix_seq=1, prefix_len=prefix_len)
    check(got[some], *kv8_ref.attend_rows(q[some], n_kv, keys))
    assert (got[4] == 5.0).all()
    again = run_decode(ctx, c, q, seq, lens, longest, prefix=p, prefix_seq=1, prefix_len=prefix_len)
    assert np.array_equal(got, again)
    assert ctx.device_status() == 0


@pytest.mark.parametrize("n_heads,n_kv,hd,B,prefix_len", [(32, 8, 128, 100, 16001), (32, 4, 64, 96, 20003),
                                                          (2, 1, 128, 65, 40000)])
def test_very_long_shared_prefix(ctx, n_heads, n_kv, hd, B, prefix_len):
    """Runs of blocks long enough for every ring to wrap and for O to leave the tensor memory several times; calls
    back to back on two batches give the same bits as alone."""
    import torch
    rs = np.random.RandomState(B)
    longest = 20
    lens = rs.randint(0, longest + 1, B)
    p = Cache(ctx, 1, prefix_len, n_kv, hd).fill(rs, [prefix_len])
    p.vs[0, :, 5000:] *= 0.01   # block scales far apart
    p.ks[0, :, prefix_len // 2] *= 3
    c = Cache(ctx, B, longest, n_kv, hd).fill(rs, lens)
    q = rs.randn(2, B, n_heads, hd).astype(np.float32)
    a, pa = c.arrays(), p.arrays()
    alone = [run_decode(ctx, c, x, None, lens, longest, prefix=p, prefix_len=prefix_len) for x in q]
    some = [0, 1, 31, 32, B // 2, B - 1]
    keys = [[(pa, 0, prefix_len), (a, b, lens[b])] for b in some]
    for got, x in zip(alone, q):
        check(got[some], *kv8_ref.attend_rows(x[some], n_kv, keys))
    dq, dl = dev(q), dev(lens.astype(np.int32))
    out = torch.zeros(12, B, n_heads, hd, device="cuda")
    torch.cuda.synchronize()
    for i in range(12):
        c.h.attention_shared_device(dq[i % 2].data_ptr(), p.h, 0, prefix_len, None, dl.data_ptr(), B, n_heads,
                                    out[i].data_ptr(), max_len=longest)
    ctx.sync()
    for i, x in enumerate(out.cpu().numpy()):
        assert np.array_equal(x, alone[i % 2]), i
    assert ctx.device_status() == 0


@pytest.mark.parametrize("n_heads,n_kv,hd,B,prefix_len", [
    (16, 1, 64, 1300, 700), (32, 4, 64, 150, 5003), (16, 2, 128, 210, 2500), (16, 1, 128, 2400, 130), (3, 3, 64, 901, 1111)])
def test_many_tiles_of_query_rows(ctx, n_heads, n_kv, hd, B, prefix_len):
    """More tiles of rows than processors, and numbers of tiles that divide evenly or not."""
    rs = np.random.RandomState(B)
    lens = rs.randint(0, 4, B)
    p = Cache(ctx, 1, prefix_len, n_kv, hd).fill(rs, [prefix_len])
    c = Cache(ctx, B, 3, n_kv, hd).fill(rs, lens)
    q = rs.randn(B, n_heads, hd).astype(np.float32)
    got = run_decode(ctx, c, q, None, lens, 3, prefix=p, prefix_len=prefix_len)
    # the same rows in other tiles
    shift = np.roll(np.arange(B), 37)
    again = run_decode(ctx, c, q[shift], shift, lens[shift], 3, prefix=p, prefix_len=prefix_len)
    a, pa = c.arrays(), p.arrays()
    some = np.unique(np.r_[0, B - 1, rs.randint(0, B, 40)])
    want, tol = kv8_ref.attend_rows(q[some], n_kv, [[(pa, 0, prefix_len), (a, b, lens[b])] for b in some])
    check(got[some], want, tol)
    check(again[np.argsort(shift)][some], want, tol)
    assert ctx.device_status() == 0


def test_long_forms_in_two_graphs_at_once():
    """The forms with workspaces (a shared prefix with split own keys, a split sequence) in graphs of two contexts
    on two streams, replayed side by side over changing lengths."""
    import torch

    import smallmind_b200 as sm
    rs = np.random.RandomState(5)
    n_heads, n_kv, hd, B, P, T = 16, 8, 128, 72, 1200, 700
    graphs = []
    for i in range(2):
        ctx = sm.CudaContext(0)
        s = torch.cuda.Stream()
        ctx.set_stream(s.cuda_stream)
        c = Cache(ctx, B, T, n_kv, hd).fill(rs, [T] * B)
        p = Cache(ctx, 1, P, n_kv, hd).fill(rs, [P])
        t = dict(q=dev(rs.randn(B, n_heads, hd).astype(np.float32)), lens=dev(np.full(B, T, np.int32)),
                 out=torch.zeros(2, B, n_heads, hd, device="cuda"))
        torch.cuda.synchronize()

        def step(c=c, p=p, t=t):
            c.h.attention_decode_device(t["q"].data_ptr(), None, t["lens"].data_ptr(), B, n_heads,
                                        t["out"][0].data_ptr(), max_len=T)
            c.h.attention_shared_device(t["q"].data_ptr(), p.h, 0, P, None, t["lens"].data_ptr(), B, n_heads,
                                        t["out"][1].data_ptr(), max_len=T)

        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
        graphs.append((ctx, s, c, p, t, step, g))
    for _ in range(3):
        want = []
        for ctx, s, c, p, t, step, g in graphs:
            t["lens"].copy_(dev(rs.randint(0, T + 1, B).astype(np.int32)))
            torch.cuda.synchronize()
            step()
            torch.cuda.synchronize()
            want.append(t["out"].clone())
            t["out"].zero_()
        torch.cuda.synchronize()
        for _ in range(4):
            for ctx, s, c, p, t, step, g in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for w, entry in zip(want, graphs):
            assert torch.equal(w, entry[4]["out"])
            some = [0, B // 2, B - 1]
            lens = entry[4]["lens"].cpu().numpy()
            a, pa, q = entry[2].arrays(), entry[3].arrays(), entry[4]["q"].cpu().numpy()
            got = w.cpu().numpy()
            check(got[0][some], *kv8_ref.attend_rows(q[some], n_kv, [[(a, b, lens[b])] for b in some]))
            check(got[1][some], *kv8_ref.attend_rows(q[some], n_kv, [[(pa, 0, P), (a, b, lens[b])] for b in some]))
    for entry in graphs:
        entry[-1].reset()
    torch.cuda.synchronize()
    for entry in graphs:
        entry[0].close()


@pytest.mark.parametrize("n,n_kv,hd,offset", [(40001, 9, 64, 0), (38011, 5, 128, 1), (70003, 1, 64, 0), (9000, 2, 64, 2)])
def test_many_rows_there_and_back(ctx, n, n_kv, hd, offset):
    """More rows than the warps that walk them, a half piece at the end of a row, padding among them."""
    import torch
    rs = np.random.RandomState(n)
    slots, tokens = 7, n // 7 + 3
    place = rs.permutation(slots * tokens)[:n]
    seq, pos = (place // tokens).astype(np.int32), (place % tokens).astype(np.int32)
    seq[::101] = -1
    live = seq >= 0
    w = n_kv * hd
    stride = w + offset
    x = rs.randn(2, n, w).astype(np.float32)
    rows = np.zeros((2, n, stride), np.float32)
    rows[:, :, :w] = x
    c = Cache(ctx, slots, tokens, n_kv, hd)
    d, ds, dp = dev(rows), dev(seq), dev(pos)
    out = torch.full((2, n, stride), 7.0, device="cuda")
    torch.cuda.synchronize()
    c.h.write_device(d[0].data_ptr(), d[1].data_ptr(), ds.data_ptr(), dp.data_ptr(), n, row_stride=stride)
    c.h.read_device(ds.data_ptr(), dp.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr(), row_stride=stride)
    assert ctx.device_status() == 0
    codes, scale = kv8_ref.quantize(x.reshape(2, n, n_kv, hd))
    want = np.full((2, n, stride), 7.0, np.float32)
    want[:, live, :w] = (codes * scale[..., None]).reshape(2, n, w)[:, live]
    assert np.array_equal(out.cpu().numpy(), want)
    k, ks, v, vs = c.arrays()
    free = np.ones((slots, tokens), bool)
    free[seq[live], pos[live]] = False
    for a in (k, v):
        assert (a.transpose(0, 2, 1, 3)[free] == 55).all()
    assert np.isnan(ks.transpose(0, 2, 1)[free]).all() and np.isnan(vs.transpose(0, 2, 1)[free]).all()


# (rows, own keys, prefix): one launch, split over the GPU, behind a short prefix, behind a long one
FORMS = [(3, 300, 0), (3, 41000, 0), (3, 50, 200), (130, 40, 1000), (130, 700, 900)]


@pytest.mark.parametrize("B,n,P", FORMS)
@pytest.mark.parametrize("k_size,v_size,q_size", [(1e-20, 1e-33, 1e20), (1e25, 1e-37, 1e-26), (1, 1e30, 1),
                                                  (1e-37, 1e-25, 1e36)])
def test_magnitudes(ctx, B, n, P, k_size, v_size, q_size):
    """Values near both ends of fp32's range: scores and results stay in it, so they are as exact as others.  (A
    result in the subnormal range is a half step of that, 2^-150, off at most; so is each of its terms.)"""
    rs = np.random.RandomState(B)
    n_heads, n_kv, hd = (4, 1, 128) if n > 10000 else (16, 8, 128)
    lens = rs.randint(n // 2, n + 1, B)
    c = Cache(ctx, B, n, n_kv, hd).fill(rs, lens)
    p = Cache(ctx, 1, max(P, 1), n_kv, hd).fill(rs, [P])
    for x in (c, p):
        x.ks *= k_size
        x.vs *= v_size
        x.vs[:, 0, 1::2] *= 1e-3
    q = (rs.randn(B, n_heads, hd) * q_size).astype(np.float32)
    q[0, 0] = 0
    got = run_decode(ctx, c, q, None, lens, n, prefix=p if P else None, prefix_len=P)
    a, pa = c.arrays(), p.arrays()
    some = [0, 1, B - 1]
    keys = [([(pa, 0, P)] if P else []) + [(a, b, lens[b])] for b in some]
    want, tol = kv8_ref.attend_rows(q[some], n_kv, keys)
    check(got[some], want, tol + 64 * 2.0 ** -150)
    assert np.isfinite(got).all() and got.any()


def test_two_host_threads():
    """Calls of every form from two host threads at once, each with its own context and stream."""
    import threading

    import torch

    import smallmind_b200 as sm
    n_heads, n_kv, hd, T, P = 16, 4, 64, 1300, 700
    failures = []

    def work(seed):
        try:
            rs = np.random.RandomState(seed)
            ctx = sm.CudaContext(0)
            s = torch.cuda.Stream()
            ctx.set_stream(s.cuda_stream)
            for B in (3, 90, 160):
                lens = rs.randint(0, T + 1, B)
                with torch.cuda.stream(s):
                    c = Cache(ctx, B, T, n_kv, hd).fill(rs, lens)
                    p = Cache(ctx, 1, P, n_kv, hd).fill(rs, [P])
                    q = rs.randn(B, n_heads, hd).astype(np.float32)
                    first = [run_decode(ctx, c, q, None, lens, T), run_decode(ctx, c, q, None, lens, T, p, 0, P)]
                    for _ in range(5):
                        again = [run_decode(ctx, c, q, None, lens, T), run_decode(ctx, c, q, None, lens, T, p, 0, P)]
                        assert all(np.array_equal(x, y) for x, y in zip(first, again))
                    a, pa = c.arrays(), p.arrays()
                some = [0, B - 1]
                check(first[0][some], *kv8_ref.attend_rows(q[some], n_kv, [[(a, b, lens[b])] for b in some]))
                keys = [[(pa, 0, P), (a, b, lens[b])] for b in some]
                check(first[1][some], *kv8_ref.attend_rows(q[some], n_kv, keys))
            assert ctx.device_status() == 0
            ctx.close()
        except BaseException as e:
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
