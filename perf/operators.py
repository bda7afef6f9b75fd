"""Workloads of the 8-bit KV cache operators, for timing them and for comparing them with their plain form.

Four operators over one cache of int8 codes ([slot][kv head][position][head dim]) with one fp32 scale for each
position and kv head:

  write   quantise K / V rows into their positions, and read the same rows back
  read    read positions back as fp32
  decode  decode attention of a ragged batch, one query row a sequence, straight from the codes
  shared  the same for a batch whose sequences all begin with one long prefix, which sits in a slot of its own

A row's scale is max|x| / 127 in fp32 and its codes are x / scale rounded to the nearest integer (ties to even).
The softmax is the framework's: weights (12 + 6x + x^2) / (12 - 6x + x^2) of x = max(score - row maximum, -87.3),
divided by their sum.
"""
import math

import numpy as np
import torch

own = False

CLAMP = -87.3


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a 16-sequence batch appends one token a sequence (32 / 4 heads of 64: the TinyLlama shape)
        dict(name="write_step", op="write", n=16, seqs=16, nh=32, nkv=4, hd=64),
        # a long prompt written in one call
        dict(name="write_prompt", op="write", n=32768, seqs=1, nh=32, nkv=8, hd=128),
        # a 2048-token prompt read back for prefill attention of the next chunk
        dict(name="read_prompt", op="read", n=2048, seqs=1, nh=32, nkv=4, hd=64),
        # the contexts of eight sequences read back
        dict(name="read_long", op="read", n=65536, seqs=8, nh=32, nkv=8, hd=128),
        # single-stream decode at the TinyLlama shape's full context
        dict(name="decode_b1", op="decode", b=1, lo=2048, hi=2048, nh=32, nkv=4, hd=64),
        # the repository's ragged attention batch
        dict(name="decode_b16_ragged", op="decode", b=16, lo=256, hi=2048, nh=32, nkv=4, hd=64),
        # odd batch, 9 / 3 heads (the SmolLM shape), lengths from a single token
        dict(name="decode_b7_odd", op="decode", b=7, lo=1, hi=777, nh=9, nkv=3, hd=64),
        # one sequence with a very long context
        dict(name="decode_b1_long", op="decode", b=1, lo=131071, hi=131071, nh=32, nkv=8, hd=128),
        # a serving batch with long contexts
        dict(name="decode_b64_8k", op="decode", b=64, lo=4096, hi=8192, nh=32, nkv=8, hd=128),
        # a small batch of chats behind one system prompt
        dict(name="shared_b8", op="shared", b=8, prefix=999, lo=1, hi=100, nh=9, nkv=3, hd=64),
        # a serving batch behind a long document
        dict(name="shared_b64", op="shared", b=64, prefix=8192, lo=1, hi=512, nh=32, nkv=4, hd=64),
        # many short answers over one very long document
        dict(name="shared_b256", op="shared", b=256, prefix=32768, lo=16, hi=512, nh=32, nkv=8, hd=128),
    ]


HEADS = [(9, 3, 64), (32, 4, 64), (8, 8, 64), (4, 2, 64), (16, 1, 64), (32, 8, 128), (12, 4, 128), (16, 16, 128)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "shared"])
    nh, nkv, hd = rng.choice(HEADS)
    if op in ("write", "read"):
        n = _log(rng, 1, 16384)
        return dict(op=op, n=n, seqs=_log(rng, 1, min(n, 64)), nh=nh, nkv=nkv, hd=hd)
    if op == "decode":
        b = _log(rng, 1, 64)
        hi = _log(rng, 1, 131072 // b)
        return dict(op=op, b=b, lo=rng.randint(1, hi), hi=hi, nh=nh, nkv=nkv, hd=hd)
    b = _log(rng, 2, 128)
    hi = _log(rng, 1, 512)
    return dict(op=op, b=b, prefix=_log(rng, 64, 16384), lo=rng.randint(0, hi), hi=hi, nh=nh, nkv=nkv, hd=hd)


def _lengths(case):
    """The batch's lengths, evenly spread from lo to hi: the same for every seed (only their order is the seed's)."""
    b, lo, hi = case["b"], case["lo"], case["hi"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def work(case):
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    held = nkv * (2 * hd + 2 * 4)  # bytes of one position: codes and scales of K and V
    if case["op"] in ("write", "read"):
        rows = 2 * 4 * case["n"] * nkv * hd  # K and V in fp32
        move = 2 * rows if case["op"] == "write" else rows
        return {"bytes": move + case["n"] * held, "flops": 4 * case["n"] * nkv * hd}
    total = sum(_lengths(case))
    keys = total + case["b"] * case.get("prefix", 0)
    return {"bytes": (total + case.get("prefix", 0)) * held + 2 * 4 * case["b"] * nh * hd, "flops": 4 * nh * hd * keys}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _heads_like(g, *shape):
    """K / V values: normal, with a few channels of each head well above the rest, as rotary keys have."""
    x = torch.randn(*shape, generator=g, device="cuda")
    x[..., :: max(1, shape[-1] // 3)] *= 4.0
    return x


def _cache(g, slots, nkv, tokens, hd):
    """A filled cache: codes and scales of K-like values."""
    x = _heads_like(g, slots, nkv, tokens, hd)
    scale = x.abs().amax(-1) / 127.0
    codes = torch.round(x.div_(scale[..., None])).clamp_(-127, 127).to(torch.int8)
    return codes, scale


def prepare(case, seed):
    g = _gen(seed)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    s = {"case": case}
    if case["op"] in ("write", "read"):
        n, seqs = case["n"], case["seqs"]
        each = (n + seqs - 1) // seqs
        s["tokens"] = tokens = each + 8
        s["slots"] = slots = seqs + 1
        order = torch.randperm(slots, generator=g, device="cuda")[:seqs].int()
        base = torch.randint(0, 8, (seqs,), generator=g, device="cuda").int()
        row = torch.arange(n, device="cuda")
        s["seq"] = order[row % seqs].contiguous()
        s["pos"] = (base[row % seqs] + (row // seqs).int()).contiguous()
        if case["op"] == "write":
            # K and V rows as a fused projection leaves them: q | k | v side by side
            s["qkv"] = _heads_like(g, n, nh + 2 * nkv, hd)
            for w in ("k", "v"):
                s[w] = torch.zeros(slots, nkv, tokens, hd, dtype=torch.int8, device="cuda")
                s[w + "_scale"] = torch.zeros(slots, nkv, tokens, device="cuda")
            return s
        for w in ("k", "v"):
            s[w], s[w + "_scale"] = _cache(g, slots, nkv, tokens, hd)
        return s
    b = case["b"]
    s["longest"] = s["tokens"] = max(1, max(_lengths(case)))
    s["slots"] = b
    s["seq"] = torch.randperm(b, generator=g, device="cuda").int()
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    s["lens"] = lens[torch.randperm(b, generator=g, device="cuda")].contiguous()
    s["q"] = torch.randn(b, nh * hd, generator=g, device="cuda")
    for w in ("k", "v"):
        s[w], s[w + "_scale"] = _cache(g, b, nkv, s["tokens"], hd)
        if case["op"] == "shared":  # the prefix is kept once, in a cache of one long slot
            s["prefix_" + w], s["prefix_" + w + "_scale"] = _cache(g, 1, nkv, case["prefix"], hd)
    return s


# ---------------------------------------------------------------- the framework's calls
_contexts = {}  # one for each device and stream that work is queued on


def _handles(s):
    """The cache handles that a program makes once and keeps beside its tensors, for the current stream."""
    device = torch.cuda.current_device()
    # the stream's number alone: torch.cuda.current_stream() takes 3 us to make an object of it
    key = device, torch._C._cuda_getCurrentRawStream(device)
    held = s.setdefault("handles", {})
    if key not in held:
        import smallmind_b200 as sm

        if key not in _contexts:
            _contexts[key] = sm.CudaContext(device)
            # torch's default stream has the number 0; as an explicit handle the legacy default stream is 1
            _contexts[key].set_stream(key[1] or 1)
        c = s["case"]

        def make(which, slots, tokens):
            at = (s[which + w].data_ptr() for w in ("k", "v", "k_scale", "v_scale"))
            return sm.KV8Cache(_contexts[key], *at, slots, tokens, c["nkv"], c["hd"])

        prefix = make("prefix_", 1, c["prefix"]) if c["op"] == "shared" else None
        held[key] = make("", s["slots"], s["tokens"]), prefix
    return held[key]


def _run_own(s):
    c = s["case"]
    h, prefix = _handles(s)
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    if c["op"] in ("write", "read"):
        n = c["n"]
        if c["op"] == "write":
            at = s["qkv"].data_ptr() + 4 * nh * hd
            h.write_device(at, at + 4 * nkv * hd, s["seq"].data_ptr(), s["pos"].data_ptr(), n,
                           row_stride=(nh + 2 * nkv) * hd)
        k = torch.empty(n, nkv, hd, device="cuda")
        v = torch.empty(n, nkv, hd, device="cuda")
        h.read_device(s["seq"].data_ptr(), s["pos"].data_ptr(), n, k.data_ptr(), v.data_ptr())
        return k, v
    out = torch.empty(c["b"], nh * hd, device="cuda")
    if c["op"] == "decode":
        h.attention_decode_device(s["q"].data_ptr(), s["seq"].data_ptr(), s["lens"].data_ptr(), c["b"], nh,
                                  out.data_ptr(), max_len=s["longest"])
    else:
        h.attention_shared_device(s["q"].data_ptr(), prefix, 0, c["prefix"], s["seq"].data_ptr(),
                                  s["lens"].data_ptr(), c["b"], nh, out.data_ptr(), max_len=s["longest"])
    return out


# ---------------------------------------------------------------- the plain forms
def _write_plain(s, w, x):
    scale = x.abs().amax(-1) / 127.0
    codes = torch.round(x.double() / scale.double()[..., None])
    codes = torch.where(scale[..., None] > 0, codes, 0.0).clamp(-127, 127).to(torch.int8)
    s[w][s["seq"].long(), :, s["pos"].long()] = codes
    s[w + "_scale"][s["seq"].long(), :, s["pos"].long()] = scale


def _read_plain(s, w):
    at = s["seq"].long(), s["pos"].long()
    return s[w][at[0], :, at[1]].float() * s[w + "_scale"][at[0], :, at[1]][..., None]


def _scores(eq, q, k, live, scale):
    s = torch.einsum(eq, q, k) * scale
    return s if live is None else s.masked_fill(~live, -math.inf)


def _weights(s, m):
    x = (s - m).clamp(min=CLAMP)
    x2 = x * x / 12.0
    e = (1.0 + 0.5 * x + x2) / (1.0 - 0.5 * x + x2)
    return torch.where(torch.isinf(s), 0.0, e)


def _attend_plain(s):
    c = s["case"]
    b, nh, nkv, hd, top = c["b"], c["nh"], c["nkv"], c["hd"], s["longest"]
    q = s["q"].view(b, nkv, nh // nkv, hd)
    scale = 1.0 / math.sqrt(hd)
    seq = s["seq"].long()
    k = s["k"][seq, :, :top].float() * s["k_scale"][seq, :, :top, None]
    v = s["v"][seq, :, :top].float() * s["v_scale"][seq, :, :top, None]
    live = (torch.arange(top, device="cuda")[None] < s["lens"][:, None])[:, None, None]
    s1 = _scores("bgrd,bgtd->bgrt", q, k, live, scale)
    m = s1.amax(-1, keepdim=True)
    if c["op"] == "shared":
        kp = s["prefix_k"][0].float() * s["prefix_k_scale"][0, :, :, None]
        vp = s["prefix_v"][0].float() * s["prefix_v_scale"][0, :, :, None]
        s2 = _scores("bgrd,gtd->bgrt", q, kp, None, scale)
        m = torch.maximum(m, s2.amax(-1, keepdim=True))
        e2 = _weights(s2, m)
        e1 = _weights(s1, m)
        total = e1.sum(-1, keepdim=True) + e2.sum(-1, keepdim=True)
        out = torch.einsum("bgrt,bgtd->bgrd", e1, v) + torch.einsum("bgrt,gtd->bgrd", e2, vp)
    else:
        e1 = _weights(s1, m)
        total = e1.sum(-1, keepdim=True)
        out = torch.einsum("bgrt,bgtd->bgrd", e1, v)
    return (out / total).reshape(b, nh * hd)


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    nh, nkv = c["nh"], c["nkv"]
    if c["op"] == "write":
        _write_plain(state, "k", state["qkv"][:, nh : nh + nkv])
        _write_plain(state, "v", state["qkv"][:, nh + nkv :])
    if c["op"] in ("write", "read"):
        return _read_plain(state, "k"), _read_plain(state, "v")
    return _attend_plain(state)


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["op"] == "write":
        got = []
        for first in (nh, nh + nkv):
            x = s["qkv"][:, first : first + nkv].cpu().numpy()
            peak = np.max(np.abs(x), axis=-1, keepdims=True)
            scale = (peak.astype(np.float64) / 127.0).astype(np.float32).astype(np.float64)  # held in fp32
            got.append(np.clip(np.rint(x.astype(np.float64) / scale), -127, 127) * scale)
        return tuple(got)
    if case["op"] == "read":
        at = s["seq"].cpu().numpy(), s["pos"].cpu().numpy()
        got = []
        for w in ("k", "v"):
            codes, scale = s[w].cpu().numpy(), s[w + "_scale"].cpu().numpy().astype(np.float64)
            got.append(codes[at[0], :, at[1]].astype(np.float64) * scale[at[0], :, at[1]][..., None])
        return tuple(got)
    seq, lens = s["seq"].tolist(), s["lens"].tolist()
    group = nh // nkv
    out = torch.empty(case["b"], nh, hd, dtype=torch.float64, device="cuda")

    def held(w, slot, head, n):
        return s[w][slot, head, :n].double() * s[w + "_scale"][slot, head, :n].double().unsqueeze(1)

    for head in range(nkv):
        kp = vp = None
        if case["op"] == "shared":
            kp, vp = (held("prefix_" + w, 0, head, case["prefix"]) for w in ("k", "v"))
        for i in range(case["b"]):
            q = s["q"][i].view(nh, hd)[head * group : (head + 1) * group].double()
            k, v = held("k", seq[i], head, lens[i]), held("v", seq[i], head, lens[i])
            parts = [(k, v)] if kp is None else [(kp, vp), (k, v)]
            z = torch.cat([q @ a.t() for a, _ in parts], 1) / math.sqrt(hd)
            z = (z - z.max(1, keepdim=True).values).clamp(min=CLAMP)
            e = (12 + 6 * z + z * z) / (12 - 6 * z + z * z)
            top, at = 0, 0
            for a, u in parts:
                top = top + e[:, at : at + a.shape[0]] @ u
                at += a.shape[0]
            out[i, head * group : (head + 1) * group] = top / e.sum(1, keepdim=True)
    return out.view(case["b"], nh * hd)
