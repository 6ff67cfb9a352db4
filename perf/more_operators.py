"""Operators of a serving loop that runs the hybrid model on caller buffers: the gated delta rule of its
linear-attention layers over a pool of states (one token a sequence, and whole prompts in chunks), the short
convolution in front of it, and the paged cache's attention for sequences that share a long prefix.

    own       False: the plain forms in torch; True: the framework's calls (chpe_amd.DeltaStates, KvPages)
    listed()  the cases by name            prepare(case, seed)  what a program holds before the call
    draw(rng) one more of the same ranges  run(state)           one pass
    work      bytes and operations         exact(case, seed)    the result in 64 bits

States are read from one slot and left in another, as a program does that may take a step back (drafts that a
check rejects) or that starts many sequences from one prompt's state.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# the linear-attention layers' key heads, value heads, head dim: the hybrid model's, then other ordinary layouts
# (a value head per key head; groups of 3 and 4; one key head)
DELTA = {"9b": (16, 32, 128), "one64": (12, 12, 64), "group3": (5, 15, 128), "group4": (4, 16, 64), "shared": (1, 6, 128)}
# query heads, kv heads, head dim: the models of this engine, then other ordinary layouts
HEADS = {
    "3b": (16, 2, 128), "9b": (16, 4, 256), "72b": (64, 8, 128), "mha64": (12, 12, 64), "gqa3": (24, 8, 128),
    "gqa6": (12, 2, 64), "mqa256": (8, 1, 256),
}
TAPS = 4
EPS = 1e-6


def listed():
    return [
        # one sequence's step of the hybrid model: latency alone
        dict(name="conv 9b f32 1 token", op="conv", heads="9b", type="f32", taps=4, rows=1, longest=1, ragged=False, fresh=False),
        # prompts of a batch
        dict(name="conv 9b bf16 6x2731", op="conv", heads="9b", type="bf16", taps=4, rows=6, longest=2731, ragged=True,
             fresh=True),
        # one sequence's step; a small batch's; a full server's, whose states pass through the chip once
        dict(name="step 9b f32 1 row", op="step", heads="9b", type="f32", rows=1, gate=True),
        dict(name="step 9b f32 33 rows", op="step", heads="9b", type="f32", rows=33, gate=True),
        dict(name="step 9b bf16 256 rows", op="step", heads="9b", type="bf16", rows=256, gate=False),
        # drafts of a batch, checked at once
        dict(name="prompt 9b f32 32x5", op="prompt", heads="9b", type="f32", rows=32, longest=5, ragged=False, gate=True,
             fresh=False),
        # a chat turn, odd length, behind the turns before it
        dict(name="prompt 9b bf16 1x501", op="prompt", heads="9b", type="bf16", rows=1, longest=501, ragged=False, gate=True,
             fresh=False),
        # one long document
        dict(name="prompt 9b f32 1x8189", op="prompt", heads="9b", type="f32", rows=1, longest=8189, ragged=False, gate=False,
             fresh=True),
        # the prompts of a batch
        dict(name="prompt 9b bf16 24x4097", op="prompt", heads="9b", type="bf16", rows=24, longest=4097, ragged=True,
             gate=False, fresh=True),
        # a few sequences behind one system prompt of the hybrid model
        dict(name="prefix 9b bf16 5 rows 1040", op="prefix", heads="9b", type="bf16", page=16, groups=1, rows=5, prefix=1040,
             rest=96, ragged=True),
        # samples of several prompts
        dict(name="prefix 9b f16 8x6 rows 2048", op="prefix", heads="9b", type="f16", page=64, groups=8, rows=48, prefix=2048,
             rest=256, ragged=True),
        # a full server behind one long document on the large model
        dict(name="prefix 72b f16 64 rows 8192", op="prefix", heads="72b", type="f16", page=16, groups=1, rows=64,
             prefix=8192, rest=129, ragged=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    while True:
        c = _draw(rng)
        if work(c)["bytes"] <= 1.3e9:  # no more than the largest listed case
            return c


def _draw(rng):
    op = rng.choice(["conv", "step", "step", "prompt", "prompt", "prompt", "prefix", "prefix", "prefix"])
    c = dict(op=op, type=rng.choice(list(TYPES)))
    if op == "prefix":
        c.update(heads=rng.choice(list(HEADS)), page=2 ** rng.randint(3, 8))
        H, KV, hd = HEADS[c["heads"]]
        rows = _log(rng, 1, 96)
        groups = 1 if rng.random() < 0.5 else rng.randint(1, rows)
        e = 4 if c["type"] == "f32" else 2
        # at most the largest listed products (against 32 bits an eighth of them) and 4 GB of keys and values
        most = 64 * 64 * 8192 * 128 // (rows * H * hd * (8 if e == 4 else 1))
        most = max(2, min(most, (4 << 30) // (KV * hd * 2 * e * rows) if groups > 1 else most, 30000))
        prefix = _log(rng, 1, most)
        rest = _log(rng, 1, max(2, min(2000, (2 << 30) // (rows * KV * hd * 2 * e), 40 * most // max(1, prefix) + 1)))
        return dict(c, groups=groups, rows=rows, prefix=prefix, rest=rest, ragged=rng.random() < 0.7)
    c.update(heads=rng.choice(list(DELTA)))
    NK, NV, hd = DELTA[c["heads"]]
    if op == "step":  # at most the largest listed states
        return dict(c, rows=_log(rng, 1, min(512, 256 * 32 * 128 * 128 // (NV * hd * hd))), gate=rng.random() < 0.6)
    rows = _log(rng, 1, 64)
    if op == "conv":
        c["taps"] = rng.choice([4, 4, 2, 3, 8])
        longest = _log(rng, 1, min(16000, 6 * 2731 * 8192 // (rows * (2 * NK + NV) * hd * (2 if c["type"] == "f32" else 1))))
    else:  # at most the largest listed tokens, and their number in a row
        c["gate"] = rng.random() < 0.4
        longest = _log(rng, 1, min(8189, 60000 // rows, 12 * 4097 * 32 * 128 // (rows * NV * hd * (2 if c["type"] == "f32" else 1))))
    return dict(c, rows=rows, longest=longest, ragged=rng.random() < 0.6, fresh=rng.random() < 0.5)


# ------------------------------------------------------------------ what a program holds
def _lens(case, seed):
    """Lengths of the rows: all alike, or spread evenly from 1 to the longest, in an order of the seed's."""
    n, top = case["rows"], case["longest"]
    if not case["ragged"]:
        return np.full(n, top)
    return np.random.default_rng(seed).permutation(np.linspace(top, 1, n).round().astype(np.int64))


def _dev(a, dt=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dt)


def _slots(st, case, seed):
    """Each row's slot before and after, in the order that a pool hands them out; -1: a new sequence."""
    n = case["rows"]
    ids = np.random.default_rng(seed + 1).permutation(2 * n + 1)
    before, after = ids[:n].copy(), ids[n:2 * n]
    if case.get("fresh"):
        before[::2] = -1
    st.update(slot_in=_dev(before), slot_out=_dev(after), before=before, after=after)
    return 2 * n + 1


def _prepare_delta(case, seed, g):
    NK, NV, hd = DELTA[case["heads"]]
    dt, rows = TYPES[case["type"]], case["rows"]
    st = dict(case=case)
    n_slots = _slots(st, case, seed)
    lens = np.ones(rows, np.int64) if case["op"] == "step" else _lens(case, seed)
    starts = np.concatenate(([0], np.cumsum(lens)))
    n, channels = int(starts[-1]), (2 * NK + NV) * hd
    st.update(lens=lens, first=starts, starts=_dev(starts), top=int(lens.max()))
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "conv":
        st["x"] = rand(n, channels).to(dt)
        st["w"] = rand(channels, case["taps"]) * 0.5
        st["conv"] = rand(n_slots, channels, case["taps"] - 1)
        st["out"] = torch.empty_like(st["x"])
        return st
    # the convolution's outputs (queries, keys and values next to each other), the gates' inputs
    mixed = torch.nn.functional.silu(rand(n, channels)).to(dt)
    st["mixed"] = mixed
    st["q"], st["k"] = (mixed[:, i * NK * hd:(i + 1) * NK * hd].view(n, NK, hd) for i in range(2))
    st["v"] = mixed[:, 2 * NK * hd:].view(n, NV, hd)
    st["a"], st["b"] = rand(n, NV), rand(n, NV)
    # decay rates from heads that keep thousands of tokens to heads that keep one
    st["A_log"] = torch.rand(NV, generator=g, device="cuda") * 7.0 - 4.5
    st["dt_bias"] = rand(NV)
    st["state"] = rand(n_slots, NV, hd, hd) * 0.3
    st["out"] = torch.empty(n, NV, hd, dtype=dt, device="cuda")
    if case["gate"]:
        st["z"] = rand(n, NV, hd).to(dt)
        st["norm_w"] = 1.0 + 0.2 * rand(hd)
    return st


def _prefix_plan(case, seed):
    """First rows of the groups, their prefixes' lengths, the rows' lengths."""
    r = np.random.default_rng(seed)
    rows, groups = case["rows"], case["groups"]
    cuts = np.sort(r.choice(np.arange(1, rows), groups - 1, replace=False)) if groups > 1 else np.zeros(0, np.int64)
    first = np.concatenate(([0], cuts, [rows]))
    prefix = np.full(groups, case["prefix"])
    if case["ragged"]:
        prefix[1:] = r.integers((case["prefix"] + 1) // 2, case["prefix"] + 1, groups - 1)
    rest = r.integers(1, case["rest"] + 1, rows) if case["ragged"] else np.full(rows, case["rest"])
    return first, prefix, np.repeat(prefix, np.diff(first)) + rest


def _prepare_prefix(case, seed, g):
    H, KV, hd = HEADS[case["heads"]]
    page, dt = case["page"], TYPES[case["type"]]
    first, prefix, lens = _prefix_plan(case, seed)
    per_row = int(-(-(case["prefix"] + case["rest"]) // page))
    # whole pages of a prefix belong to all rows of its group, the page in which it ends to each row
    table = np.full((case["rows"], per_row), -1, np.int64)
    used, copies = 0, []
    for i, p in enumerate(prefix):
        shared = p // page
        for r in range(first[i], first[i + 1]):
            if r == first[i]:
                table[r, :shared] = np.arange(used, used + shared)
                used += shared
            else:
                table[r, :shared] = table[first[i], :shared]
            mine = -(-lens[r] // page) - shared
            table[r, shared:shared + mine] = np.arange(used, used + mine)
            used += mine
            if p % page and r != first[i]:
                copies.append((table[r, shared], table[first[i], shared], p % page))
    order = np.random.default_rng(seed + 1).permutation(used + 3)  # as a pool hands them out
    k, v = (torch.randn(used + 3, KV, page, hd, generator=g, device="cuda").to(dt) for _ in "kv")
    for dst, src, m in copies:
        for x in (k, v):
            x[order[dst], :, :m] = x[order[src], :, :m]
    table = np.where(table >= 0, order[table], 0)
    st = dict(case=case, k=k, v=v, table=_dev(table), first=first, prefix=prefix, lens=lens, d_lens=_dev(lens),
              d_first=_dev(first), d_prefix=_dev(prefix), pages=table)
    st["q"] = torch.randn(case["rows"], H, hd, generator=g, device="cuda") * 2.0  # scores spread over a few units
    st["out"] = torch.empty_like(st["q"])
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = (_prepare_prefix if case["op"] == "prefix" else _prepare_delta)(case, seed, g)
    if own:
        sys.path.insert(0, str(Path.cwd() / "chpe-qwen-engine_amd"))
        import chpe_amd as ca
        if case["op"] == "prefix":
            st["handle"] = ca.KvPages(st["k"], st["v"], st["table"])
            need = st["handle"].prefix_workspace(HEADS[case["heads"]][0], case["groups"], case["prefix"], case["rest"])
        elif case["op"] == "conv":
            st["handle"] = ca.DeltaConv(st["conv"], st["w"])
            need = 0
        else:
            st["handle"] = ca.DeltaStates(st["state"], DELTA[case["heads"]][0])
            need = 0 if case["op"] == "step" else st["handle"].prompt_workspace(int(st["first"][-1]), case["rows"], case["gate"])
        if need:
            st["workspace"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
    return st


# ------------------------------------------------------------------ the framework's calls
def _run_own(st):
    c, h = st["case"], st["handle"]
    if c["op"] == "conv":
        h.apply(st["x"], st["starts"], st["slot_in"], st["slot_out"], out=st["out"])
    elif c["op"] == "step":
        h.step(st["q"], st["k"], st["v"], st["a"], st["b"], st["A_log"], st["dt_bias"], st["slot_in"], st["slot_out"],
               z=st.get("z"), norm_w=st.get("norm_w"), eps=EPS, out=st["out"])
    elif c["op"] == "prompt":
        h.prompt(st["q"], st["k"], st["v"], st["a"], st["b"], st["A_log"], st["dt_bias"], st["starts"], st["slot_in"],
                 st["slot_out"], z=st.get("z"), norm_w=st.get("norm_w"), eps=EPS, out=st["out"], workspace=st["workspace"])
    else:
        h.prefix_attention(st["q"], st["d_lens"], st["d_first"], st["d_prefix"], c["prefix"], c["rest"], out=st["out"],
                           workspace=st["workspace"])


# ------------------------------------------------------------------ the plain forms
def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _taken(pool, slots, like):
    """What the slots hold, zeros for -1."""
    x = pool[slots.clamp(min=0).long()].to(like)
    return torch.where((slots >= 0).view(-1, *[1] * (x.dim() - 1)), x, torch.zeros_like(x))


def _plain_conv(st):
    x, w, starts, P = st["x"].float(), st["w"], st["starts"].long(), st["w"].shape[1] - 1
    row = torch.repeat_interleave(torch.arange(st["case"]["rows"], device="cuda"), starts[1:] - starts[:-1], output_size=x.shape[0])
    # every row's inputs behind the P that came before them
    at = torch.arange(x.shape[0], device="cuda") + P * (row + 1)
    ext = torch.empty(x.shape[0] + P * st["case"]["rows"], x.shape[1], device="cuda")
    head = (starts[:-1] + P * torch.arange(st["case"]["rows"], device="cuda"))[:, None] + torch.arange(P, device="cuda")
    ext[head] = _taken(st["conv"], st["slot_in"], torch.float32).transpose(1, 2)
    ext[at] = x
    y = torch.zeros_like(x)
    for j in range(P + 1):
        y += w[:, j] * ext[at - P + j]
    st["out"].copy_(_silu(y))
    st["conv"][st["slot_out"].long()] = ext[head + (starts[1:] - starts[:-1])[:, None]].transpose(1, 2)


def _gates(st):
    x = st["a"] + st["dt_bias"]
    softplus = torch.where(x > 0, x, torch.zeros_like(x)) + torch.log1p(torch.exp(-x.abs()))
    return torch.exp(-torch.exp(st["A_log"]) * softplus), 1.0 / (1.0 + torch.exp(-st["b"]))


def _unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _plain_delta(st):
    c = st["case"]
    NK, NV, hd = DELTA[c["heads"]]
    decay, beta = _gates(st)
    k, q, v = _unit(st["k"].float()), _unit(st["q"].float()) / math.sqrt(hd), st["v"].float()
    order = np.argsort(-st["lens"], kind="stable")
    starts, lens = _dev(st["first"][order], torch.long), st["lens"][order]
    S = _taken(st["state"], st["slot_in"], torch.float32)[_dev(order, torch.long)]
    out = torch.zeros(v.shape, device="cuda")
    for t in range(st["top"]):
        n = int((lens > t).sum())  # the rows that have a token t
        at, s = starts[:n] + t, S[:n]
        kt = k[at].repeat_interleave(NV // NK, 1)[..., None]
        qt = q[at].repeat_interleave(NV // NK, 1)[..., None]
        s *= decay[at][..., None, None]
        d = (v[at] - (s * kt).sum(-2)) * beta[at][..., None]
        s += kt * d[..., None, :]
        out[at] = (s * qt).sum(-2)
    if c["gate"]:
        out = out / torch.sqrt((out * out).mean(-1, keepdim=True) + EPS) * st["norm_w"] * _silu(st["z"].float())
    st["out"].copy_(out)
    st["state"][st["slot_out"].long()[_dev(order, torch.long)]] = S


def _slots_of(pages, ids, n):
    """[kv heads][n][dim] of the first n slots of these pages, in 32 bits."""
    x = pages[ids[:-(-n // pages.shape[2])].long()].transpose(0, 1)
    return x.reshape(x.shape[0], -1, x.shape[-1])[:, :n].float()


def _plain_prefix(st):
    c = st["case"]
    H, KV, hd = HEADS[c["heads"]]
    gq, page = H // KV, c["page"]
    for i, p in enumerate(st["prefix"].tolist()):
        r0, r1 = int(st["first"][i]), int(st["first"][i + 1])
        n, off = r1 - r0, p // page
        top = int(st["lens"][r0:r1].max()) - p
        k, v = (_slots_of(x, st["table"][r0], p) for x in (st["k"], st["v"]))
        q = st["q"][r0:r1].reshape(n, KV, gq, hd).transpose(0, 1) / math.sqrt(hd)
        s = torch.matmul(q.reshape(KV, n * gq, hd), k.transpose(1, 2).contiguous()).reshape(KV, n, gq, p)
        # the rows' own slots, from the page in which the prefix ends
        ids = st["table"][r0:r1, off:off + -(-(p % page + top) // page)].long()
        k2, v2 = (x[ids].permute(2, 0, 1, 3, 4).reshape(KV, n, -1, hd)[:, :, p % page:p % page + top].float()
                  for x in (st["k"], st["v"]))
        s2 = torch.matmul(q, k2.transpose(2, 3).contiguous())
        seen = torch.arange(top, device="cuda") < (st["d_lens"][r0:r1] - p)[:, None]
        s2 = torch.where(seen[None, :, None], s2, torch.full_like(s2, -math.inf))
        m = torch.maximum(s.amax(-1, keepdim=True), s2.amax(-1, keepdim=True))
        s, s2 = torch.exp(s - m), torch.exp(s2 - m)
        o = torch.matmul(s.reshape(KV, n * gq, p), v).reshape(KV, n, gq, hd) + torch.matmul(s2, v2)
        o = o / (s.sum(-1, keepdim=True) + s2.sum(-1, keepdim=True))
        st["out"][r0:r1] = o.transpose(0, 1).reshape(n, H, hd)


def run(st):
    op = st["case"]["op"]
    if own:
        _run_own(st)
    else:
        {"conv": _plain_conv, "step": _plain_delta, "prompt": _plain_delta, "prefix": _plain_prefix}[op](st)
    if op == "prefix":
        return [st["out"]]
    return [st["out"], st["conv" if op == "conv" else "state"]]


# ------------------------------------------------------------------ bytes and operations
def _mean_tokens(case):
    n, top = case["rows"], case["longest"]
    return n * top if not case["ragged"] or n == 1 else n * (top + 1) / 2


def work(case):
    e, n = (4 if case["type"] == "f32" else 2), case["rows"]
    if case["op"] == "prefix":
        H, KV, hd = HEADS[case["heads"]]
        mean = lambda lo, hi: (lo + hi) / 2 if case["ragged"] else hi  # noqa: E731
        rest = n * mean(1, case["rest"])
        prefix = case["prefix"] + (case["groups"] - 1) * mean((case["prefix"] + 1) // 2, case["prefix"])
        return dict(bytes=2 * KV * hd * e * (rest + prefix) + 8 * n * H * hd,
                    flops=4 * H * hd * (rest + prefix * n / case["groups"]))
    NK, NV, hd = DELTA[case["heads"]]
    read = n // 2 if case.get("fresh") else n
    if case["op"] == "conv":
        t, C, T = _mean_tokens(case), (2 * NK + NV) * hd, case["taps"]
        return dict(bytes=2 * t * C * e + 4 * C * T + 4 * C * (T - 1) * (n + read), flops=t * C * (2 * T + 4))
    t = n if case["op"] == "step" else _mean_tokens(case)
    return dict(bytes=t * ((2 * NK + 2 * NV + (NV if case["gate"] else 0)) * hd * e + 8 * NV) + 4 * NV * hd * hd * (n + read),
                flops=t * NV * hd * hd * 7)


# ------------------------------------------------------------------ the results in 64 bits
def _exact_conv(case, seed, st):
    x, w, P = st["x"].double(), st["w"].double(), case["taps"] - 1
    out, conv = torch.empty_like(x), st["conv"].double()
    new = {}
    for r in range(case["rows"]):
        lo, hi = int(st["first"][r]), int(st["first"][r + 1])
        before = conv[int(st["before"][r])] if st["before"][r] >= 0 else torch.zeros_like(conv[0])
        seq = torch.cat((before, x[lo:hi].t()), 1)
        y = (seq.unfold(1, P + 1, 1) * w[:, None]).sum(-1)
        out[lo:hi] = (y * torch.sigmoid(y)).t()
        new[int(st["after"][r])] = seq[:, hi - lo:]
    for slot, s in new.items():
        conv[slot] = s
    return [out, conv]


def _exact_delta(case, seed, st):
    NK, NV, hd = DELTA[case["heads"]]
    k, q = (torch.nn.functional.normalize(torch.cat((x.double(), torch.full_like(x[..., :1].double(), 1e-3)), -1),
                                          dim=-1, eps=0.0)[..., :hd].repeat_interleave(NV // NK, 1) for x in (st["k"], st["q"]))
    v, beta = st["v"].double(), torch.sigmoid(st["b"].double())
    decay = torch.exp(-st["A_log"].double().exp() * torch.nn.functional.softplus(st["a"].double() + st["dt_bias"].double(), threshold=700.0))
    out, state = torch.empty(v.shape, dtype=torch.float64, device="cuda"), st["state"].double()
    new = {}
    if case["op"] == "step":  # all rows at once
        S = _taken(st["state"], st["slot_in"], torch.float64).reshape(-1, hd, hd)
        kk = k.reshape(-1, hd, 1)
        S = S * decay.reshape(-1, 1, 1)
        S = S - torch.bmm(kk * beta.reshape(-1, 1, 1), torch.bmm(kk.transpose(1, 2).contiguous(), S)) + kk * (beta[..., None] * v).reshape(-1, 1, hd)
        out = torch.bmm(q.reshape(-1, 1, hd), S).reshape(out.shape) / hd ** 0.5
        state[st["slot_out"].long()] = S.reshape(-1, NV, hd, hd)
    else:
        eye = torch.eye(hd, dtype=torch.float64, device="cuda")
        for r in range(case["rows"]):
            S = state[int(st["before"][r])].clone() if st["before"][r] >= 0 else torch.zeros_like(state[0])
            for t in range(int(st["first"][r]), int(st["first"][r + 1])):
                kt = k[t][..., None]
                M = decay[t][:, None, None] * (eye - (beta[t][:, None, None] * kt) * kt.transpose(1, 2))
                S = torch.baddbmm((beta[t][:, None, None] * kt) * v[t][:, None], M, S)
                out[t] = torch.bmm(q[t][:, None], S)[:, 0] * hd ** -0.5
            new[int(st["after"][r])] = S
        for slot, s in new.items():
            state[slot] = s
    if case["gate"]:
        z = st["z"].double()
        out = out * (out.square().mean(-1, keepdim=True) + EPS).rsqrt() * st["norm_w"].double() * (z * torch.sigmoid(z))
    return [out, state]


def _exact_prefix(case, seed, st):
    H, KV, hd = HEADS[case["heads"]]
    first, prefix, lens = _prefix_plan(case, seed)
    out = torch.empty(case["rows"], H, hd, dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens.tolist()):
        g = int(np.searchsorted(first, r, "right")) - 1
        at = np.arange(n)
        page = np.where(at < prefix[g], st["pages"][first[g]][at // case["page"]], st["pages"][r][at // case["page"]])
        page, off = _dev(page, torch.long), _dev(at % case["page"], torch.long)
        k, v = st["k"][page, :, off].double().transpose(0, 1), st["v"][page, :, off].double().transpose(0, 1)
        s = torch.matmul(st["q"][r].double().reshape(KV, H // KV, hd), k.transpose(1, 2).contiguous())
        out[r] = torch.matmul((s * hd ** -0.5).softmax(-1), v.contiguous()).reshape(H, hd)
    return [out]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "prefix":
        return _exact_prefix(case, seed, st)
    return (_exact_conv if case["op"] == "conv" else _exact_delta)(case, seed, st)
