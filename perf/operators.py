"""What is measured of the rotary embedding, the paged append and the paged attention.

Three operators that serve together: positions rotate queries and keys
(``rotary``), a batch's new keys and values go into a page pool with that
rotation applied on the way (``append``), and the new queries attend to the
pages (``attention``).  A batch is packed: the new tokens of all sequences lie
one behind the other, ``q_start [B+1]`` says where each sequence's begin,
``kv_len [B]`` how many tokens it has with the new ones, and
``block_table [B, W]`` which pages of the pool hold them.

``run`` is the plain form (elementary torch operations in fp32, angles in
fp64) or, where ``own`` is true, the framework's calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# -- cases ---------------------------------------------------------------------------


def _rotary(name, **kw):
    c = dict(name=name, op="rotary", B=1, T=64, H=8, Hk=8, D=64, R=0, dtype="bf16", base=10000.0, sections="",
             interleaved=False, offset=0, grad=False)
    c.update(kw)
    return c


def _paged(name, op, **kw):
    c = dict(name=name, op=op, B=1, new=1, singles=0, past=0, H=32, Hk=8, D=128, page=16, dtype="bf16", causal=True,
             window=0, base=10000.0, shape_seed=1)
    c.update(kw)
    return c


def listed():
    return [
        # the README example's projections: small fp32 tensors, a call's latency
        _rotary("rotary_readme_f32", B=2, T=64, H=8, Hk=8, D=64, dtype="f32"),
        # a training step at the prefill benchmark's sequence and heads: forward and both gradients
        _rotary("rotary_train_bf16", B=1, T=8192, H=32, Hk=32, D=128, grad=True),
        # a video clip's patches in fp16: three axes, adjacent pairs, an odd grid of 13 x 27 x 35
        _rotary("rotary_video_f16", B=2, T=13 * 27 * 35, H=16, Hk=16, D=64, dtype="f16", sections="8,12,12",
                interleaved=True),
        # one decode step of 64 sequences over the decode benchmark's 256-token pages
        _paged("append_decode_bf16", "append", B=64, new=1, past=2048, page=256),
        # a prefill batch of ragged prompts behind ragged histories, 16-token pages
        _paged("append_prefill_f16", "append", B=7, new=4000, past=5000, H=32, Hk=32, page=16, dtype="f16",
               shape_seed=2),
        # one request's next token: the smallest attention call
        _paged("decode_one_bf16", "attention", B=1, new=1, past=4097),
        # the decode benchmark's batch with grouped key heads: ragged caches of up to 32768 tokens
        _paged("decode_batch_bf16", "attention", B=32, new=1, past=32768, page=256, shape_seed=3),
        # one key head to a query head, fp16, a page that divides no tile
        _paged("decode_mha_f16", "attention", B=9, new=1, past=9000, H=16, Hk=16, D=64, page=24, dtype="f16",
               shape_seed=4),
        # the long-context benchmark's 256-query chunk over a 131072-token cache
        _paged("chunk_long_bf16", "attention", B=1, new=256, past=131072 - 256, H=64, Hk=8, page=256),
        # prompts prefilled in chunks over histories of different lengths
        _paged("chunk_prefill_bf16", "attention", B=4, new=2048, past=8192, H=32, Hk=8, page=16, shape_seed=5),
        # a serving step: running sequences' single tokens beside two prompts' chunks, fp16
        _paged("mixed_step_f16", "attention", B=34, new=700, singles=32, past=3000, H=16, Hk=16, D=64, page=16,
               dtype="f16", shape_seed=6),
        # fp32 with the README example's heads, a chunk behind an odd history
        _paged("chunk_f32", "attention", B=2, new=64, past=1000, H=8, Hk=8, D=64, page=16, dtype="f32",
               shape_seed=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([64, 128, 128, 40, 72, 256])
    Hk = rng.choice([1, 2, 4, 8, 16])
    if op == "rotary":
        T, B = _log(rng, 1, 16384), rng.choice([1, 1, 2, 3])
        sections = ""
        R = rng.choice([0, 0, D // 4 * 2])
        if rng.random() < 0.4:  # time, height, width: a quarter, the rest in two
            half = (R or D) // 2
            t, h = half // 4, (half - half // 4) // 2
            sections = "%d,%d,%d" % (t, h, half - t - h)
        return dict(op=op, B=B, T=max(1, T // B), H=Hk * rng.choice([1, 2, 4]), Hk=Hk, D=D, R=R, dtype=dtype,
                    base=rng.choice([10000.0, 500000.0]), sections=sections, interleaved=rng.random() < 0.3,
                    offset=rng.choice([0, 77, 100000]), grad=rng.random() < 0.5)
    c = _paged("", op, H=Hk * rng.choice([1, 2, 4, 8]), Hk=Hk, D=D, page=rng.choice([8, 16, 24, 32, 64, 100, 256]),
               dtype=dtype, shape_seed=rng.randrange(1 << 20))
    del c["name"]
    c["B"] = _log(rng, 1, 48)
    if op == "append":
        c["new"] = _log(rng, 1, max(2, 24000 // c["B"]))
        c["past"] = _log(rng, 1, max(2, 24000 // c["B"]))
        return c
    shape = rng.choice(["decode", "chunk", "mixed"])
    if shape == "decode":
        c["new"] = rng.choice([1, 1, 2, 5])
        c["past"] = _log(rng, 1, min(32768, 400000 // c["B"]))
    else:
        c["B"] = max(1, c["B"] // 4) if shape == "chunk" else max(2, c["B"])
        c["singles"] = 0 if shape == "chunk" else c["B"] - 1 - rng.randrange(min(2, c["B"] - 1))
        c["new"] = _log(rng, 3, 1500)
        c["past"] = _log(rng, 1, 8000 if shape == "chunk" else 4000)
    c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 2000)])
    c["causal"] = c["window"] > 0 or rng.random() < 0.9
    while True:  # no more work than the largest listed case, and scores of a size that the plain form can hold
        new, past = _lengths(c)
        pairs = sum(n * (n + p) for n, p in zip(new, past)) * c["H"] * c["D"]
        if pairs <= 2 ** 36 and c["B"] * max(new) * (max(past) + max(new)) * c["H"] <= 2 ** 31 and \
                c["B"] * (max(past) + max(new)) * c["Hk"] * c["D"] <= 2 ** 31:
            return c
        if c["new"] > 3 and c["new"] >= c["past"] // 4:
            c["new"] = c["new"] * 2 // 3
        else:
            c["past"] = max(1, c["past"] * 2 // 3)


def _lengths(c):
    """New and earlier tokens of each sequence: the last ones bring one token each, the others up to
    ``new`` behind histories of up to ``past``."""
    r = random.Random(c["shape_seed"])
    new = [1 if b >= c["B"] - c["singles"] else c["new"] if b == 0 else r.randint((c["new"] + 1) // 2, c["new"])
           for b in range(c["B"])]
    past = [c["past"] if b == 0 else r.randint(c["past"] // 4, c["past"]) for b in range(c["B"])]
    return new, past


# -- inputs --------------------------------------------------------------------------


def _sections(c):
    return [int(x) for x in c["sections"].split(",")] if c["sections"] else None


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPE[c["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dt)

    H, Hk, D = c["H"], c["Hk"], c["D"]
    s = {"case": c}
    if c["op"] == "rotary":
        B, T = c["B"], c["T"]
        # a projection's output [B, T, H*D], read as [B, H, T, D]
        s["q"] = randn(B, T, H, D).transpose(1, 2)
        s["k"] = randn(B, T, Hk, D).transpose(1, 2)
        if c["sections"]:
            # a clip's patch grid (the grid of the case's T, or as square as it goes), each axis counted on its own
            frames = next(f for f in (13, 5, 3, 2, 1) if T % f == 0)
            wide = max(w for w in range(1, int(math.isqrt(T // frames)) + 1) if (T // frames) % w == 0)
            i = torch.arange(T, device="cuda")
            s["positions"] = torch.stack([i // (T // frames), i // wide % (T // frames // wide), i % wide]) + c["offset"]
        else:
            s["positions"] = None
        if c["grad"]:
            s["q"].requires_grad_()
            s["k"].requires_grad_()
            s["gq"] = randn(B, T, H, D).transpose(1, 2)
            s["gk"] = randn(B, T, Hk, D).transpose(1, 2)
        return s
    new, past = _lengths(c)
    page, N = c["page"], sum(new)
    need = [-(-(n + p) // page) for n, p in zip(new, past)]
    W, pages = max(need), sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    start = torch.tensor([0] + need[:-1], device="cuda").cumsum(0)
    col = torch.arange(W, device="cuda")
    have = torch.tensor(need, device="cuda")
    table = order[(start[:, None] + col).clamp(max=pages - 1)]
    s["block_table"] = torch.where(col < have[:, None], table, torch.zeros_like(table)).contiguous()
    s["kv_len"] = torch.tensor([n + p for n, p in zip(new, past)], device="cuda", dtype=torch.int32)
    s["q_start"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    s["key_pool"] = randn(pages, Hk, page, D)
    s["value_pool"] = randn(pages, Hk, page, D)
    s["max_q_len"], s["max_kv_len"] = max(new), max(n + p for n, p in zip(new, past))
    # scores with a standard deviation of about two: neither flat nor a single key's
    s["q"] = randn(N, H, D, scale=2.0)
    if c["op"] == "append":
        s["k"], s["v"] = randn(N, Hk, D), randn(N, Hk, D)
    return s


# -- the plain form ------------------------------------------------------------------


def _turn(x, angles, interleaved):
    """fp32 ``x [..., D]`` rotated by fp64 ``angles [..., R/2]`` in its first R dimensions, pairs ``(i, i + R/2)``
    or ``(2i, 2i + 1)``."""
    half = angles.shape[-1]
    cos, sin = angles.cos().float(), angles.sin().float()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([y, x[..., 2 * half:]], dim=-1)


def _angles(positions, R, base, sections):
    """fp64 angles ``[T, R/2]`` of positions ``[T]``, or ``[A, T]`` with the frequencies dealt out in sections."""
    half = R // 2
    freq = float(base) ** (torch.arange(half, dtype=torch.float64, device=positions.device) * (-2.0 / R))
    if sections is None:
        return positions.double()[:, None] * freq
    axis = torch.repeat_interleave(torch.arange(len(sections), device=positions.device),
                                   torch.tensor(sections, device=positions.device))
    return positions.double().t()[:, axis] * freq


def _plain_rotary(s):
    c, q, k = s["case"], s["q"].detach(), s["k"].detach()
    pos = s["positions"]
    if pos is None:
        pos = torch.arange(c["T"], device=q.device) + c["offset"]
    ang = _angles(pos, c["R"] or c["D"], c["base"], _sections(c))
    out = {"q": _turn(q.float(), ang, c["interleaved"]).to(q.dtype),
           "k": _turn(k.float(), ang, c["interleaved"]).to(k.dtype)}
    if c["grad"]:  # the transposed rotation, by the negative angle
        out["dq"] = _turn(s["gq"].float(), -ang, c["interleaved"]).to(q.dtype)
        out["dk"] = _turn(s["gk"].float(), -ang, c["interleaved"]).to(k.dtype)
    return out


def _token_places(s):
    """Of each packed token: its sequence, its position in it, and the pool page and slot of that position."""
    c, start = s["case"], s["q_start"].long()
    i = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(start[1:], i, right=True)
    pos = s["kv_len"].long()[seq] - start[seq + 1] + i
    return seq, pos, s["block_table"][seq, pos // c["page"]].long(), pos % c["page"]


def _plain_append(s):
    c = s["case"]
    _, pos, page, slot = _token_places(s)
    ang = _angles(pos, c["D"], c["base"], None)[:, None]
    s["key_pool"][page, :, slot] = _turn(s["k"].float(), ang, False).to(s["k"].dtype)
    s["value_pool"][page, :, slot] = s["v"]
    return {"key_pool": s["key_pool"], "value_pool": s["value_pool"],
            "q": _turn(s["q"].float(), ang, False).to(s["q"].dtype)}


def _plain_attention(s):
    """Every sequence padded to the longest: gathered pages, masked scores, softmax, weighted values."""
    c = s["case"]
    B, H, Hk, D, most = c["B"], c["H"], c["Hk"], c["D"], s["max_q_len"]
    seq, pos, _, _ = _token_places(s)
    local = torch.arange(s["q"].shape[0], device="cuda") - s["q_start"].long()[seq]
    q = s["q"].new_zeros(B, most, H, D)
    q[seq, local] = s["q"]
    qpos = torch.full((B, most), -1, device="cuda")
    qpos[seq, local] = pos
    table = s["block_table"].long()

    def gathered(pool):  # [B, Hk, W * page, D]
        return pool[table].permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D).float()

    j = torch.arange(table.shape[1] * c["page"], device="cuda")
    seen = j < s["kv_len"].long()[:, None, None]
    if c["causal"]:
        seen = seen & (j <= qpos[:, :, None])
    if c["window"]:
        seen = seen & (j > qpos[:, :, None] - c["window"])
    rows = q.view(B, most, Hk, H // Hk, D).transpose(1, 2).reshape(B, Hk, most * (H // Hk), D).float()
    p = torch.matmul(rows, gathered(s["key_pool"]).transpose(2, 3)).mul_(D ** -0.5)
    p.masked_fill_(~seen.repeat_interleave(H // Hk, 1)[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    total = p.sum(-1, keepdim=True)
    # the values of slots that nobody has written yet are not read as numbers
    v = gathered(s["value_pool"]).masked_fill_(~(j < s["kv_len"].long()[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(p, v).div_(total).nan_to_num_(0.0)
    out = out.view(B, Hk, most, H // Hk, D).transpose(1, 2).reshape(B, most, H, D)
    return out[seq, local].to(s["q"].dtype)


# -- the framework's calls -------------------------------------------------------------


def _embedding(s):
    """The rotary embedding that a program keeps beside its weights."""
    if "embedding" not in s:
        from avqa_b200 import RotaryEmbedding
        c = s["case"]
        s["embedding"] = RotaryEmbedding(c["D"], base=c["base"], rotary_dim=c.get("R") or None,
                                         sections=_sections(c) if c["op"] == "rotary" else None,
                                         interleaved=c.get("interleaved", False))
    return s["embedding"]


def _own_rotary(s):
    c = s["case"]
    q, k = _embedding(s)(s["q"], s["k"], positions=s["positions"], offset=0 if c["sections"] else c["offset"])
    out = {"q": q, "k": k}
    if c["grad"]:
        out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
    return out


def _own_append(s):
    from avqa_b200 import ops
    q = ops.paged_append(s["k"], s["v"], s["key_pool"], s["value_pool"], s["block_table"], s["kv_len"], s["q_start"],
                         q=s["q"], rotary=_embedding(s))
    return {"key_pool": s["key_pool"], "value_pool": s["value_pool"], "q": q}


def _own_attention(s):
    from avqa_b200 import ops
    c = s["case"]
    return ops.paged_attention(s["q"], s["key_pool"], s["value_pool"], s["block_table"], s["kv_len"], s["q_start"],
                               causal=c["causal"], window=c["window"], max_q_len=s["max_q_len"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "attention": _own_attention}[op](state)
    return {"rotary": _plain_rotary, "append": _plain_append, "attention": _plain_attention}[op](state)


# -- work and exact values -------------------------------------------------------------


def _pairs(c):
    """Visible (query, key) pairs of a batch, and the keys that at least one query sees."""
    pairs = keys = 0
    for n, p in zip(*_lengths(c)):
        if not c["causal"]:
            pairs, keys = pairs + n * (n + p), keys + n + p
        elif not c["window"]:
            pairs, keys = pairs + n * p + n * (n + 1) // 2, keys + n + p
        else:
            w = c["window"]
            pairs += sum(min(w, p + i + 1) for i in range(n))
            keys += min(n + p, n + w - 1)
    return pairs, keys


def work(c):
    size = {"f32": 4, "bf16": 2, "f16": 2}[c["dtype"]]
    H, Hk, D = c["H"], c["Hk"], c["D"]
    if c["op"] == "rotary":
        rows = c["B"] * c["T"] * (H + Hk)
        passes = 2 if c["grad"] else 1
        pos = 0 if not c["sections"] else 3 * 8 * c["T"]
        return {"bytes": passes * (2 * rows * D * size + pos), "flops": passes * rows * 3 * (c["R"] or D)}
    new, past = _lengths(c)
    N = sum(new)
    lists = 4 * sum(-(-(n + p) // c["page"]) for n, p in zip(new, past)) + 8 * c["B"]
    if c["op"] == "append":
        return {"bytes": 2 * N * (H + 2 * Hk) * D * size + 8 * c["B"] + 4 * N, "flops": 3 * N * (H + Hk) * D}
    pairs, keys = _pairs(c)
    return {"bytes": 2 * N * H * D * size + 2 * keys * Hk * D * size + lists, "flops": 4 * pairs * H * D}


def _exact_turn(x, pos, c, sign):
    """x [..., D] as complex numbers times exp(i * angle), in 64 bits; pos [A, T] on the tokens of x's dim -2."""
    R = (c.get("R") or c["D"]) if c["op"] == "rotary" else c["D"]
    half = R // 2
    per = (_sections(c) or [half]) if c["op"] == "rotary" else [half]
    cols = []
    for a, n in enumerate(per):
        for i in range(sum(per[:a]), sum(per[:a]) + n):
            cols.append(pos[a].double() / c["base"] ** (2.0 * i / R))
    ang = sign * torch.stack(cols, -1)
    rot = torch.polar(torch.ones_like(ang), ang)
    y = x.double().clone()
    if c.get("interleaved"):
        z = torch.complex(y[..., 0:R:2].contiguous(), y[..., 1:R:2].contiguous()) * rot
        y[..., 0:R:2], y[..., 1:R:2] = z.real, z.imag
    else:
        z = torch.complex(y[..., :half].contiguous(), y[..., half:R].contiguous()) * rot
        y[..., :half], y[..., half:R] = z.real, z.imag
    return y


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rotary":
        pos = s["positions"]
        if pos is None:
            pos = (c["offset"] + torch.arange(c["T"], device="cuda"))[None]
        out = {n: _exact_turn(s[n].detach(), pos, c, 1.0) for n in ("q", "k")}
        if c["grad"]:
            out |= {"d" + n: _exact_turn(s["g" + n], pos, c, -1.0) for n in ("q", "k")}
        return out
    new, past = _lengths(c)
    starts = [sum(new[:b]) for b in range(c["B"])]
    page = c["page"]
    if c["op"] == "append":
        kp, vp = s["key_pool"].double(), s["value_pool"].double()
        q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, (n, p, at) in enumerate(zip(new, past, starts)):
            pos = torch.arange(p, p + n, device="cuda")
            where = s["block_table"][b].long()[pos // page], pos % page
            rows = slice(at, at + n)
            kp[where[0], :, where[1]] = _exact_turn(s["k"][rows].transpose(0, 1), pos[None], c, 1.0).transpose(0, 1)
            vp[where[0], :, where[1]] = s["v"][rows].double()
            q[rows] = _exact_turn(s["q"][rows].transpose(0, 1), pos[None], c, 1.0).transpose(0, 1)
        return {"key_pool": kp, "value_pool": vp, "q": q}
    if 4 * _pairs(c)[0] * c["H"] * c["D"] > 4e12:
        return None
    G = c["H"] // c["Hk"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (n, p, at) in enumerate(zip(new, past, starts)):
        L = n + p
        pages = s["block_table"][b, :-(-L // page)].long()
        kb = s["key_pool"][pages].transpose(0, 1).reshape(c["Hk"], -1, c["D"])[:, :L]
        vb = s["value_pool"][pages].transpose(0, 1).reshape(c["Hk"], -1, c["D"])[:, :L]
        at_pos = torch.arange(p, L, device="cuda")[:, None]
        j = torch.arange(L, device="cuda")[None]
        hidden = torch.zeros(n, L, dtype=torch.bool, device="cuda")
        if c["causal"]:
            hidden |= j > at_pos
        if c["window"]:
            hidden |= at_pos - j >= c["window"]
        for h in range(c["H"]):
            x = s["q"][at:at + n, h].double() @ kb[h // G].double().t() / math.sqrt(c["D"])
            x[hidden] = -math.inf
            out[at:at + n, h] = torch.softmax(x, -1) @ vb[h // G].double()
    return out
