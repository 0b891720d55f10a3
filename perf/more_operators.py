"""Cases of the operators of a step of speculative sampling over sequences that share a prompt: rotary positions, attention
over the 4-bit cache with a window and first positions that stay visible (sinks), attention of groups of sequences that share a
prefix, and the verification of drafted tokens. Shapes are those of the model driver's configurations (qwen35.py) and of common
grouped-query heads.

The cache holds, per sequence and KV head, one record for every 32 positions (NB = dim / 32 blocks of Q4_0 values along
the head):
    key quants   [sub 2][c][g 4][p 16][b][e 4]  byte of block 4 c + b (b < min(NB, 4)) at position 16 sub + p: low nibble the
                                                element 32 block + 4 g + e, high nibble the one 16 further
    value quants [c][g 4][n 16][b][sub 2][r 4]  byte of block 2 c + b (b < min(NB, 2)) at position 16 sub + 4 g + r: low
                                                nibble the element 32 block + n, high nibble the one 16 further
    key scales   [g 4][block NB][sub 2][r 4]    fp16, position 16 sub + 4 g + r
    value scales likewise
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fpga-llama-gguf_amd")
DEV = "cuda"
HEADS = [(16, 4, 256), (8, 2, 256), (16, 4, 128), (4, 1, 128), (32, 8, 128), (8, 8, 64), (6, 2, 32)]


def _attn(groups, members, tokens, heads, prefix, len, window=0, sinks=0, ragged=False) -> dict:
    """prefix < 0: every sequence has its whole cache (members 1)."""
    h, hk, hd = heads
    return {"kind": "attn", "groups": groups, "members": members, "tokens": tokens, "heads": h, "kv_heads": hk, "dim": hd,
            "prefix": prefix, "len": len, "window": window, "sinks": sinks, "ragged": ragged}


def _rope(seqs, tokens, heads, rot, layout, scaling, base, far, ragged=False) -> dict:
    h, hk, hd = heads
    return {"kind": "rope", "seqs": seqs, "tokens": tokens, "heads": h, "kv_heads": hk, "dim": hd, "rot": rot, "layout": layout,
            "scaling": scaling, "base": base, "far": far, "ragged": ragged}


def _verify(seqs, drafts, vocab, temp=1.0, rows=True, masked=False, ragged=False) -> dict:
    """rows: the draft's logits are given; without them its tokens are certain (found in the prompt, say)."""
    return {"kind": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "temp": temp, "rows": rows, "masked": masked,
            "ragged": ragged}


def listed() -> list[dict]:
    return [
        # four samples of one short prompt, in the driver's own attention layer: what a launch costs
        {"name": "samples 1x4 behind 512 d256", **_attn(1, 4, 1, (16, 4, 256), 512, 128)},
        # many chats behind one system prompt, each at a place of its own, some not in use
        {"name": "chats 1x32 behind 8192 d128", **_attn(1, 32, 1, (32, 8, 128), 8192, 1024, ragged=True)},
        # samples of two long documents
        {"name": "samples 2x16 behind 30000 d256", **_attn(2, 16, 1, (16, 4, 256), 30000, 640)},
        # a few drafted tokens of a few sequences, a window that reaches into the prefix, odd sizes
        {"name": "drafts 3x5x4 behind 1503 d64", **_attn(3, 5, 4, (8, 8, 64), 1503, 301, 1000, 3, True)},
        # one token of an endless stream: a window and the first tokens of a long cache
        {"name": "stream 1x32768 w4096+4 d256", **_attn(1, 1, 1, (16, 4, 256), -1, 32768, 4096, 4)},
        # 32 sequences in lockstep, each at a position of its own
        {"name": "lockstep 32x8192 w1024+64 d128", **_attn(32, 1, 1, (32, 8, 128), -1, 8192, 1024, 64, True)},
        # a chunk of a long prompt
        {"name": "prompt 512 at 7680 w1024+4 d256", **_attn(1, 1, 512, (16, 4, 256), -1, 8192, 1024, 4)},
        # one token of the driver's model: 64 of 256 elements turn
        {"name": "rope 1 h16/4 d256 half 64", **_rope(1, 1, (16, 4, 256), 64, "half", "none", 1e7, 640)},
        # a whole prompt at far positions of a stretched context, whole heads, pairs of neighbours
        {"name": "rope 4096 h32/8 d128 pairs", **_rope(1, 4096, (32, 8, 128), 128, "pairs", "yarn", 1e6, 131072)},
        # four drafted tokens of one sequence
        {"name": "verify 1x4 of 151936", **_verify(1, 4, 151936)},
        # those of a batch
        {"name": "verify 32x4 of 151936", **_verify(32, 4, 151936, temp=0.8)},
        # tokens found in the prompt, an odd vocabulary, part of it ruled out, fewer of them for some
        {"name": "verify 61x3 of 32003 certain", **_verify(61, 3, 32003, rows=False, masked=True, ragged=True)},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number whose logarithm is spread evenly over lo..hi."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _draw(rng) -> dict:
    kind = rng.choice(["shared", "shared", "sinks", "rope", "verify"])
    ragged = rng.random() < 0.5
    if kind == "shared":
        members = _spread(rng, 2, 32)
        tokens = 1 if rng.random() < 0.6 else rng.randint(2, 8)
        n = tokens + _spread(rng, 1, 1024)
        prefix = _spread(rng, 32, 30000)
        window = _spread(rng, 16, prefix + n) if rng.random() < 0.3 else 0
        return _attn(_spread(rng, 1, 8), members, tokens, rng.choice(HEADS), prefix, n, window, rng.randint(0, 70) if window else 0, ragged)
    if kind == "sinks":
        n = _spread(rng, 64, 32768)
        tokens = 1 if rng.random() < 0.5 else _spread(rng, 2, min(n, 512))
        return _attn(_spread(rng, 1, 32), 1, tokens, rng.choice(HEADS), -1, n, _spread(rng, 16, min(n, 4096)), _spread(rng, 1, 100), ragged)
    if kind == "rope":
        h, hk, hd = heads = rng.choice(HEADS)
        seqs = _spread(rng, 1, 32)
        tokens = 1 if rng.random() < 0.4 else _spread(rng, 2, 4096 // seqs)
        return _rope(seqs, tokens, heads, rng.choice([hd, hd, hd // 2, hd // 4, hd // 2 - 6]), rng.choice(["half", "pairs"]),
                     rng.choice(["none", "linear", "yarn", "factors"]), rng.choice([1e4, 5e5, 1e6, 1e7]), tokens + _spread(rng, 1, 1 << 18), ragged)
    return _verify(_spread(rng, 1, 64), rng.randint(1, 8), _spread(rng, 1000, 151936), rng.choice([0.6, 0.8, 1.0, 1.0]), rng.random() < 0.7,
                   rng.random() < 0.3, ragged)


def draw(rng) -> dict:
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["kind"], (0, 0))
        most[c["kind"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        c = _draw(rng)
        w = work(c)
        size = c["groups"] * c["members"] * c["len"] + c["groups"] * max(c["prefix"], 0) if c["kind"] == "attn" else 0
        if w["bytes"] <= most[c["kind"]][0] and w["flops"] <= most[c["kind"]][1] and size <= 32 * 8192:
            if size * (c["kv_heads"] * c["dim"] if size else 0) <= 32 * 8192 * 1024:
                return c


# ---- the cache ----------------------------------------------------------------------------------------------------
def _quantize(x: torch.Tensor):
    """Q4_0 of the last axis in FP32, in blocks of 32: nibbles [..., nb, 32] and fp16 scales [..., nb]."""
    b = x.unflatten(-1, (-1, 32))
    top = b.gather(-1, b.abs().argmax(-1, keepdim=True))
    d = top / -8
    inv = torch.where(d != 0, 1 / d, 0)
    q = (b * inv + 8.5).clamp(0, 15).to(torch.uint8)
    return q, d[..., 0].half()


def _records(kq, kd, vq, vd) -> torch.Tensor:
    """Nibbles [S, H, L, NB, 32] and scales [S, H, L, NB] (L a multiple of 32) as records [S, H, L / 32, 36 * 32 NB]."""
    s, h, n, nb, _ = kq.shape
    t, kc, vc = n // 32, max(1, nb // 4), max(1, nb // 2)
    pack = lambda q: q[..., :16] | q[..., 16:] << 4  # noqa: E731
    k = pack(kq).view(s, h, t, 2, 16, kc, nb // kc, 4, 4).permute(0, 1, 2, 3, 5, 7, 4, 6, 8)
    v = pack(vq).view(s, h, t, 2, 4, 4, vc, nb // vc, 16).permute(0, 1, 2, 6, 4, 8, 7, 3, 5)
    d = [x.view(s, h, t, 2, 4, 4, nb).permute(0, 1, 2, 4, 6, 3, 5).reshape(s, h, t, -1).view(torch.uint8) for x in (kd, vd)]
    return torch.cat([k.reshape(s, h, t, -1), v.reshape(s, h, t, -1), *d], -1)


def _values(rec: torch.Tensor, nb: int):
    """Keys and values [S, H, L, 32 NB] that the records stand for, in FP32."""
    s, h, t, _ = rec.shape
    hd, kc, vc = 32 * nb, max(1, nb // 4), max(1, nb // 2)
    kq, vq, kd, vd = rec.split([16 * hd, 16 * hd, 2 * hd, 2 * hd], -1)
    scale = [x.contiguous().view(torch.half).view(s, h, t, 4, nb, 2, 4).permute(0, 1, 2, 5, 3, 6, 4).reshape(s, h, 32 * t, nb, 1)
             for x in (kd, vd)]
    k = kq.reshape(s, h, t, 2, kc, 4, 16, nb // kc, 4).permute(0, 1, 2, 3, 6, 4, 7, 5, 8).reshape(s, h, 32 * t, nb, 16)
    v = vq.reshape(s, h, t, vc, 4, 16, nb // vc, 2, 4).permute(0, 1, 2, 7, 4, 8, 3, 6, 5).reshape(s, h, 32 * t, nb, 16)
    return [((torch.cat([q & 15, q >> 4], -1).float() - 8) * d.float()).flatten(-2) for q, d in zip((k, v), scale)]


# ---- inputs -------------------------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(DEV).manual_seed(seed)


def _places(case: dict, seqs: int, tokens: int, most: int, uniform) -> tuple:
    """The sequences' first positions and numbers of tokens; ragged: places of their own, fewer tokens, one of them not in use."""
    pos, num = torch.full((seqs,), most - tokens, device=DEV), torch.full((seqs,), tokens, device=DEV)
    if case["ragged"]:
        pos = ((most - tokens + 1) * uniform(seqs)).long().clamp(max=most - tokens)
        num = 1 + (tokens * uniform(seqs)).long().clamp(max=tokens - 1)
        if seqs > 2:
            pos[1], num[1] = -1, 0
    return pos.int(), num.int()


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    normal = lambda *n: torch.randn(*n, generator=g, device=DEV)  # noqa: E731
    uniform = lambda *n: torch.rand(*n, generator=g, device=DEV)  # noqa: E731
    st = {"case": case}
    if case["kind"] == "attn":
        s, t, h, hk, hd = case["groups"] * case["members"], *(case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        gain = (0.3 * normal(2, hk, 1, hd)).exp()  # channels of unlike size

        def cache(seqs, n):
            n = -(-n // 32) * 32
            kv = [_quantize(normal(seqs, hk, n, hd) * gain[i]) for i in range(2)]
            return _records(*kv[0], *kv[1]).contiguous()

        st["cache"] = cache(s, case["len"])  # the tokens' own keys and values stored already
        if case["prefix"] >= 0:
            st["prefix"] = cache(case["groups"], case["prefix"])
            n = torch.full((case["groups"],), case["prefix"], device=DEV)
            if case["ragged"]:
                n = (n * (0.5 + 0.5 * uniform(case["groups"]))).long()
            st["prefix_len"] = n.int()
        st["pos"], st["num"] = _places(case, s, t, case["len"], uniform)
        st["q"] = 1.5 * normal(s, t, h, hd)
        st["y"] = torch.zeros(s, t, h, hd, device=DEV)
        return st
    if case["kind"] == "rope":
        s, t, h, hk, hd = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim"))
        st["pos"], st["num"] = _places(case, s, t, case["far"], uniform)
        st["q"], st["k"] = normal(s, t, h, hd), normal(s, t, hk, hd)
        st["q_out"], st["k_out"] = torch.zeros_like(st["q"]), torch.zeros_like(st["k"])
        if case["scaling"] == "factors":  # a model's own stretch of every pair
            st["factors"] = (1 + 7 * uniform(case["rot"] // 2).sort()[0]).cpu().double().numpy()
        return st
    s, k, n = (case[x] for x in ("seqs", "drafts", "vocab"))
    x = 2.5 * normal(s, k + 1, n)
    if case["masked"]:  # tokens that a grammar rules out
        x[uniform(s, k + 1, n) < 0.4] = -math.inf
    st["target"] = x
    y = x[:, :k] + 1.0 * normal(s, k, n)  # a smaller model's, somewhat off
    if case["rows"]:
        st["draft"] = y
    c = torch.softmax(y.double() / case["temp"], -1).cumsum(-1)
    st["token"] = torch.searchsorted(c, (uniform(s, k, 1).double() * c[..., -1:]), right=True)[..., 0].clamp(max=n - 1).int()
    st["uniform"] = uniform(s, k + 1)
    num = torch.full((s,), k, device=DEV)
    if case["ragged"]:
        num = ((k + 1) * uniform(s)).long().clamp(max=k)
        if s > 2:
            num[1] = -1  # not in use
    st["num"] = num.int()
    st["n_accept"] = torch.full((s,), -1, dtype=torch.int32, device=DEV)
    st["out"] = torch.full((s, k + 1), -1, dtype=torch.int32, device=DEV)
    st["logp"] = torch.zeros(s, k + 1, device=DEV)
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(st: dict):
    if own:
        return _own(st)
    return {"attn": _plain_attn, "rope": _plain_rope, "verify": _plain_verify}[st["case"]["kind"]](st)


def _plain_attn(st):
    case = st["case"]
    groups, mem, t, h, hk, hd = (case[k] for k in ("groups", "members", "tokens", "heads", "kv_heads", "dim"))
    s, g = groups * mem, h // hk
    at = st["pos"].long()[:, None] + torch.arange(t, device=DEV)  # the tokens' places in their own caches
    live = (torch.arange(t, device=DEV) < st["num"][:, None]) & (st["pos"][:, None] >= 0)
    plen = st["prefix_len"].long().repeat_interleave(mem)[:, None] if "prefix" in st else torch.zeros(s, 1, dtype=torch.long, device=DEV)
    far = at + plen
    q = st["q"].view(s, t, hk, g, hd).permute(0, 2, 1, 3, 4)

    def scores(q, k):
        return torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)

    def hide(x, place, j):  # x [s, hk, t, g, n]: places j of the sequences, positions `place` of theirs
        seen = live[..., None] & (place <= far[..., None])
        if case["window"]:
            seen &= (place > far[..., None] - case["window"]) | (place < case["sinks"])
        x.masked_fill_(~(seen & j)[:, None, :, None], -math.inf)

    k, v = _values(st["cache"], hd // 32)
    j = torch.arange(k.shape[2], device=DEV)
    x = scores(q.reshape(s, hk, t * g, hd), k).view(s, hk, t, g, -1)
    hide(x, plen[..., None] + j, torch.ones_like(j, dtype=torch.bool))
    top = x.amax(-1, keepdim=True)
    if "prefix" in st:
        pk, pv = _values(st["prefix"], hd // 32)
        j = torch.arange(pk.shape[2], device=DEV)
        shared = q.view(groups, mem, hk, t, g, hd).transpose(1, 2).reshape(groups, hk, mem * t * g, hd)
        px = scores(shared, pk).view(groups, hk, mem, t, g, -1).transpose(1, 2).reshape(s, hk, t, g, -1)
        hide(px, j, j < plen[..., None])
        top = torch.maximum(top, px.amax(-1, keepdim=True))
    top = top.clamp(min=-1e30)
    x = torch.exp(x - top)
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(s, hk, t * g, -1), v).view(s, hk, t, g, hd)
    if "prefix" in st:
        px = torch.exp(px - top)
        total += px.sum(-1, keepdim=True)
        px = px.view(groups, mem, hk, t, g, -1).transpose(1, 2).reshape(groups, hk, mem * t * g, -1)
        y += torch.matmul(px, pv).view(groups, hk, mem, t, g, hd).transpose(1, 2).reshape(s, hk, t, g, hd)
    return {"y": (y / total.clamp(min=1e-30)).permute(0, 2, 1, 3, 4).reshape(s, t, h, hd)}


# Scaled positions: linear, a context stretched 4 times; YaRN, one of 32768 stretched 4 times with the usual ramp; a factor a pair.
STRETCH, CONTEXT, FAST, SLOW = 4.0, 32768, 32.0, 1.0


def _plain_rope(st):
    case = st["case"]
    s, t, hd, rot = (case[k] for k in ("seqs", "tokens", "dim", "rot"))
    i = torch.arange(rot // 2, device=DEV, dtype=torch.double)
    theta, size = case["base"] ** (-2 * i / rot), 1.0
    if case["scaling"] == "linear":
        theta = theta / STRETCH
    elif case["scaling"] == "factors":
        theta = theta / torch.from_numpy(st["factors"]).to(DEV)
    elif case["scaling"] == "yarn":
        low, high = (rot * math.log(CONTEXT / (2 * math.pi * b)) / (2 * math.log(case["base"])) for b in (FAST, SLOW))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        theta = theta * (1 - ramp) + theta / STRETCH * ramp
        size = 0.1 * math.log(STRETCH) + 1
    at = st["pos"].long()[:, None] + torch.arange(t, device=DEV)
    live = ((torch.arange(t, device=DEV) < st["num"][:, None]) & (st["pos"][:, None] >= 0))[..., None, None]
    angle = at.double()[..., None, None] * theta
    c, n = (angle.cos() * size).float(), (angle.sin() * size).float()
    out = {}
    for name in ("q", "k"):
        x = st[name]
        if case["layout"] == "half":
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            y = torch.cat([a * c - b * n, a * n + b * c, x[..., rot:]], -1)
        else:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.cat([torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2), x[..., rot:]], -1)
        out[name] = torch.where(live, y, 0)
    return out


def _plain_verify(st):
    case = st["case"]
    s, k, n = (case[x] for x in ("seqs", "drafts", "vocab"))
    num, token, u = st["num"].long(), st["token"].long(), st["uniform"].double()

    def dist(x):  # in 64 bits: sums of many terms next to a random number
        e = torch.exp((x.double() - x.amax(-1, keepdim=True)) / case["temp"])
        return e / e.sum(-1, keepdim=True)

    p = dist(st["target"])
    if "draft" in st:
        q = dist(st["draft"])
        qd = q.gather(-1, token[..., None])[..., 0]
    else:
        q, qd = None, torch.ones_like(u[:, :k])
    pd = p[:, :k].gather(-1, token[..., None])[..., 0]
    ok = (u[:, :k] * qd < pd) & (torch.arange(k, device=DEV) < num[:, None])
    a = ok.long().cumprod(-1).sum(-1)  # tokens accepted before the first that is not
    row = torch.arange(s, device=DEV)
    w = p[row, a]
    turned = (a < num)[:, None]
    before = a.clamp(max=k - 1)
    if q is not None:
        less = q[row, before]
    else:
        less = torch.zeros_like(w).scatter_(-1, token[row, before][:, None], 1.0)
    w = torch.where(turned, (w - less).clamp(min=0), w)
    c = w.cumsum(-1)
    new = torch.searchsorted(c, u[:, k:] * c[:, -1:], right=True)[:, 0].clamp(max=n - 1)
    j = torch.arange(k + 1, device=DEV)
    padded = torch.cat([token, token.new_zeros(s, 1)], -1)
    out = torch.where(j < a[:, None], padded, torch.where(j == a[:, None], new[:, None], -1))
    out = torch.where((num >= 0)[:, None], out, -1)
    logp = p.gather(-1, out.clamp(min=0)[..., None])[..., 0].log()
    return {"n_accept": torch.where(num >= 0, a, -1).int(), "out": out.int(), "logp": torch.where(out >= 0, logp, 0).float()}


def _own(st):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import gemvq as gq
    case, stream = st["case"], torch.cuda.current_stream().cuda_stream
    p = lambda x: x.data_ptr()  # noqa: E731
    if case["kind"] == "attn":
        s, t, h, hk, hd = case["groups"] * case["members"], *(case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        shared = "prefix" in st
        if "handle" not in st:
            st["handle"] = gq.Kv4(p(st["cache"]), s, 32 * st["cache"].shape[2], hk, hd)
            if shared:
                st["prefix_handle"] = gq.Kv4(p(st["prefix"]), case["groups"], 32 * st["prefix"].shape[2], hk, hd)
                need = gq.kv4_attn_shared_work(st["handle"], st["prefix_handle"], t, h)
            else:
                need = gq.kv4_attn_sink_work(st["handle"], t, h)
            st["work"] = torch.empty(need, dtype=torch.uint8, device=DEV)
        rest = (p(st["q"]), h * hd, hd, p(st["y"]), h * hd, t, h, p(st["pos"]), p(st["num"]), case["window"], case["sinks"],
                1 / math.sqrt(hd), p(st["work"]), st["work"].numel(), stream)
        if shared:
            gq.kv4_attn_shared_static(st["handle"], st["prefix_handle"], p(st["prefix_len"]), *rest)
        else:
            gq.kv4_attn_sink_static(st["handle"], *rest)
        return {"y": st["y"]}
    if case["kind"] == "rope":
        s, t, h, hk, hd, rot = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "rot"))
        if "freqs" not in st:
            how = {"none": {}, "linear": {"factor": STRETCH}, "factors": {"factors": st.get("factors")},
                   "yarn": {"factor": STRETCH, "yarn_ctx": CONTEXT, "beta_fast": FAST, "beta_slow": SLOW}}[case["scaling"]]
            st["freqs"] = torch.from_numpy(gq.rope_freqs(rot, case["base"], **how)).to(DEV)
            rows = [gq.RopeRows(p(st[n]), p(st[n + "_out"]), m * hd, hd, m * hd, hd, m) for n, m in (("q", h), ("k", hk))]
            st["rows"] = (gq.RopeRows * 2)(*rows)
        gq.rope_static(st["rows"], s, t, hd, rot, gq.ROPE_HALF if case["layout"] == "half" else gq.ROPE_PAIRS, p(st["freqs"]),
                       p(st["pos"]), p(st["num"]), stream)
        return {"q": st["q_out"], "k": st["k_out"]}
    s, k, n = (case[x] for x in ("seqs", "drafts", "vocab"))
    if "work" not in st:
        st["work"] = torch.empty(gq.draft_work(s, k, n), dtype=torch.uint8, device=DEV)
    draft = p(st["draft"]) if case["rows"] else 0
    gq.draft_verify_static(p(st["target"]), n, draft, n, n, s, k, p(st["token"]), p(st["num"]), p(st["uniform"]), case["temp"],
                           case["temp"], p(st["n_accept"]), p(st["out"]), p(st["logp"]), p(st["work"]), st["work"].numel(), stream)
    return {"n_accept": st["n_accept"], "out": st["out"], "logp": st["logp"]}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case: dict) -> dict:
    if case["kind"] == "attn":
        s, t, h, hk, hd = case["groups"] * case["members"], *(case[k] for k in ("tokens", "heads", "kv_heads", "dim"))
        share = 0.5 if case["ragged"] else 1.0  # sequences at places of their own: half of the positions on average
        rows = s * t * (0.5 if case["ragged"] and t > 1 else 1.0)
        mine, pre = case["len"] * share, max(case["prefix"], 0) * (0.75 if case["ragged"] else 1.0)
        each, own_seen, pre_seen = pre + mine - t / 2, mine, pre
        if case["window"]:
            each = min(each, case["window"] + case["sinks"])
            own_seen = min(mine, case["window"] + t + case["sinks"])
            pre_seen = min(pre, max(0, case["window"] + t - mine * 0.5) + case["sinks"])
        return {"bytes": (s * own_seen + case["groups"] * pre_seen) * hk * hd * 9 / 8 + 8 * rows * hd * h,
                "flops": 4 * rows * h * hd * max(each, 1)}
    if case["kind"] == "rope":
        rows = case["seqs"] * case["tokens"] * (0.5 if case["ragged"] and case["tokens"] > 1 else 1.0)
        n = rows * (case["heads"] + case["kv_heads"])
        return {"bytes": 8 * n * case["dim"], "flops": 3 * n * case["rot"]}
    rows = case["seqs"] * (case["drafts"] * (2 if case["rows"] else 1) * (0.5 if case["ragged"] else 1.0) + 1)
    return {"bytes": 4 * rows * case["vocab"], "flops": 4 * rows * case["vocab"]}


# ---- the outputs in 64 bits -------------------------------------------------------------------------------------------
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "rope": _exact_rope, "verify": _exact_verify}[case["kind"]](case, st)


def _where_in_record(hd: int):
    """The byte, the shift and the scale's place in a record of every (position, element), keys and values."""
    p, e = (torch.arange(32, device=DEV)[:, None], torch.arange(hd, device=DEV)[None])
    nb, blk, i = hd // 32, e // 32, e % 16
    half, kb, vb = e % 32 // 16, min(nb, 4), min(nb, 2)
    k = (p // 16) * 8 * hd + (blk // 4) * 1024 + ((i // 4) * 16 + p % 16) * 4 * kb + blk % 4 * 4 + i % 4
    v = 16 * hd + (blk // 2) * 1024 + (p % 16 // 4 * 16 + i) * 8 * vb + blk % 2 * 8 + p // 16 * 4 + p % 4
    d = 16 * hd + (p % 16 // 4 * nb + blk) * 8 + p // 16 * 4 + p % 4  # in fp16 units from the record's start
    return k, v, 4 * half.expand(32, hd), d, d + hd


def _exact_attn(case, st):
    mem, t, h, hk, hd = (case[k] for k in ("members", "tokens", "heads", "kv_heads", "dim"))
    s = case["groups"] * mem
    kat, vat, shift, kd, vd = _where_in_record(hd)

    def unpack(rec):
        sc = rec.view(torch.half)
        k = ((rec[:, kat] >> shift & 15).double() - 8) * sc[:, kd].double()
        v = ((rec[:, vat] >> shift & 15).double() - 8) * sc[:, vd].double()
        return k.view(-1, hd), v.view(-1, hd)

    y = torch.zeros(s, t, h, hd, dtype=torch.float64, device=DEV)
    pos, num = st["pos"].tolist(), st["num"].tolist()
    plen = st["prefix_len"].tolist() if "prefix" in st else [0] * s
    for kh in range(hk):
        held = None  # a group's keys and values of the prefix
        for i in range(s):
            if pos[i] < 0 or num[i] == 0:
                continue
            m, g = pos[i] + num[i], i // mem
            k, v = (x[:m] for x in unpack(st["cache"][i, kh, : -(-m // 32)]))
            n = plen[g]
            if n:
                if held is None or held[0] != g:
                    held = (g, *(x[:n] for x in unpack(st["prefix"][g, kh, : -(-n // 32)])))
                k, v = torch.cat([held[1], k]), torch.cat([held[2], v])
            at = n + pos[i] + torch.arange(num[i], device=DEV)
            j = torch.arange(n + m, device=DEV)
            seen = j <= at[:, None]
            if case["window"]:
                seen &= (j > at[:, None] - case["window"]) | (j < case["sinks"])
            kt = k.t().contiguous()
            for qh in range(kh * h // hk, (kh + 1) * h // hk):
                x = (st["q"][i, : num[i], qh].double() @ kt) * hd ** -0.5
                y[i, : num[i], qh] = torch.softmax(torch.where(seen, x, -math.inf), -1) @ v
    return {"y": y}


def _exact_rope(case, st):
    """Each pair as a complex number, turned."""
    s, t, hd, rot, base = (case[k] for k in ("seqs", "tokens", "dim", "rot", "base"))
    theta, size = np.array([base ** (-2 * i / rot) for i in range(rot // 2)]), 1.0
    if case["scaling"] == "linear":
        theta = theta / STRETCH
    elif case["scaling"] == "factors":
        theta = theta / st["factors"]
    elif case["scaling"] == "yarn":
        # pairs that turn more than FAST times over the context stay, those below SLOW times are slowed down
        edge = [rot * math.log(CONTEXT / (b * 2 * math.pi)) / math.log(base) / 2 for b in (FAST, SLOW)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), rot - 1)
        for i in range(rot // 2):
            part = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            theta[i] *= 1 - part + part / STRETCH
        size = 1 + 0.1 * math.log(STRETCH)
    pos, num = st["pos"].cpu().numpy(), st["num"].cpu().numpy()
    out = {}
    for name in ("q", "k"):
        x = st[name].cpu().double().numpy()
        y = x.copy()
        for i in range(s):
            z = np.exp(1j * np.outer(pos[i] + np.arange(t), theta))[:, None] * size
            if case["layout"] == "half":
                w = (x[i, ..., :rot // 2] + 1j * x[i, ..., rot // 2:rot]) * z
                y[i, ..., :rot // 2], y[i, ..., rot // 2:rot] = w.real, w.imag
            else:
                w = (x[i, ..., 0:rot:2] + 1j * x[i, ..., 1:rot:2]) * z
                y[i, ..., 0:rot:2], y[i, ..., 1:rot:2] = w.real, w.imag
            y[i, num[i] if pos[i] >= 0 else 0:] = 0
        out[name] = torch.from_numpy(y)
    return out


def _exact_verify(case, st):
    s, k, n, temp = (case[x] for x in ("seqs", "drafts", "vocab", "temp"))
    token, u, num = (st[x].cpu().numpy() for x in ("token", "uniform", "num"))
    x = st["target"].cpu().numpy()
    d = st["draft"].cpu().numpy() if case["rows"] else None

    def dist(row):
        z = row.astype(np.float64) / temp
        e = np.exp(z - z.max())
        return e / e.sum()

    n_accept, out, logp = np.full(s, -1, np.int32), np.full((s, k + 1), -1, np.int32), np.zeros((s, k + 1))
    for i in range(s):
        if num[i] < 0:
            continue
        for a in range(num[i] + 1):
            p = dist(x[i, a])
            if a == num[i]:
                w = p
                break
            if d is not None:
                q = dist(d[i, a])
            else:
                q = np.zeros(n)
                q[token[i, a]] = 1.0
            if not float(u[i, a]) * q[token[i, a]] < p[token[i, a]]:
                w = np.maximum(p - q, 0)
                break
            out[i, a], logp[i, a] = token[i, a], math.log(p[token[i, a]])
        n_accept[i] = a
        c = np.cumsum(w)
        out[i, a] = min(int(np.searchsorted(c, float(u[i, k]) * c[-1], side="right")), n - 1)
        logp[i, a] = math.log(p[out[i, a]])
    return {"n_accept": torch.from_numpy(n_accept), "out": torch.from_numpy(out), "logp": torch.from_numpy(logp)}
