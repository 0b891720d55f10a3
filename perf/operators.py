"""Cases of the operators of a search over several continuations: attention over a cache held in 4 bits (and the storing
of new keys and values into it), the selection of a beam search over beams and vocabulary, and the reordering of the
beams' states. Shapes are those of the model driver's configurations (qwen35.py) and of common grouped-query heads.

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


def listed() -> list[dict]:
    return [
        # one token of the driver's own attention layer at the end of its default context: what a launch costs
        {"name": "decode 1x640 h16/4 d256", "kind": "attn", "seqs": 1, "tokens": 1, "heads": 16, "kv_heads": 4, "dim": 256,
         "len": 640, "window": 0, "ragged": False},
        # the same layer over a long cache: few rows, one long axis
        {"name": "decode 1x32768 h16/4 d256", "kind": "attn", "seqs": 1, "tokens": 1, "heads": 16, "kv_heads": 4,
         "dim": 256, "len": 32768, "window": 0, "ragged": False},
        # 32 sequences in lockstep, each at a position of its own, some of them not in use
        {"name": "lockstep 32x8192 h32/8 d128", "kind": "attn", "seqs": 32, "tokens": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "len": 8192, "window": 0, "ragged": True},
        # a chunk of a long prompt
        {"name": "prompt 512 at 7680 h16/4 d256", "kind": "attn", "seqs": 1, "tokens": 512, "heads": 16, "kv_heads": 4,
         "dim": 256, "len": 8192, "window": 0, "ragged": False},
        # a few drafted tokens of a few sequences, a sliding window, a head for every query head, odd sizes
        {"name": "draft 7x5 at 1503 h8/8 d64", "kind": "attn", "seqs": 7, "tokens": 5, "heads": 8, "kv_heads": 8, "dim": 64,
         "len": 1503, "window": 1000, "ragged": True},
        # the new keys and values of a lockstep step
        {"name": "store 32x1 h8 d128", "kind": "store", "seqs": 32, "tokens": 1, "heads": 8, "kv_heads": 8, "dim": 128,
         "len": 2048, "ragged": True},
        # those of a whole prompt
        {"name": "store 1x1983 h4 d256", "kind": "store", "seqs": 1, "tokens": 1983, "heads": 4, "kv_heads": 4, "dim": 256,
         "len": 2000, "ragged": False},
        # one prompt, a few beams
        {"name": "select 1x4 of 151936", "kind": "select", "groups": 1, "beams": 4, "vocab": 151936, "eos": False,
         "masked": False},
        # several prompts at once
        {"name": "select 8x8 of 151936", "kind": "select", "groups": 8, "beams": 8, "vocab": 151936, "eos": True,
         "masked": False},
        # many small searches with an odd vocabulary, part of it masked, some beams at their end
        {"name": "select 61x5 of 32003", "kind": "select", "groups": 61, "beams": 5, "vocab": 32003, "eos": True,
         "masked": True},
        # the states of a hybrid model's beams: DeltaNet rows, conv windows, short caches
        {"name": "reorder 1x4 hybrid at 640", "kind": "reorder", "groups": 1, "beams": 4, "rec_layers": 24, "rec_heads": 32,
         "attn_layers": 8, "kv_heads": 4, "dim": 256, "prompt": 512, "len": 640},
        # caches alone, several groups, behind a shared prompt
        {"name": "reorder 4x8 caches at 2000", "kind": "reorder", "groups": 4, "beams": 8, "rec_layers": 0, "rec_heads": 0,
         "attn_layers": 8, "kv_heads": 4, "dim": 256, "prompt": 301, "len": 2000},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number whose logarithm is spread evenly over lo..hi."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng) -> dict:
    kind = rng.choice(["attn", "attn", "attn", "store", "select", "select", "reorder"])
    if kind in ("attn", "store"):
        h, hk, dim = rng.choice(HEADS)
        seqs = _spread(rng, 1, 32)
        if kind == "store":
            tokens = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, 1983 // seqs))
            return {"kind": kind, "seqs": seqs, "tokens": tokens, "heads": h, "kv_heads": hk, "dim": dim,
                    "len": tokens + rng.randint(0, 500), "ragged": rng.random() < 0.5}
        n = _spread(rng, 1, min(32768, 32 * 8192 * 1024 // (seqs * hk * dim)))
        most = min(n, 512, 512 * 8192 * 4096 // (seqs * n * h * dim))
        tokens = 1 if most < 2 or rng.random() < 0.5 else _spread(rng, 2, most)
        return {"kind": kind, "seqs": seqs, "tokens": tokens, "heads": h, "kv_heads": hk, "dim": dim, "len": n,
                "window": _spread(rng, 1, n) if rng.random() < 0.3 else 0, "ragged": rng.random() < 0.5}
    if kind == "select":
        vocab = _spread(rng, 1000, 151936)
        beams = rng.randint(1, 32)
        return {"kind": kind, "groups": _spread(rng, 1, min(64, max(1, 64 * 151936 // (vocab * beams)))), "beams": beams,
                "vocab": vocab, "eos": rng.random() < 0.5, "masked": rng.random() < 0.3}
    beams = rng.randint(2, 32)
    _, hk, dim = rng.choice(HEADS)
    groups = rng.randint(1, max(1, 32 // beams))
    n = _spread(rng, 16, 64000 // (groups * beams))
    return {"kind": kind, "groups": groups, "beams": beams, "rec_layers": rng.randint(0, 48 // (groups * beams)),
            "rec_heads": rng.choice([2, 16, 32]), "attn_layers": rng.randint(1, 8), "kv_heads": hk, "dim": dim,
            "prompt": rng.randint(0, n - 1), "len": n}


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


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    normal = lambda *n: torch.randn(*n, generator=g, device=DEV)  # noqa: E731
    uniform = lambda *n: torch.rand(*n, generator=g, device=DEV)  # noqa: E731
    st = {"case": case}
    if case["kind"] in ("attn", "store"):
        s, t, h, hk, hd, n = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "len"))
        ctx = -(-n // 32) * 32
        gain = (0.3 * normal(2, hk, 1, hd)).exp()  # channels of unlike size
        kv = [_quantize(normal(s, hk, ctx, hd) * gain[i]) for i in range(2)]
        st["cache"] = _records(*kv[0], *kv[1]).contiguous()
        del kv
        st["ctx"] = ctx
        st["k"], st["v"] = (normal(s, t, hk, hd) * gain[i, :, 0] for i in range(2))
        # the tokens' first positions; ragged: sequences at places of their own, with fewer tokens, one of them not in use
        pos, num = torch.full((s,), n - t, device=DEV), torch.full((s,), t, device=DEV)
        if case["ragged"]:
            pos = ((n - t + 1) * uniform(s)).long().clamp(max=n - t)
            num = 1 + (t * uniform(s)).long().clamp(max=t - 1)
            if s > 2:
                pos[1], num[1] = -1, 0
        st["pos"], st["num"] = pos.int(), num.int()
        if case["kind"] == "attn":
            st["q"] = 1.5 * normal(s, t, h, hd)
            st["y"] = torch.zeros(s, t, h, hd, device=DEV)
        else:
            st["k_out"], st["v_out"] = torch.zeros_like(st["k"]), torch.zeros_like(st["v"])
        return st
    r = case["groups"] * case["beams"]
    if case["kind"] == "select":
        x = 2.5 * normal(r, case["vocab"])
        if case["masked"]:  # tokens that a grammar rules out, and one beam that has no way on
            x[uniform(r, case["vocab"]) < 0.4] = -math.inf
            x[r // 2] = -math.inf
        st["logits"] = x
        st["score"] = -20 * uniform(r)
        st["eos"] = 2 if case["eos"] else -1
        st["last"] = torch.where(uniform(r) < 0.2, 2, 5).int()
        return st
    lr, la, ch, row = case["rec_layers"], case["attn_layers"], 256 * case["rec_heads"], case["kv_heads"] * case["dim"]
    ctx = case["len"] + 64
    st["rec"], st["conv"] = normal(lr, r, case["rec_heads"] * 128 * 128), normal(lr, r, 3 * ch)
    st["kv"] = [normal(2, r, ctx, row).half() for _ in range(la)]
    st["ids"] = torch.randint(0, 151936, (r, ctx), generator=g, device=DEV, dtype=torch.int32)
    st["parent"] = (case["beams"] * uniform(case["groups"], case["beams"]) ** 2).int()  # the better beams have more heirs
    used = case["len"] - (0.2 * (case["len"] - case["prompt"]) * uniform(case["groups"], 1)).int()
    st["used"] = used.expand(-1, case["beams"]).reshape(-1).contiguous().int()  # positions so far, by group
    return st


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(st: dict):
    if own:
        return _own(st)
    return {"attn": _plain_attn, "store": _plain_store, "select": _plain_select, "reorder": _plain_reorder}[st["case"]["kind"]](st)


def _plain_attn(st):
    case = st["case"]
    s, t, h, hk, hd = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim"))
    k, v = _values(st["cache"], hd // 32)
    at = st["pos"].long()[:, None] + torch.arange(t, device=DEV)  # the tokens' positions
    live = (torch.arange(t, device=DEV) < st["num"][:, None]) & (st["pos"][:, None] >= 0)
    src = torch.arange(s, device=DEV)[:, None].expand(s, t)
    for new, old in ((st["k"], k), (st["v"], v)):
        q, d = _quantize(new)
        old[src[live], :, at[live]] = ((q.float() - 8) * d.float()[..., None]).flatten(-2)[live]
    g = h // hk
    q = st["q"].view(s, t, hk, g, hd).permute(0, 2, 1, 3, 4).reshape(s, hk, t * g, hd)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(hd)
    j = torch.arange(k.shape[2], device=DEV)
    seen = (j <= at[..., None]) & (j > at[..., None] - (case["window"] or 1 << 30)) & live[..., None]
    x.view(s, hk, t, g, -1).masked_fill_(~seen[:, None, :, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    y = torch.matmul(x, v) / x.sum(-1, keepdim=True).clamp(min=1e-30)
    return {"y": y.view(s, hk, t, g, hd).permute(0, 2, 1, 3, 4).reshape(s, t, h, hd)}


def _plain_store(st):
    case, out = st["case"], {}
    live = (torch.arange(case["tokens"], device=DEV) < st["num"][:, None]) & (st["pos"][:, None] >= 0)
    for name in ("k", "v"):  # what the cache then holds at the tokens' positions
        q, d = _quantize(st[name])
        out[name] = torch.where(live[..., None, None], ((q.float() - 8) * d.float()[..., None]).flatten(-2), 0)
    return out


def _plain_select(st):
    case = st["case"]
    g, b, n = case["groups"], case["beams"], case["vocab"]
    x = st["logits"].double()  # two beams' candidates may be next to each other
    top = x.amax(-1, keepdim=True)
    lse = top + torch.exp(x - top.clamp(min=-1e300)).sum(-1, keepdim=True).log()
    c = torch.where(top == -math.inf, -math.inf, x - lse) + st["score"].double()[:, None]
    over = (st["last"] == st["eos"])[:, None]
    at = torch.arange(n, device=DEV) == st["eos"]
    c = torch.where(over, torch.where(at, st["score"].double()[:, None], -math.inf), c).view(g, b * n)
    best, flat = torch.sort(c, dim=-1, descending=True, stable=True)
    best, flat = best[:, :b], flat[:, :b]
    return {"score": best.float(), "token": (flat % n).int(), "parent": (flat // n).int()}


def _plain_reorder(st):
    case = st["case"]
    g, b = case["groups"], case["beams"]
    rows = (st["parent"].long() + b * torch.arange(g, device=DEV)[:, None]).view(-1)
    st["rec"].copy_(st["rec"][:, rows])
    st["conv"].copy_(st["conv"][:, rows])
    j = torch.arange(st["ids"].shape[1], device=DEV)
    moved = (j >= case["prompt"]) & (j < st["used"][rows][:, None])
    for kv in st["kv"]:
        kv.copy_(torch.where(moved[..., None], kv[:, rows], kv))
    st["ids"].copy_(torch.where(moved, st["ids"][rows], st["ids"]))
    return {"rec": st["rec"], "conv": st["conv"], "kv": st["kv"], "ids": st["ids"]}


def _own(st):
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    import gemvq as gq
    case, stream = st["case"], torch.cuda.current_stream().cuda_stream
    p = lambda x: x.data_ptr()  # noqa: E731
    if case["kind"] in ("attn", "store"):
        s, t, h, hk, hd = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim"))
        if "handle" not in st:
            st["handle"] = gq.Kv4(p(st["cache"]), s, st["ctx"], hk, hd)
            st["work"] = torch.empty(gq.kv4_attn_work(st["handle"], t, h), dtype=torch.uint8, device=DEV)
        kv = st["handle"]
        gq.kv4_store_static(kv, p(st["k"]), p(st["v"]), hk * hd, t, p(st["pos"]), p(st["num"]), stream)
        if case["kind"] == "store":
            gq.kv4_load_static(kv, p(st["k_out"]), p(st["v_out"]), hk * hd, t, p(st["pos"]), p(st["num"]), stream)
            return {"k": st["k_out"], "v": st["v_out"]}
        gq.kv4_attn_static(kv, p(st["q"]), h * hd, hd, p(st["y"]), h * hd, t, h, p(st["pos"]), p(st["num"]), case["window"],
                           1 / math.sqrt(hd), p(st["work"]), st["work"].numel(), stream)
        return {"y": st["y"]}
    g, b = case["groups"], case["beams"]
    if case["kind"] == "select":
        n = case["vocab"]
        if "work" not in st:
            st["work"] = torch.empty(gq.beam_work(g, b, n), dtype=torch.uint8, device=DEV)
            st["out"] = {"score": torch.empty(g, b, device=DEV), "token": torch.empty(g, b, dtype=torch.int32, device=DEV),
                         "parent": torch.empty(g, b, dtype=torch.int32, device=DEV)}
        o = st["out"]
        gq.beam_select_static(p(st["logits"]), n, n, g, b, p(st["score"]), p(st["last"]), st["eos"], p(o["score"]), p(o["token"]),
                              p(o["parent"]), p(st["work"]), st["work"].numel(), stream)
        return o
    if "arrays" not in st:
        ar, ids, used = [], st["ids"], p(st["used"])
        for x in (st["rec"], st["conv"]):
            if x.numel():
                ar.append(gq.BeamArray(p(x), 4 * x.shape[2], 4 * x.shape[1] * x.shape[2], x.shape[0], 0, 1, 4 * x.shape[2]))
        for x in st["kv"]:
            row = 2 * x.shape[3]
            ar.append(gq.BeamArray(p(x), x.shape[2] * row, x.shape[1] * x.shape[2] * row, 2, case["prompt"], x.shape[2], row, 1,
                                   used, 1))
        ar.append(gq.BeamArray(p(ids), 4 * ids.shape[1], 0, 1, case["prompt"], ids.shape[1], 4, 1, used, 1))
        st["arrays"] = (gq.BeamArray * len(ar))(*ar)
    gq.beam_reorder_static(st["arrays"], p(st["parent"]), g, b, stream)
    return {"rec": st["rec"], "conv": st["conv"], "kv": st["kv"], "ids": st["ids"]}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case: dict) -> dict:
    if case["kind"] == "attn":
        s, t, h, hk, hd, n = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "len"))
        share = 0.5 if case["ragged"] else 1.0  # sequences at places of their own: half of the positions on average
        seen = n * share
        wide = min(seen, case["window"] + t) if case["window"] else seen  # positions that some token of a sequence sees
        each = min(seen, case["window"]) if case["window"] else max(1.0, seen - t / 2)
        rows = s * t * (0.5 if case["ragged"] and t > 1 else 1.0)
        return {"bytes": s * hk * hd * wide * 9 / 8 + 4 * rows * hd * (2 * h + 2 * hk), "flops": 4 * rows * h * hd * each}
    if case["kind"] == "store":
        n = case["seqs"] * case["tokens"] * (0.5 if case["ragged"] and case["tokens"] > 1 else 1.0) * case["kv_heads"] * case["dim"]
        return {"bytes": n * 2 * (4 + 9 / 16 + 9 / 16 + 4), "flops": 8 * n}  # stored, then read back
    if case["kind"] == "select":
        n = case["groups"] * case["beams"] * case["vocab"] * (0.8 if case["eos"] else 1.0)
        return {"bytes": 4 * n, "flops": 4 * n}
    r, ch = case["groups"] * case["beams"], 256 * case["rec_heads"]
    span = 0.9 * (case["len"] - case["prompt"])
    row = case["rec_layers"] * 4 * (case["rec_heads"] * 128 * 128 + 3 * ch) + span * (case["attn_layers"] * 4 * case["kv_heads"] * case["dim"] + 4)
    # most beams take another's row, and somewhat over half of the beams have an heir
    return {"bytes": 0.85 * r * row + 0.6 * r * row, "flops": 0}


# ---- the outputs in 64 bits -------------------------------------------------------------------------------------------
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "store": _exact_store, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](case, st)


def _blocks(x: torch.Tensor) -> torch.Tensor:
    """What Q4_0 holds of each row, in 64 bits; the choice of each value is made in FP32, as the format's is."""
    b = x.cpu().numpy().reshape(-1, 32)
    m = b[np.arange(len(b)), np.abs(b).argmax(1)]
    d = (m / np.float32(-8)).astype(np.float32)
    inv = np.divide(np.float32(1), d, out=np.zeros_like(d), where=d != 0)
    q = np.clip(np.trunc((b * inv[:, None]).astype(np.float32) + np.float32(8.5)), 0, 15).astype(np.float64) - 8
    return torch.from_numpy((q * d.astype(np.float16).astype(np.float64)[:, None]).reshape(x.shape)).to(DEV)


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
    s, t, h, hk, hd = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim"))
    kat, vat, shift, kd, vd = _where_in_record(hd)
    knew, vnew = _blocks(st["k"]), _blocks(st["v"])
    y = torch.zeros(s, t, h, hd, dtype=torch.float64, device=DEV)
    pos, num = st["pos"].tolist(), st["num"].tolist()
    for i in range(s):
        if pos[i] < 0 or num[i] == 0:
            continue
        m = pos[i] + num[i]
        at = pos[i] + torch.arange(num[i], device=DEV)
        j = torch.arange(m, device=DEV)
        seen = (j <= at[:, None]) & ((j > at[:, None] - case["window"]) if case["window"] else True)
        for kh in range(hk):
            rec = st["cache"][i, kh, : -(-m // 32)]
            sc = rec.view(torch.half)
            k = ((rec[:, kat] >> shift & 15).double() - 8) * sc[:, kd].double()
            v = ((rec[:, vat] >> shift & 15).double() - 8) * sc[:, vd].double()
            k, v = k.view(-1, hd)[:m], v.view(-1, hd)[:m]
            k[pos[i]:], v[pos[i]:] = knew[i, : num[i], kh], vnew[i, : num[i], kh]
            kt = k.t().contiguous()
            for qh in range(kh * h // hk, (kh + 1) * h // hk):
                x = (st["q"][i, : num[i], qh].double() @ kt) * hd ** -0.5
                y[i, : num[i], qh] = torch.softmax(torch.where(seen, x, -math.inf), -1) @ v
    return {"y": y}


def _exact_store(case, st):
    out = {}
    for name in ("k", "v"):
        x = _blocks(st[name])
        for i, (p, n) in enumerate(zip(st["pos"].tolist(), st["num"].tolist())):
            x[i, (n if p >= 0 else 0):] = 0
        out[name] = x
    return out


def _exact_select(case, st):
    b, n = case["beams"], case["vocab"]
    x, score = st["logits"].cpu().double().numpy(), st["score"].cpu().double().numpy()
    last = st["last"].cpu().numpy()
    out = {"score": [], "token": [], "parent": []}
    for g in range(case["groups"]):
        found = []  # each beam's own best, by value and then by index
        for i in range(b):
            r = g * b + i
            if last[r] == st["eos"]:
                found.append((score[r], i, st["eos"]))
                others = [k for k in range(b + 1) if k != st["eos"]][:b]
                found += [(-math.inf, i, k) for k in others]
                continue
            top = x[r].max()
            lp = np.full(n, -math.inf) if top == -math.inf else x[r] - top - math.log(np.exp(x[r] - top).sum())
            few = min(b, n)
            edge = np.partition(lp, n - few)[n - few]
            above = np.nonzero(lp > edge)[0]
            at = np.concatenate([above, np.nonzero(lp == edge)[0][: few - len(above)]])
            found += [(score[r] + lp[k], i, int(k)) for k in at]
        found.sort(key=lambda c: (-c[0], c[1], c[2]))
        for name, c in (("score", 0), ("parent", 1), ("token", 2)):
            out[name].append([f[c] for f in found[:b]])
    return {"score": torch.tensor(out["score"], dtype=torch.float64), "token": torch.tensor(out["token"], dtype=torch.int32),
            "parent": torch.tensor(out["parent"], dtype=torch.int32)}


def _exact_reorder(case, st):
    b = case["beams"]
    parent, used = st["parent"].view(-1).tolist(), st["used"].tolist()
    new = {k: st[k].clone() for k in ("rec", "conv", "ids")}
    kv = [x.clone() for x in st["kv"]]
    for r, par in enumerate(parent):
        src = r // b * b + par
        span = slice(case["prompt"], used[src])
        new["rec"][:, r], new["conv"][:, r] = st["rec"][:, src], st["conv"][:, src]
        new["ids"][r, span] = st["ids"][src, span]
        for to, x in zip(kv, st["kv"]):
            to[:, r, span] = x[:, src, span]
    return {"rec": new["rec"], "conv": new["conv"], "kv": kv, "ids": new["ids"]}
