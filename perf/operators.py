"""Rotary positions, filling a KV cache, and attention over a cache held in 4 bits, as cases that can be timed and checked.

A case is a dict of plain values.  ``kind`` names the operator it goes through:

  rope     ``torch.ops.fa_b200.rope``: rotary positions of q and k, with the gradients where ``train`` is true
  append   ``fa.cache_append``: the newest tokens' k and v into a KV cache (16-bit, e4m3 or 4-bit; dense or paged), with
           the rotation of q and k on the way.  Rows of a 4-bit cache come back as values through ``fa.cache_read_u4``
  read     ``fa.cache_read_u4``: rows of a 4-bit cache as 16-bit values
  attend   ``fa.decode_gqa_u4``: grouped-query attention of the newest token(s) over a 4-bit cache

``own`` chooses between the library's calls and the same formulas in elementary torch operations (32-bit arithmetic,
angles in 64, rounded once at the end).  ``exact`` is written from the definitions in 64 bits, apart from both.

The 4-bit cache: along the head dimension two codes share a byte (the even element in the low half), and every 64 elements
have an fp16 (scale, offset), value = offset + scale * code.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CACHE_ELEMS = 2.2e9      # most elements of K and V in a drawn 4-bit cache
ATTEND_STEPS = 2.7e11    # most floating-point operations of a drawn attention over several tokens
ROPE_ELEMS = 1.6e8       # most elements of q and k in a drawn rotation


def _library():
    from __graft_entry__ import load_module, load_package
    return load_package(), load_module("torch_op")


def listed():
    return [
        # Positions of one short prompt, half layout, small heads: the smallest rotation.
        dict(name="rope_f16_d64_b1h12s512", kind="rope", dtype="f16", b=1, hq=12, hkv=12, s=512, d=64, rot=64,
             interleaved=False, train=False, base=1e4, far=0),
        # A training step's rotation, forward and backward: grouped heads, neighbouring pairs, half of the head rotated.
        dict(name="rope_bf16_d128_b2hq32hkv8s4096_train", kind="rope", dtype="bf16", b=2, hq=32, hkv=8, s=4096, d=128,
             rot=64, interleaved=True, train=True, base=5e5, far=0),
        # One decode step of a batch fills a paged 16-bit cache (the smallest append).
        dict(name="append_bf16_paged_b16t1", kind="append", dtype="bf16", cache="bf16", b=16, hq=32, hkv=8, t=1, kv=4096,
             d=128, rot=128, interleaved=False, base=1e4, page=16, ragged=True, padded=False),
        # A chunk of a prompt into a dense 8-bit cache, q as codes for the attention that follows.
        dict(name="append_bf16_e4m3_b8t512", kind="append", dtype="bf16", cache="e4m3", b=8, hq=32, hkv=8, t=512, kv=4096,
             d=128, rot=128, interleaved=False, base=1e4, page=0, ragged=False, padded=False),
        # A decode step of a batch into a 4-bit cache.
        dict(name="append_f16_u4_b32t1", kind="append", dtype="f16", cache="u4", b=32, hq=32, hkv=8, t=1, kv=8192, d=128,
             rot=128, interleaved=True, base=1e4, page=0, ragged=True, padded=False),
        # A chunk of a left-padded batch of prompts into a paged 4-bit cache.
        dict(name="append_bf16_u4_paged_b8t512", kind="append", dtype="bf16", cache="u4", b=8, hq=32, hkv=8, t=512,
             kv=4096, d=128, rot=128, interleaved=False, base=5e5, page=16, ragged=True, padded=True),
        # A few hundred rows of one short sequence read back from an odd row on.
        dict(name="read_f16_u4_d64_b1n300", kind="read", dtype="f16", b=1, hkv=12, kv=1537, n=300, d=64, page=0,
             ragged=False),
        # Long prefixes read back from pages.
        dict(name="read_bf16_u4_paged_b4n16384", kind="read", dtype="bf16", b=4, hkv=8, kv=16384, n=16384, d=128, page=64,
             ragged=True),
        # Decode of two short sequences of odd length: the smallest attention, where latency counts.
        dict(name="attend_f16_u4_d64_b2kv1537", kind="attend", dtype="f16", b=2, hq=12, hkv=4, t=1, kv=1537, d=64, page=0,
             ragged=False),
        # A serving step: a batch of sequences of different lengths over pages.
        dict(name="attend_bf16_u4_paged_b16kv4096", kind="attend", dtype="bf16", b=16, hq=32, hkv=8, t=1, kv=4096, d=128,
             page=16, ragged=True),
        # A large batch over long sequences: the largest traffic.
        dict(name="attend_bf16_u4_b32kv16384", kind="attend", dtype="bf16", b=32, hq=32, hkv=8, t=1, kv=16384, d=128,
             page=0, ragged=False),
        # The next 512 tokens of prompts on 4-bit prefixes of 3584 keys: the largest contraction.
        dict(name="attend_f16_u4_b8kv4096t512", kind="attend", dtype="f16", b=8, hq=32, hkv=8, t=512, kv=4096, d=128,
             page=0, ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "read", "attend", "attend", "attend"])
    dtype, d = rng.choice(["f16", "bf16"]), rng.choice([64, 128])
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 3, 4, 5, 7, 8])
    rot, interleaved = rng.choice([d, d, d // 2, 16]), rng.random() < 0.5
    base = rng.choice([1e4, 5e5])
    if kind == "rope":
        b, s = _log(rng, 1, 8), _log(rng, 60, 8192)
        while b * s * (hkv * group + hkv) * d > ROPE_ELEMS:
            s = s * 3 // 4
        return dict(kind=kind, dtype=dtype, b=b, hq=hkv * group, hkv=hkv, s=s, d=d, rot=rot, interleaved=interleaved,
                    train=rng.random() < 0.5, base=base, far=rng.choice([0, 0, 1000, 1000003]))
    b, kv = _log(rng, 1, 48), _log(rng, 60, 32768)
    page = rng.choice([0, 16, 64])
    while 2.0 * b * hkv * kv * d > CACHE_ELEMS:
        kv = kv * 3 // 4
    if kind == "append":
        kv = min(kv, 8192)
        t = rng.choice([1, 1, 2, 4, _log(rng, 5, min(kv, 1024))])
        while 1.0 * b * t * hkv * (group + 2) * d > ROPE_ELEMS / 4:
            t = t * 3 // 4
        cache = rng.choice([dtype, "u4", "u4", "e4m3" if d == 128 else dtype])
        return dict(kind=kind, dtype=dtype, cache=cache, b=b, hq=hkv * group, hkv=hkv, t=t, kv=kv, d=d, rot=rot,
                    interleaved=interleaved, base=base, page=page, ragged=rng.random() < 0.6, padded=rng.random() < 0.3)
    if kind == "read":
        n = _log(rng, 1, kv)
        while 2.0 * b * hkv * n * d > ROPE_ELEMS:
            n = n * 3 // 4
        return dict(kind=kind, dtype=dtype, b=b, hkv=hkv, kv=kv, n=n, d=d, page=page, ragged=rng.random() < 0.6)
    t = rng.choice([1, 1, 1, 2, 4, 6, _log(rng, 8, 256)])
    t = min(t, kv)
    while t > 1 and 4.0 * b * hkv * group * t * kv * d > ATTEND_STEPS:
        t = max(1, t * 3 // 4)
    while t > 1 and 4.0 * b * hkv * group * t * kv > 2.2e9:
        t = max(1, t * 3 // 4)
    return dict(kind=kind, dtype=dtype, b=b, hq=hkv * group, hkv=hkv, t=t, kv=kv, d=d, page=page, ragged=rng.random() < 0.6)


# ------------------------------------------------------------------------------------------- inputs
def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _inv_freq(c):
    """Rotations of pair i in radians per position, as the paper on rotary positions has them: base ** (-2i / rot)."""
    return torch.tensor([c["base"] ** (-2.0 * i / c["rot"]) for i in range(c["rot"] // 2)], dtype=torch.float64)


def _codes(x):
    """The 4-bit form of 16-bit rows [..., D]: codes uint8 [..., D/2], (scale, offset) fp16 [..., D/64, 2]."""
    xg = x.float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, 64))
    z = xg.amin(-1).half()
    s = ((xg.amax(-1) - z.float()) * (1.0 / 15.0)).half()
    inv = torch.where(s > 0, 1.0 / s.float(), torch.zeros_like(s, dtype=torch.float32))
    c = ((xg - z.float().unsqueeze(-1)) * inv.unsqueeze(-1)).round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.stack((s, z), -1)


def _values(codes, params):
    """fp32 values of 4-bit rows."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, 64)).float()
    return (c * params[..., 0:1].float() + params[..., 1:2].float()).flatten(-2)


def prepare(case, seed):
    c, g = case, torch.Generator(device=DEV).manual_seed(seed)
    st = dict(case=c)
    if c["kind"] == "rope":
        t = TYPES[c["dtype"]]
        st.update(inv_freq=_inv_freq(c), q=_normal(g, t, c["b"], c["hq"], c["s"], c["d"]),
                  k=_normal(g, t, c["b"], c["hkv"], c["s"], c["d"]))
        # positions: those of a prompt's own rows, or of rows far into a long context, another start for each sequence
        st["positions"] = None
        if c["far"]:
            start = torch.randint(0, c["far"], (c["b"], 1), generator=g, device=DEV)
            st["positions"] = (start + torch.arange(c["s"], device=DEV)).to(torch.int32)
        if c["train"]:
            st["q"].requires_grad_(True)
            st["k"].requires_grad_(True)
            st["gq"], st["gk"] = _normal(g, t, *st["q"].shape), _normal(g, t, *st["k"].shape)
        return st
    _prepare_cache(st, c, g)
    t = TYPES[c["dtype"]]
    if c["kind"] == "append":
        # one projection's output: q, k and v of a token lie side by side
        width = (c["hq"] + 2 * c["hkv"]) * c["d"]
        st["qkv"] = _normal(g, t, c["b"], c["t"], width)
        st["inv_freq"] = _inv_freq(c)
        st["q_out"] = torch.empty((c["b"], c["t"], c["hq"], c["d"]), device=DEV,
                                  dtype=torch.float8_e4m3fn if c["cache"] == "e4m3" else t)
        st["new"] = None
        if c["padded"]:
            st["new"] = torch.randint(0, c["t"] + 1, (c["b"],), generator=g, device=DEV, dtype=torch.int32)
        if c["cache"] == "e4m3":
            for n in "qkv":
                st[n + "_scale"] = 0.008 + 0.004 * torch.rand((c["b"] * c["hkv"],), generator=g, device=DEV)
    if c["kind"] == "attend":
        st["q"] = _normal(g, t, c["b"], c["t"], c["hq"], c["d"])
        st["scale"] = 1.0 / math.sqrt(c["d"])
        st["o"] = torch.empty_like(st["q"])
        st["lse"] = torch.empty((c["b"], c["t"], c["hq"]), device=DEV, dtype=torch.float32)
    rows = {"append": c.get("t"), "read": c.get("n")}.get(c["kind"])
    if c["kind"] == "read" or c.get("cache") == "u4":            # the rows that are read back
        st["first"] = st["lens_all"] - rows if c["kind"] == "append" else torch.clamp(st["lens_all"] - rows, min=0) // 2
        st["first"] = st["first"].to(torch.int32)
        for n in "kv":
            st[n + "_rows"] = torch.empty((c["b"], rows, c["hkv"], c["d"]), device=DEV, dtype=t)
    return st


def _prepare_cache(st, c, g):
    """A cache of normal rows: 4-bit ones head-major [blocks, Hkv, rows, ...], the others [blocks, rows, Hkv, D]; a block is
    a page or a whole sequence."""
    b, hkv, kv, d, page = c["b"], c["hkv"], c["kv"], c["d"], c["page"]
    n_pages = -(-kv // page) if page else 1
    rows = page or kv
    blocks = b * n_pages
    kind = c.get("cache", "u4")
    for n in "kv":
        if kind == "u4":
            codes = torch.empty((blocks, hkv, rows, d // 2), device=DEV, dtype=torch.uint8)
            params = torch.empty((blocks, hkv, rows, d // 64, 2), device=DEV, dtype=torch.float16)
            step = max(1, (1 << 26) // (hkv * rows * d))
            for i in range(0, blocks, step):
                m = min(step, blocks - i)
                x = torch.randn((m, hkv, rows, d), generator=g, device=DEV, dtype=torch.float32)
                codes[i:i + m], params[i:i + m] = _codes(x.to(TYPES[c["dtype"]]))
            st[n + "_codes"], st[n + "_params"] = codes, params
        elif kind == "e4m3":
            x = torch.randn((blocks, rows, hkv, d), generator=g, device=DEV, dtype=torch.float32)
            st[n + "_cache"] = (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        else:
            st[n + "_cache"] = _normal(g, TYPES[kind], blocks, rows, hkv, d)
    st["lens"] = None
    if c["ragged"]:
        st["lens"] = torch.randint(min(kv, max(1, c.get("t", 1), kv // 16)), kv + 1, (b,), generator=g, device=DEV,
                                   dtype=torch.int32)
        st["lens"][0] = kv
    st["lens_all"] = torch.full((b,), kv, device=DEV, dtype=torch.int32) if st["lens"] is None else st["lens"]
    st["table"] = None
    if page:
        st["table"] = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32).view(b, n_pages)


# ------------------------------------------------------------------------------------------- one pass
def run(st):
    return {"rope": _rope, "append": _append, "read": _read, "attend": _attend}[st["case"]["kind"]](st)


def _rotate(x, cos, sin, rot, interleaved):
    """x [..., D] fp32 with cos, sin [..., rot/2]; the elements past `rot` stay."""
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    y1, y2 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _rope(st):
    c = st["case"]
    if own:
        op = _library()[1]
        q, k = op.rope(st["q"], st["k"], st["inv_freq"], st["positions"], c["interleaved"])
        if not c["train"]:
            return q, k
        return (q, k, *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"])))
    pos = torch.arange(c["s"], device=DEV)[None] if st["positions"] is None else st["positions"]
    ang = pos.double()[:, None, :, None] * st["inv_freq"].to(DEV)
    cos, sin = ang.cos().float(), ang.sin().float()
    t = TYPES[c["dtype"]]
    q, k = (_rotate(st[n].detach().float(), cos, sin, c["rot"], c["interleaved"]).to(t) for n in "qk")
    if not c["train"]:
        return q, k
    return (q, k, *(_rotate(st[n].float(), cos, -sin, c["rot"], c["interleaved"]).to(t) for n in ("gq", "gk")))


def _cache_args(st):
    """How the library is told where the cache's rows are."""
    c = st["case"]
    hkv, d, page = c["hkv"], c["d"], c["page"]
    rows = page or c["kv"]
    u4 = c.get("cache", "u4") == "u4"
    row, head, block = (d // 2, rows * d // 2, hkv * rows * d // 2) if u4 else (hkv * d, d, rows * hkv * d)
    kw = dict(kv_strides=(block, head, row), seq_lens=st["lens"])
    if u4:
        pairs = d // 64
        kw.update(param_strides=(hkv * rows * pairs, rows * pairs, pairs))
    if page:
        kw.update(block_table=st["table"], block_table_stride=st["table"].shape[1], page_size=page,
                  num_pages=st["table"].numel())
    return kw


def _read_back(st, fa, n):
    c = st["case"]
    fa.cache_read_u4(st["k_codes"], st["k_params"], st["v_codes"], st["v_params"], st["k_rows"], st["v_rows"], c["b"],
                     c["hkv"], c["kv"], c["d"], n, dtype=c["dtype"], first_rows=st["first"], **_cache_args(st),
                     stream=torch.cuda.current_stream())
    return st["k_rows"], st["v_rows"]


def _row_places(st, rows):
    """[B, N] row numbers within the sequences -> their places in the cache seen as one list of rows, clamped to valid ones."""
    page, kv = st["case"]["page"], st["case"]["kv"]
    r = rows.clamp(0, kv - 1).long()
    if not page:
        return torch.arange(r.shape[0], device=DEV)[:, None] * kv + r
    return st["table"].long().gather(1, r // page) * page + r % page


def _rows_u4(st, n, rows):
    """fp32 values [B, N, Hkv, D] of the given rows of a 4-bit cache; those that no sequence has are zero."""
    at = _row_places(st, rows)
    codes, params = st[n + "_codes"], st[n + "_params"]
    per = codes.shape[2]
    x = _values(codes[at // per, :, at % per], params[at // per, :, at % per])
    live = (rows >= 0) & (rows < st["lens_all"][:, None])
    return torch.where(live[:, :, None, None], x, torch.zeros_like(x))


def _read(st):
    c = st["case"]
    if own:
        return _read_back(st, _library()[0], c["n"])
    t = TYPES[c["dtype"]]
    rows = st["first"].long()[:, None] + torch.arange(c["n"], device=DEV)
    return tuple(_rows_u4(st, n, rows).to(t) for n in "kv")


def _append(st):
    c = st["case"]
    b, t, hq, hkv, d = c["b"], c["t"], c["hq"], c["hkv"], c["d"]
    dt = TYPES[c["dtype"]]
    x = st["qkv"]
    q, k, v = x[..., :hq * d], x[..., hq * d:(hq + hkv) * d], x[..., (hq + hkv) * d:]
    u4, e4m3 = c["cache"] == "u4", c["cache"] == "e4m3"
    caches = [st[n + ("_codes" if u4 else "_cache")] for n in "kv"]
    if own:
        fa = _library()[0]
        kw = _cache_args(st)
        if u4:
            kw.update(k_params=st["k_params"], v_params=st["v_params"])
        if e4m3:
            kw.update(q_scale=st["q_scale"], k_scale=st["k_scale"], v_scale=st["v_scale"])
        width = x.shape[-1]
        fa.cache_append(k, v, *caches, b, t, hkv, c["kv"], d, dtype=c["dtype"], cache_dtype=c["cache"], q=q,
                        q_out=st["q_out"], num_q_heads=hq, token_strides=(width, width, width), num_new=st["new"],
                        inv_freq=st["inv_freq"], rotary_dim=c["rot"], interleaved=c["interleaved"], **kw,
                        stream=torch.cuda.current_stream())
        if u4:
            return (st["q_out"], *_read_back(st, fa, t))
        return (st["q_out"], *caches)
    rows = st["lens_all"].long()[:, None] - t + torch.arange(t, device=DEV)            # [B, T]
    live = rows >= 0
    if st["new"] is not None:
        live &= torch.arange(t, device=DEV) >= t - st["new"].long()[:, None]
    ang = rows.double()[:, :, None, None] * st["inv_freq"].to(DEV)
    cos, sin = ang.cos().float(), ang.sin().float()
    q, k, v = q.unflatten(-1, (hq, d)), k.unflatten(-1, (hkv, d)), v.unflatten(-1, (hkv, d))
    q, k = (_rotate(y.float(), cos, sin, c["rot"], c["interleaved"]).to(dt) for y in (q, k))
    q = torch.where(live[:, :, None, None], q, torch.zeros_like(q))
    if e4m3:
        q, k, v = (_to_e4m3(y, st[n + "_scale"].view(b, 1, hkv, 1)) for n, y in (("q", q), ("k", k), ("v", v)))
    at = _row_places(st, rows)[live]
    for n, y, cache in (("k", k, caches[0]), ("v", v, caches[1])):
        if u4:
            codes, params = _codes(y[live])
            per = cache.shape[2]
            cache[at // per, :, at % per] = codes
            st[n + "_params"][at // per, :, at % per] = params
        elif e4m3:
            cache.view(torch.uint8).view(-1, hkv, d)[at] = y[live].view(torch.uint8)
        else:
            cache.view(-1, hkv, d)[at] = y[live]
    if u4:
        return (q, *(_rows_u4(st, n, rows).to(dt) for n in "kv"))
    return (q, *caches)


def _to_e4m3(y, scale):
    """16-bit [B, T, H, D] as e4m3 codes, scale [B, 1, Hkv, 1] of the head's group."""
    yg = y.float().unflatten(2, (scale.shape[2], -1))
    return (yg * (1.0 / scale).unsqueeze(-1)).clamp(-448, 448).flatten(2, 3).to(torch.float8_e4m3fn)


def _attend(st):
    c = st["case"]
    b, t, hq, hkv, kv, d = c["b"], c["t"], c["hq"], c["hkv"], c["kv"], c["d"]
    if own:
        fa = _library()[0]
        if "ws" not in st:                                       # a serving program keeps its workspace
            st["ws"] = torch.empty(fa.decode_gqa_u4_workspace_bytes(b, hq, hkv, t, kv, d), device=DEV, dtype=torch.uint8)
        fa.decode_gqa_u4(st["q"], st["k_codes"], st["k_params"], st["v_codes"], st["v_params"], st["o"], st["lse"], b, hq,
                         hkv, kv, d, st["scale"], dtype=c["dtype"], num_q_tokens=t, workspace=st["ws"],
                         workspace_bytes=st["ws"].numel(), **_cache_args(st), stream=torch.cuda.current_stream())
        return st["o"], st["lse"]
    k, v = (_dense_u4(st, n) for n in "kv")                      # [B, Hkv, rows, D]
    q = st["q"].float().unflatten(2, (hkv, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    s = q @ k.transpose(-1, -2) * st["scale"]                    # [B, Hkv, T * group, rows]
    last = st["lens_all"].long()[:, None] - t + torch.arange(t, device=DEV)            # last key that token sees
    last = last.repeat_interleave(hq // hkv, 1)[:, None, :, None]
    s = s.masked_fill(torch.arange(s.shape[-1], device=DEV) > last, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    l = p.sum(-1, keepdim=True)
    o = p @ v / torch.where(l > 0, l, torch.ones_like(l))
    lse = m + torch.log(l)
    o, lse = (y.unflatten(2, (t, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3) for y in (o, lse))
    return o.to(TYPES[c["dtype"]]), lse[..., 0]


def _dense_u4(st, n):
    codes, params = st[n + "_codes"], st[n + "_params"]
    if st["table"] is not None:
        codes = codes[st["table"].long()].transpose(1, 2).flatten(2, 3)
        params = params[st["table"].long()].transpose(1, 2).flatten(2, 3)
    return _values(codes, params)


# ------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    d = c["d"]
    row4 = d / 2 + d / 64 * 4                                    # bytes of a 4-bit row
    if c["kind"] == "rope":
        n = c["b"] * c["s"] * (c["hq"] + c["hkv"]) * d
        return {"bytes": (8.0 if c["train"] else 4.0) * n, "flops": (6.0 if c["train"] else 3.0) * n * c["rot"] / d}
    if c["kind"] == "append":
        fresh = c["b"] * c["t"] * (0.5 if c["padded"] else 1.0)  # mean number of tokens that are appended
        q, kv = c["hq"] * d, 2 * c["hkv"] * d
        out = {"u4": 2 * c["hkv"] * row4, "e4m3": kv}.get(c["cache"], 2 * kv)
        back = c["b"] * c["t"] * (2 * c["hkv"] * row4 + 2 * kv) if c["cache"] == "u4" else 0.0
        q_out = c["b"] * c["t"] * q * (1 if c["cache"] == "e4m3" else 2)
        return {"bytes": fresh * (2 * q + 2 * kv + out) + q_out + back, "flops": fresh * 3.0 * (q + kv / 2)}
    if c["kind"] == "read":
        return {"bytes": c["b"] * c["n"] * 2 * c["hkv"] * (row4 + 2 * d), "flops": c["b"] * c["n"] * 4.0 * c["hkv"] * d}
    lo = min(c["kv"], max(1, c["t"], c["kv"] // 16))
    mean = (c["kv"] + (c["b"] - 1) * (lo + c["kv"]) / 2) / c["b"] if c["ragged"] else c["kv"]
    return {"bytes": c["b"] * (mean * 2 * c["hkv"] * row4 + c["t"] * c["hq"] * (4 * d + 4)),
            "flops": 4.0 * c["b"] * c["hq"] * c["t"] * max(1.0, mean - (c["t"] - 1) / 2) * d}


# ------------------------------------------------------------------------------------------- 64 bits
def _angles64(pos, inv_freq):
    a = pos.to(torch.float64).unsqueeze(-1) * inv_freq.to(pos.device)
    return torch.polar(torch.ones_like(a), a)


def _turn64(x, turn, interleaved):
    """x [..., D] in 64 bits, pairs as complex numbers times `turn` [..., rot/2]."""
    half = turn.shape[-1]
    x = x.double()
    y = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * turn
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    return y


def _four_bits64(x):
    """What 4 bits keep of 16-bit rows [..., D]."""
    g = x.double().reshape(*x.shape[:-1], -1, 64)
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    z = lo.to(torch.float16).double()
    s = ((hi - z) / 15).to(torch.float16).double()
    code = torch.where(s > 0, torch.round((g - z) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(g))
    return (z + s * code.clamp(0, 15)).reshape(x.shape)


def _unpacked64(st, n, b):
    """Values [rows, Hkv, D] in 64 bits of the whole of sequence b in a 4-bit cache."""
    where = [b] if st["table"] is None else st["table"][b].tolist()
    codes, params = st[n + "_codes"][where].to(torch.int32), st[n + "_params"][where].double()
    c = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), device=DEV, dtype=torch.float64)
    c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
    c = c.reshape(*c.shape[:-1], -1, 64) * params[..., :1] + params[..., 1:]
    return c.flatten(-2).transpose(1, 2).flatten(0, 1)


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] == "rope":
        pos = torch.arange(c["s"], device=DEV)[None] if st["positions"] is None else st["positions"]
        turn = _angles64(pos, st["inv_freq"])[:, None]
        out = [_turn64(st[n].detach(), turn, c["interleaved"]) for n in "qk"]
        if c["train"]:                                           # the rotation's transpose turns back
            out += [_turn64(st[n], turn.conj(), c["interleaved"]) for n in ("gq", "gk")]
        return tuple(out)
    lens = st["lens_all"].tolist()
    if c["kind"] == "read":
        out = []
        for n in "kv":
            x = torch.zeros((c["b"], c["n"], c["hkv"], c["d"]), device=DEV, dtype=torch.float64)
            for b, first in enumerate(st["first"].tolist()):
                lo, hi = max(0, first), min(lens[b], first + c["n"])
                if hi > lo:
                    x[b, lo - first:hi - first] = _unpacked64(st, n, b)[lo:hi]
            out.append(x)
        return tuple(out)
    if c["kind"] == "append":
        return _append64(c, st, lens)
    group, out, lse = c["hq"] // c["hkv"], [], []
    for b in range(c["b"]):
        k, v = (_unpacked64(st, n, b)[:lens[b]] for n in "kv")
        q = st["q"][b].double().reshape(c["t"], c["hkv"], group, c["d"])
        s = torch.einsum("thgd,jhd->thgj", q, k) * st["scale"]
        first_hidden = (lens[b] - c["t"] + torch.arange(c["t"], device=DEV) + 1)[:, None, None, None]
        s = torch.where(torch.arange(lens[b], device=DEV) < first_hidden, s, torch.full_like(s, -math.inf))
        l = torch.logsumexp(s, -1)
        p = torch.exp(s - torch.where(torch.isfinite(l), l, torch.zeros_like(l))[..., None])
        out.append(torch.einsum("thgj,jhd->thgd", p, v).reshape(c["t"], c["hq"], c["d"]))
        lse.append(l.reshape(c["t"], c["hq"]))
    return torch.stack(out), torch.stack(lse)


def _append64(c, st, lens):
    b, t, hq, hkv, d = c["b"], c["t"], c["hq"], c["hkv"], c["d"]
    x = st["qkv"].reshape(b, t, hq + 2 * hkv, d)
    rows = torch.tensor([[n - t + i for i in range(t)] for n in lens], device=DEV)
    turn = _angles64(rows, st["inv_freq"])[:, :, None]
    q, k, v = _turn64(x[:, :, :hq], turn, c["interleaved"]), _turn64(x[:, :, hq:hq + hkv], turn, c["interleaved"]), x[:, :, hq + hkv:]
    new = [t] * b if st["new"] is None else st["new"].tolist()
    caches = []
    for n, y in (("k", k), ("v", v)):
        if c["cache"] == "u4":                                   # the rows come back, the appended ones among them
            whole = torch.zeros((b, t, hkv, d), device=DEV, dtype=torch.float64)
            fresh = _four_bits64(y.to(TYPES[c["dtype"]]))
            for i in range(b):
                lo = max(0, t - lens[i])                         # first token that has a row
                old = _unpacked64(st, n, i)
                whole[i, lo:] = old[lens[i] - t + lo:lens[i]]
                lo = max(lo, t - new[i])
                whole[i, lo:] = fresh[i, lo:]
            caches.append(whole)
            continue
        cache = st[n + "_cache"].double()
        if c["cache"] == "e4m3":
            y = (y.double() / st[n + "_scale"].double().reshape(b, 1, hkv, 1)).clamp(-448, 448)
        for i in range(b):
            lo = max(0, t - lens[i], t - new[i])
            if lo < t:
                r = rows[i, lo:]
                if c["page"]:
                    cache[st["table"][i].long()[r // c["page"]], r % c["page"]] = y[i, lo:].double()
                else:
                    cache[i, r] = y[i, lo:].double()
        caches.append(cache)
    if c["cache"] == "e4m3":
        q = (q / st["q_scale"].double().reshape(b, 1, hkv, 1).repeat_interleave(hq // hkv, 2)).clamp(-448, 448)
    for i in range(b):
        q[i, :max(0, t - lens[i], t - new[i])] = 0
    return (q, *caches)
