"""Timed cases of the operators around a prompt: attention over packed prompts, norm and rotation of query and key heads, quantised
rows into the paged caches and back.

`run` computes them in elementary torch operations, or with `own` set through this package. Both take what `prepare` gives.
"""
import math

import torch

own = False

_BF, _F16, _F32 = torch.bfloat16, torch.float16, torch.float32
_DT = {"bf16": _BF, "f16": _F16}
_BLOCK = 128


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a short instruction to a small layer: latency is all there is
        dict(name="attention_prompt_17", op="attention", q_lens="17", k_lens="17", hq=8, hkv=2, dqk=64, dv=64, dtype="f16", lse=True),
        # one long prompt of a layer with grouped heads
        dict(name="attention_prompt_8192", op="attention", q_lens="8192", k_lens="8192", hq=32, hkv=8, dqk=128, dv=128, dtype="bf16",
             lse=False),
        # prompts short enough that the indexer would select all of their keys: dense, the latent rows expanded to 128 heads of 192 | 128
        dict(name="attention_latent_prompts", op="attention", q_lens="2047,1311,129,608", k_lens="2047,1311,129,608", hq=128, hkv=128,
             dqk=192, dv=128, dtype="bf16", lse=False),
        # a chunk of a long prompt behind what its earlier chunks left, and a shorter one of another sequence in the same step
        dict(name="attention_chunk_512_of_32k", op="attention", q_lens="512,77", k_lens="32768,5000", hq=64, hkv=8, dqk=128, dv=128,
             dtype="f16", lse=True),
        # a decode step: one token a sequence
        dict(name="attention_tokens_16", op="attention", q_lens=",".join(["1"] * 16),
             k_lens="16384,15999,12288,9001,8192,8191,6500,4097,4096,3000,2048,2047,1025,513,129,1", hq=64, hkv=8, dqk=128, dv=128,
             dtype="bf16", lse=False),
        # a decode step's heads, far positions, frequencies scaled for a context 40 times the trained one
        dict(name="norm_rope_64", op="norm_rope", t=64, hq=32, hkv=8, dq=128, dk=128, rotary=128, layout="half", last=False, norm=True,
             scaled=True, far=131072, dtype="bf16"),
        # a whole prompt's heads
        dict(name="norm_rope_16384", op="norm_rope", t=16384, hq=32, hkv=8, dq=128, dk=128, rotary=64, layout="half", last=False,
             norm=True, scaled=False, far=16384, dtype="f16"),
        # the latent path: the last 64 dims of 192-wide query heads and the one rope key, pairs side by side, written in halves
        dict(name="rope_latent_4097", op="norm_rope", t=4097, hq=128, hkv=1, dq=192, dk=64, rotary=64, layout="deinterleave", last=True,
             norm=False, scaled=True, far=65536, dtype="bf16"),
        # a decode step's rows into the split caches
        dict(name="cache_write_64", op="write", t=64, width=512, rope=True, packed=False, pages=512, dtype="bf16"),
        # a chunk's rows into the packed cache
        dict(name="cache_write_packed_8191", op="write", t=8191, width=512, rope=True, packed=True, pages=256, dtype="bf16"),
        # one short prefix back
        dict(name="cache_read_packed_129", op="read", lens="129", width=512, rope=True, packed=True, pages=64, dtype="bf16"),
        # the earlier context of four sequences back, for the attention of their next chunks
        dict(name="cache_read_4x24k", op="read", lens="32768,30001,24576,12345", width=512, rope=True, packed=False, pages=1024,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm_rope", "write", "read"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "attention":
        dqk, dv, hkv, g = rng.choice([(64, 64, rng.choice([1, 2, 8]), rng.choice([1, 4, 8])),
                                      (128, 128, rng.choice([1, 4, 8]), rng.choice([1, 3, 4, 8, 16])),
                                      (192, 128, rng.choice([16, 64]), 1)])
        b = _log(rng, 1, 24)
        kind = rng.choice(["prompts", "chunks", "tokens"])
        while True:
            longest = _log(rng, 1, 8192 if kind != "tokens" else 65536)
            kl = [max(1, int(longest * rng.uniform(0.05, 1.0))) for _ in range(b)]
            ql = list(kl) if kind == "prompts" else [1] * b if kind == "tokens" else [min(x, _log(rng, 1, 700)) for x in kl]
            # what the plain form lays out (score tiles of the longest sequence for all) and the work stay below the listed cases'
            if b * hkv * g * max(ql) * max(kl) <= 1 << 30 and sum(kl) * hkv * (dqk + dv) <= 1 << 30:
                break
        return dict(op=op, q_lens=",".join(map(str, ql)), k_lens=",".join(map(str, kl)), hq=hkv * g, hkv=hkv, dqk=dqk, dv=dv,
                    dtype=dtype, lse=rng.random() < 0.5)
    if op == "norm_rope":
        norm = rng.random() < 0.6
        d, rotary = rng.choice([(64, 64), (128, 128), (128, 64), (256, 128), (96, 32)])
        hq, hkv = rng.choice([(32, 8), (16, 2), (8, 8), (64, 4)])
        return dict(op=op, t=_log(rng, 1, 12000), hq=hq, hkv=hkv, dq=d, dk=d, rotary=rotary,
                    layout=rng.choice(["half", "interleaved", "deinterleave"]), last=rng.random() < 0.3, norm=norm,
                    scaled=rng.random() < 0.5, far=_log(rng, 512, 1 << 20), dtype=dtype)
    packed = rng.random() < 0.5
    width = 512 if packed else rng.choice([128, 512, 1024])
    rope = packed or width == 512
    if op == "write":
        return dict(op=op, t=_log(rng, 1, 16000), width=width, rope=rope, packed=packed, pages=256, dtype="bf16" if rope else dtype)
    b = _log(rng, 1, 32)
    longest = _log(rng, 1, 60000 // b)
    return dict(op=op, lens=",".join(str(max(1, int(longest * rng.uniform(0.1, 1.0)))) for _ in range(b)), width=width, rope=rope,
                packed=packed, pages=1024, dtype="bf16" if rope else dtype)


def _lens(text):
    return [int(x) for x in text.split(",")]


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _inv_freq(case):
    """Angles a position, in 64 bits: base^(-2i/r), the slow ones stretched 40 times where a case's context is longer than the trained
    one (a ramp between the dimensions that turn 32 times and once over 4096 positions), and the factor on cosine and sine."""
    r, base = case["rotary"], 10000.0
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if not case["scaled"]:
        return f, 1.0
    factor, trained = 40.0, 4096

    def dim_of(turns):
        return r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(dim_of(32.0)), 0), min(math.ceil(dim_of(1.0)), r - 1)
    ramp = ((torch.arange(r // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _rows(g, rows, width):
    """Rows as a norm leaves them, with the outlying dims and rows that a quantisation per group is for."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    x[:, ::97] *= 8
    x[::61] *= 20
    return x


def _quantised(x, groups):
    y = x.view(x.shape[0], groups, -1)
    top = y.abs().amax(-1, keepdim=True)
    return torch.round(y * (127 / top)).to(torch.int8).view(x.shape), (top / 127)[..., 0].contiguous()


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    s = {}
    if case["op"] == "attention":
        ql, kl = _lens(case["q_lens"]), _lens(case["k_lens"])
        tq, tk = sum(ql), sum(kl)
        s["q"] = torch.randn(tq, case["hq"], case["dqk"], generator=g, device="cuda", dtype=dt)
        if case["dqk"] == 192:  # the up-projection leaves a head's key and value dims side by side; the rope dims are all heads' own
            up = torch.randn(tk, case["hkv"], 256, generator=g, device="cuda", dtype=dt)
            rope = torch.randn(tk, 1, 64, generator=g, device="cuda", dtype=dt)
            s["k"] = torch.cat([up[..., :128], rope.expand(-1, case["hkv"], -1)], -1)
            s["v"] = up[..., 128:]
        else:
            s["k"] = torch.randn(tk, case["hkv"], case["dqk"], generator=g, device="cuda", dtype=dt)
            s["v"] = torch.randn(tk, case["hkv"], case["dv"], generator=g, device="cuda", dtype=dt)
        s["cu_q"] = torch.tensor(_cu(ql), dtype=torch.int32, device="cuda")
        s["cu_k"] = torch.tensor(_cu(kl), dtype=torch.int32, device="cuda")
    elif case["op"] == "norm_rope":
        t = case["t"]
        s["q"] = torch.randn(t, case["hq"], case["dq"], generator=g, device="cuda").mul_(1.7).to(dt)
        s["k"] = torch.randn(t, case["hkv"], case["dk"], generator=g, device="cuda").mul_(0.6).to(dt)
        start = torch.randint(0, max(1, case["far"] - t), (1,), generator=g, device="cuda")
        s["positions"] = start + torch.arange(t, device="cuda")
        if case["norm"]:
            s["wq"] = (1 + 0.2 * torch.randn(case["dq"], generator=g, device="cuda")).to(dt)
            s["wk"] = (1 + 0.2 * torch.randn(case["dk"], generator=g, device="cuda")).to(dt)
        f, amplitude = _inv_freq(case)
        s["inv_freq"], s["amplitude"] = f.cuda(), amplitude
    else:
        rows, w = case["pages"] * _BLOCK, case["width"]
        n, sc = _quantised(_rows(g, rows, w), w // 128)
        r = torch.randn(rows, 64, generator=g, device="cuda", dtype=_BF) if case["rope"] else None
        if case["packed"]:
            s["packed"] = torch.cat([n, r.view(torch.int8), sc.view(torch.int8)], 1)
        else:
            s["nope"], s["rope"], s["scales"] = n, r, sc
        if case["op"] == "write":
            s["x"] = _rows(g, case["t"], w).to(dt)
            s["xr"] = torch.randn(case["t"], 64, generator=g, device="cuda", dtype=_BF) if case["rope"] else None
            s["index"] = torch.randperm(rows, generator=g, device="cuda")[:case["t"]]
        else:
            lens = _lens(case["lens"])
            blocks = [-(-n // _BLOCK) for n in lens]
            free = torch.randperm(case["pages"], generator=g, device="cuda")
            table = torch.full((len(lens), max(blocks)), -1, dtype=torch.int32, device="cuda")
            at = 0
            for i, n in enumerate(blocks):
                table[i, :n] = free[at:at + n]
                at += n
            s["table"] = table
            s["cu"] = torch.tensor(_cu(lens), dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    dt = _DT[case["dtype"]]
    if case["op"] == "attention":
        ql = _lens(case["q_lens"])
        s["mq"], s["mk"] = max(ql), max(_lens(case["k_lens"]))
        s["out"] = torch.empty(sum(ql), case["hq"], case["dv"], dtype=dt, device="cuda")
        s["lse"] = torch.empty(case["hq"], sum(ql), dtype=_F32, device="cuda") if case["lse"] else None
    elif case["op"] == "norm_rope":
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        if own:
            import pypto_b200

            scaling = dict(type="yarn", factor=40.0, original_max_position=4096) if case["scaled"] else None
            s["rotary"] = pypto_b200.RotaryFrequencies(case["rotary"], 10000.0, scaling=scaling, device="cuda")
    elif case["op"] == "read":
        rows = sum(_lens(case["lens"]))
        s["out"] = torch.empty(rows, case["width"], dtype=dt, device="cuda")
        s["out_rope"] = torch.empty(rows, 64, dtype=_BF, device="cuda") if case["rope"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    return {"attention": _attention, "norm_rope": _norm_rope, "write": _write, "read": _read}[s["case"]["op"]](s)


def _attention(s):
    c = s["case"]
    scale = c["dqk"] ** -0.5
    if own:
        import pypto_b200

        pypto_b200.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["out"], scale, lse_out=s["lse"])
        return [s["out"], s["lse"]] if c["lse"] else s["out"]
    # all sequences padded to the longest
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    lq, lk = cu_q.diff()[:, None], cu_k.diff()[:, None]
    b, hkv, g = lq.shape[0], c["hkv"], c["hq"] // c["hkv"]
    iq, ik = torch.arange(s["mq"], device="cuda")[None], torch.arange(s["mk"], device="cuda")[None]
    at_q, at_k = (cu_q[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1), (cu_k[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    q = s["q"][at_q].float().view(b, s["mq"], hkv, g, -1).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * s["mq"], -1)
    k = s["k"][at_k].float().permute(0, 2, 3, 1)
    v = s["v"][at_k].float().permute(0, 2, 1, 3)
    x = torch.matmul(q, k).mul_(scale).view(b, hkv, g, s["mq"], s["mk"])
    seen = (ik < lk)[:, None] & (ik[:, None] <= (iq + lk - lq)[..., None])  # [b, mq, mk]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hkv, g * s["mq"], -1), v).view(b, hkv, g, s["mq"], -1) / total.clamp(min=1e-30)
    # back to packed rows
    row = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu_q[1:], row, right=True)
    pos = row - cu_q[seq]
    out = o.permute(0, 3, 1, 2, 4).reshape(b, s["mq"], c["hq"], -1)[seq, pos].to(s["q"].dtype)
    if not c["lse"]:
        return out
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(b, s["mq"], c["hq"])[seq, pos].t().contiguous()
    return [out, lse]


def _turned(x, w, cos, sin, c):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    r = c["rotary"]
    at = x.shape[-1] - r if c["last"] else 0
    z = y[..., at:at + r]
    a, b = (z[..., :r // 2], z[..., r // 2:]) if c["layout"] == "half" else (z[..., ::2], z[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    z = torch.stack([a, b], -1).flatten(-2) if c["layout"] == "interleaved" else torch.cat([a, b], -1)
    return torch.cat([y[..., :at], z, y[..., at + r:]], -1).to(x.dtype)


def _norm_rope(s):
    c = s["case"]
    if own:
        import pypto_b200

        pypto_b200.qk_norm_rope(s["q"], s["k"], s["positions"], s["rotary"], s["q_out"], s["k_out"], query_weight=s.get("wq"),
                                key_weight=s.get("wk"), eps=1e-6, layout=c["layout"], rope_last=c["last"])
        return [s["q_out"], s["k_out"]]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["amplitude"]).float()[:, None], (angle.sin() * s["amplitude"]).float()[:, None]
    return [_turned(s["q"], s.get("wq"), cos, sin, c), _turned(s["k"], s.get("wk"), cos, sin, c)]


def _write(s):
    c = s["case"]
    if own:
        import pypto_b200

        pypto_b200.kv_cache_write(s["x"], s["xr"], s["index"], s.get("nope"), s.get("rope"), s.get("scales"),
                                  packed_kv_cache=s.get("packed"))
    else:
        y = s["x"].float().view(c["t"], -1, 128)
        top = y.abs().amax(-1, keepdim=True)
        up = torch.div(torch.full_like(top, 127.0), top)
        n = torch.round(y * up).to(torch.int8).view(c["t"], -1)
        sc = up[..., 0].reciprocal()
        if c["packed"]:
            s["packed"][s["index"]] = torch.cat([n, s["xr"].view(torch.int8), sc.view(torch.int8)], 1)
        else:
            s["nope"][s["index"]] = n
            s["scales"][s["index"]] = sc
            if c["rope"]:
                s["rope"][s["index"]] = s["xr"]
    return [s["packed"]] if c["packed"] else [s["nope"], s["scales"], s["rope"]]


def _read(s):
    c = s["case"]
    if own:
        import pypto_b200

        pypto_b200.kv_cache_read(s.get("nope"), s.get("rope"), s.get("scales"), s["table"], s["cu"], s["out"], s["out_rope"], _BLOCK,
                                 packed_kv_cache=s.get("packed"))
        return [s["out"], s["out_rope"]]
    cu = s["cu"].long()
    row = torch.arange(s["out"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], row, right=True)
    pos = row - cu[seq]
    at = s["table"][seq, pos // _BLOCK].long() * _BLOCK + pos % _BLOCK
    if c["packed"]:
        rows = s["packed"][at]
        n, r, sc = rows[:, :512], rows[:, 512:640].contiguous().view(_BF), rows[:, 640:].contiguous().view(_F32)
    else:
        n, r, sc = s["nope"][at], s["rope"][at] if c["rope"] else None, s["scales"][at]
    return [(n.float().view(row.shape[0], -1, 128) * sc[..., None]).view(row.shape[0], -1).to(s["out"].dtype), r]


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        ql, kl = _lens(case["q_lens"]), _lens(case["k_lens"])
        hq, hkv, dqk, dv = case["hq"], case["hkv"], case["dqk"], case["dv"]
        pairs = sum(q * k - q * (q - 1) // 2 for q, k in zip(ql, kl))
        return {"bytes": 2 * sum(ql) * hq * (dqk + dv) + 2 * sum(kl) * hkv * (dqk + dv) + (4 * sum(ql) * hq if case["lse"] else 0),
                "flops": 2 * pairs * hq * (dqk + dv)}
    if case["op"] == "norm_rope":
        n = case["t"] * (case["hq"] * case["dq"] + case["hkv"] * case["dk"])
        turned = case["t"] * (case["hq"] + case["hkv"]) * case["rotary"]
        return {"bytes": 4 * n + 8 * case["t"], "flops": (4 * n if case["norm"] else 0) + 3 * turned}
    w, rope = case["width"], 64 if case["rope"] else 0
    row = w + 4 * (w // 128) + 2 * rope
    if case["op"] == "write":
        return {"bytes": case["t"] * (2 * w + 2 * rope + 8 + row), "flops": 3 * case["t"] * w}
    n = sum(_lens(case["lens"]))
    return {"bytes": n * (row + 2 * w + 2 * rope) + 4 * (n // _BLOCK), "flops": n * w}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "norm_rope":
        return [_exact_heads(case, s["q"].double(), s.get("wq"), s), _exact_heads(case, s["k"].double(), s.get("wk"), s)]
    if case["op"] == "write":
        if case["packed"]:
            return None  # bytes
        # a value halfway between two steps goes by the rounding of the scale: no 64-bit value of the whole numbers
        scales = s["scales"].double()
        for j in range(case["width"] // 128):
            scales[s["index"], j] = s["x"][:, 128 * j:128 * j + 128].double().abs().max(1).values / 127
        rope = None
        if case["rope"]:
            rope = s["rope"].double()
            rope[s["index"]] = s["xr"].double()
        return [None, scales, rope]
    rows, ropes, cu = [], [], _cu(_lens(case["lens"]))
    for i in range(len(cu) - 1):
        n = cu[i + 1] - cu[i]
        pages = s["table"][i].tolist()[:-(-n // _BLOCK)]
        at = torch.cat([torch.arange(p * _BLOCK, (p + 1) * _BLOCK, device="cuda") for p in pages])[:n]
        if case["packed"]:
            raw = s["packed"].index_select(0, at)
            sc = raw[:, 640:656].contiguous().view(_F32).double()
            ropes.append(raw[:, 512:640].contiguous().view(_BF).double())
            raw = raw[:, :512].double()
        else:
            raw, sc = s["nope"].index_select(0, at).double(), s["scales"].index_select(0, at).double()
            if case["rope"]:
                ropes.append(s["rope"].index_select(0, at).double())
        rows.append(raw * sc.repeat_interleave(128, 1))
    return [torch.cat(rows), torch.cat(ropes) if case["rope"] else None]


def _exact_attention(case, s):
    ql, kl = _lens(case["q_lens"]), _lens(case["k_lens"])
    cq, ck, g = _cu(ql), _cu(kl), case["hq"] // case["hkv"]
    out = torch.empty(sum(ql), case["hq"], case["dv"], dtype=torch.float64, device="cuda")
    lse = torch.empty(case["hq"], sum(ql), dtype=torch.float64, device="cuda")
    for i, (nq, nk) in enumerate(zip(ql, kl)):
        future = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1)
        for h in range(case["hq"]):
            q = s["q"][cq[i]:cq[i + 1], h].double() / math.sqrt(case["dqk"])
            x = q @ s["k"][ck[i]:ck[i + 1], h // g].double().T
            x[future] = -math.inf
            lse[h, cq[i]:cq[i + 1]] = torch.logsumexp(x, 1)
            out[cq[i]:cq[i + 1], h] = torch.softmax(x, 1) @ s["v"][ck[i]:ck[i + 1], h // g].double()
    return [out, lse] if case["lse"] else out


def _exact_heads(case, x, w, s):
    if w is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
    y, r = x.clone(), case["rotary"]
    at = x.shape[-1] - r if case["last"] else 0
    turn = torch.polar(torch.full((case["t"], r // 2), s["amplitude"], dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["inv_freq"]))[:, None]
    side = case["layout"] != "half"
    i = at + torch.arange(r // 2, device="cuda") * (2 if side else 1)
    j = i + (1 if side else r // 2)
    z = torch.complex(x[..., i], x[..., j]) * turn
    if case["layout"] == "deinterleave":
        i = at + torch.arange(r // 2, device="cuda")
        j = i + r // 2
    y[..., i], y[..., j] = z.real, z.imag
    return y
