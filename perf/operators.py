"""What is measured of the operators around a layer's projections: rotary positions in their layouts, the norm of every
query and key head with the rotation in the same pass, the same for rows on their way into the paged cache, positions
and cache slots from request lengths, and a mixture-of-experts layer for a few tokens.

``listed()`` and ``draw(rng)`` give cases, ``prepare`` makes what a caller holds before the call, ``run`` makes one pass:
in the operators' plain form in 32 bits (``own`` false) or through the framework (``own`` true).  ``exact`` states the
results from the definitions in 64 bits and ``work`` the bytes and operations that a pass cannot do without.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ----------------------------------------------------------------------------- cases
def listed():
    yarn = {"scaling": "yarn", "factor": 4.0, "original": 32768}
    return [
        # one short prompt through a small model whose heads are rotated in part: latency decides
        dict(name="rotary_short", op="rotary", T=37, nq=14, nkv=2, D=64, R=32, interleaved=False, dtype="fp16",
             theta=1e4, max_pos=4096, scaling="none", factor=1.0, original=4096),
        # a training micro-batch with adjacent pairs on half of each head, positions far out under a stretched context
        dict(name="rotary_long", op="rotary", T=16384, nq=32, nkv=8, D=128, R=64, interleaved=True, dtype="bf16",
             theta=1e6, max_pos=131072, **yarn),
        # the smallest training batch of a model with head norms, ragged
        dict(name="norm_short", op="norm", T=301, nq=2, nkv=1, D=128, R=128, interleaved=False, dtype="bf16", theta=1e4,
             max_pos=4096, scaling="none", factor=1.0, original=4096),
        # an ordinary micro-batch of the 32 / 4 head mixture-of-experts model, forward and backward
        dict(name="norm_train", op="norm", T=4097, nq=32, nkv=4, D=128, R=128, interleaved=False, dtype="bf16", theta=1e6,
             max_pos=32768, scaling="none", factor=1.0, original=32768),
        # a full micro-batch of the same model
        dict(name="norm_long", op="norm", T=16384, nq=32, nkv=4, D=128, R=128, interleaved=False, dtype="bf16", theta=1e6,
             max_pos=131072, **yarn),
        # one decode step of 64 sequences: split projection sums become heads and cache rows
        dict(name="cache_decode", op="cache", T=64, parts=4, nq=32, nkv=4, D=128, R=128, interleaved=False, dtype="bf16",
             theta=1e6, max_pos=32768, scaling="none", factor=1.0, original=32768, block=32, hole=0.1, normed=True),
        # prompts of a prefill batch: rows to heads and cache rows
        dict(name="cache_prefill", op="cache", T=8191, parts=0, nq=32, nkv=4, D=128, R=128, interleaved=False,
             dtype="bf16", theta=1e6, max_pos=32768, scaling="none", factor=1.0, original=32768, block=32, hole=0.0,
             normed=True),
        # three requests arrive: positions and slots of their prompts
        dict(name="layout_few", op="layout", B=3, longest=700, block=32, cached=0.3),
        # a full rollout batch whose prompts share cached prefixes
        dict(name="layout_batch", op="layout", B=512, longest=4000, block=32, cached=0.6),
        # experts of one token, of a small batch and of a decode batch; sizes of the 128-expert model
        dict(name="moe_one", op="moe", T=1, E=128, k=8, H=2048, F=768, norm=True, dead=0.0),
        dict(name="moe_small", op="moe", T=9, E=128, k=8, H=2048, F=768, norm=True, dead=0.0),
        dict(name="moe_batch", op="moe", T=64, E=128, k=8, H=2048, F=768, norm=True, dead=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "cache", "layout", "moe"])
    if op == "layout":
        return dict(op=op, B=_log_int(rng, 1, 512), longest=_log_int(rng, 1, 4000), block=rng.choice([8, 16, 32, 64]),
                    cached=rng.choice([0.0, 0.3, 0.8]))
    if op == "moe":
        T = _log_int(rng, 1, 64)
        if rng.random() < 0.5:
            E, k, H, F = 128, 8, 2048, 768
        else:
            E = rng.randint(4, 200)
            k = rng.randint(1, min(8, E))
            H, F = 8 * rng.randint(8, 256), 8 * rng.randint(4, 96)
        return dict(op=op, T=T, E=E, k=k, H=H, F=F, norm=rng.random() < 0.7, dead=rng.choice([0.0, 0.0, 0.3]))
    D = rng.choice([64, 80, 96, 128, 128, 192, 256])
    nkv = rng.randint(1, 8)
    nq = nkv * rng.randint(1, 8 if op != "rotary" else 6)
    R = rng.choice([D, D, D // 2, D // 4])
    scaling = rng.choice(["none", "linear", "llama3", "yarn"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    # rows of at most 160 MB, so that no drawn case outgrows the largest listed one
    most = min(16384 if op != "cache" else 8192, int(160e6 / ((nq + 2 * nkv) * D * (4 if dtype == "fp32" else 2))))
    c = dict(op=op, T=_log_int(rng, 1, most), nq=nq, nkv=nkv, D=D, R=R, interleaved=rng.random() < 0.4, dtype=dtype,
             theta=rng.choice([1e4, 5e5, 1e6]), max_pos=rng.choice([4096, 32768, 131072]), scaling=scaling,
             factor=rng.choice([2.0, 4.0, 8.0]), original=rng.choice([2048, 8192, 32768]))
    if op == "cache":
        parts = rng.choice([0, 0, 1, 3, 8])
        if parts:  # sums of a split projection belong to decode batches and come out in bf16
            c.update(T=min(c["T"], 512), dtype="bf16")
        c.update(parts=parts, block=rng.choice([16, 32, 64]), hole=rng.choice([0.0, 0.2]), normed=rng.random() < 0.6)
    return c


# ----------------------------------------------------------------------------- inputs
_EPS = 1e-6


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _scaling_dict(case):
    kind = case["scaling"]
    if kind == "none":
        return None
    d = {"rope_type": kind, "factor": case["factor"]}
    if kind in ("llama3", "yarn"):
        d["original_max_position_embeddings"] = case["original"]
    if kind == "llama3":
        d.update(low_freq_factor=1.0, high_freq_factor=4.0)
    return d


def _table(case):
    """``[max_pos, R]``: cosines, then sines, of every position's angles (64-bit angles, stored in 32)."""
    if own:
        from skyrl_b200.ops import elementwise

        return elementwise.build_rope_table(case["max_pos"], case["R"], case["theta"], "cuda",
                                            scaling=_scaling_dict(case))
    R, f = case["R"], case["factor"]
    e = torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R
    inv, gain = case["theta"] ** -e, 1.0
    if case["scaling"] == "linear":
        inv = inv / f
    elif case["scaling"] == "llama3":
        wave = 2 * math.pi / inv
        s = ((case["original"] / wave - 1.0) / 3.0).clamp(0.0, 1.0)
        inv = s * inv + (1 - s) * inv / f
    elif case["scaling"] == "yarn":
        def turn(n):
            return R * math.log(case["original"] / (n * 2 * math.pi)) / (2 * math.log(case["theta"]))

        lo, hi = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), R - 1)
        ramp = ((torch.arange(R // 2, dtype=torch.float64, device="cuda") - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = ramp * inv / f + (1 - ramp) * inv
        gain = 0.1 * math.log(f) + 1.0
    ang = torch.arange(case["max_pos"], dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return (torch.cat([ang.cos(), ang.sin()], dim=-1) * gain).float()


def _packed_positions(T, max_pos, g):
    """Positions of packed sequences: runs that start anywhere below ``max_pos`` and count up."""
    at = torch.arange(T, device="cuda")
    start = torch.randint(0, max(1, max_pos - 600), (T // 512 + 1,), generator=g, device="cuda")
    return ((start[at // 512] + at % 512) % max_pos).to(torch.int32)


def _rows(case, seed):
    """Inputs of the three operators on packed rows (everything but the table)."""
    g = _gen(seed)
    T, D = case["T"], case["D"]
    W = (case["nq"] + 2 * case["nkv"]) * D
    dt = _DTYPES[case["dtype"]]
    st = {"case": case, "pos": _packed_positions(T, case["max_pos"], g)}
    # heads of a projection differ in size, and a few channels stand out
    gain = torch.exp(0.7 * torch.randn(W, generator=g, device="cuda"))
    if case.get("parts"):
        st["x"] = torch.randn(case["parts"], T, W, generator=g, device="cuda") * (gain / math.sqrt(case["parts"]))
    else:
        st["x"] = (torch.randn(T, W, generator=g, device="cuda") * gain).to(dt)
    if case["op"] == "norm" or case.get("normed"):
        st["qw"] = (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dt)
        st["kw"] = (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dt)
    if case["op"] != "cache":
        st["dy"] = (torch.randn(T, W, generator=g, device="cuda") * 0.02).to(dt)
        return st
    bs = case["block"]
    blocks = T // bs + 3
    order = torch.randperm(blocks, generator=g, device="cuda")
    at = torch.arange(T, device="cuda")
    slots = order[at // bs] * bs + at % bs
    empty = torch.rand(T, generator=g, device="cuda") < case["hole"]
    st["slots"] = torch.where(empty, torch.full_like(slots, -1), slots).to(torch.int32)
    st["k_cache"] = torch.zeros(blocks, bs, case["nkv"], D, device="cuda", dtype=dt)
    st["v_cache"] = torch.zeros_like(st["k_cache"])
    return st


def _layout_lengths(case):
    """Length and cached start of every request: spread over the range, some empty, the longest among them.  They go by
    the case, so that the number of rows does too; which request has which goes by the seed."""
    B, bs, out = case["B"], case["block"], []
    for i in range(B):
        n = int(case["longest"] * ((i * 0.6180339887498949) % 1.0) + 0.5) if i else case["longest"]
        hit = (i * 0.7548776662466927) % 1.0 < case["cached"]
        out.append((n, int(n * ((i * 0.5698402909980532) % 1.0)) // bs * bs if hit else 0))
    return out


def _layout_inputs(case, seed):
    g = _gen(seed)
    B, bs = case["B"], case["block"]
    pairs = torch.tensor(_layout_lengths(case), dtype=torch.int32, device="cuda")
    pairs = pairs[torch.randperm(B, generator=g, device="cuda")]
    width = case["longest"] // bs + 1
    tables = torch.randperm(B * width + 7, generator=g, device="cuda")[: B * width].view(B, width)
    # the caller knows the lengths on the host, and with them the number of rows; a few rows stay over as padding
    total = sum(n - c for n, c in _layout_lengths(case)) + 5
    return {"case": case, "tables": tables.to(torch.int32), "lens": pairs[:, 0].contiguous(),
            "starts": pairs[:, 1].contiguous(), "total": total}


def _moe_inputs(case, seed):
    g = _gen(seed)
    T, E, H, F = case["T"], case["E"], case["H"], case["F"]
    bf = torch.bfloat16

    def weights(*shape):
        w = torch.empty(*shape, device="cuda", dtype=bf)
        return w.normal_(0.0, 0.02, generator=g)

    st = {"case": case, "h": torch.randn(T, H, generator=g, device="cuda").to(bf),
          "router": (torch.randn(E, H, generator=g, device="cuda") * (1.5 / math.sqrt(H))).to(bf),
          "wgu": weights(E, 2 * F, H), "wd": weights(E, H, F), "live": None}
    if case["dead"] > 0:  # rows of a decode batch whose sequence has ended
        st["live"] = (torch.rand(T, generator=g, device="cuda") >= case["dead"]).to(torch.int32)
    return st


def prepare(case, seed):
    if case["op"] == "layout":
        return _layout_inputs(case, seed)
    if case["op"] == "moe":
        return _moe_inputs(case, seed)
    st = _rows(case, seed)
    st["table"] = _table(case)
    return st


# ----------------------------------------------------------------------------- one pass
def _angles(st):
    c = st["case"]
    cs = st["table"][st["pos"].long()]
    return cs[:, None, : c["R"] // 2], cs[:, None, c["R"] // 2 :]


def _pairs(x, c):
    """The two members of every rotated pair, and what is left of the head."""
    R = c["R"]
    if c["interleaved"]:
        return x[..., 0:R:2], x[..., 1:R:2], x[..., R:]
    return x[..., : R // 2], x[..., R // 2 : R], x[..., R:]


def _join(a, b, rest, c):
    rot = torch.stack([a, b], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([a, b], dim=-1)
    return torch.cat([rot, rest], dim=-1)


def _turn(x, cos, sin, c):
    a, b, rest = _pairs(x, c)
    return _join(a * cos - b * sin, b * cos + a * sin, rest, c)


def _heads(x, c):
    x = x.float().view(x.shape[0], c["nq"] + 2 * c["nkv"], c["D"])
    return x[:, : c["nq"]], x[:, c["nq"] : c["nq"] + c["nkv"]], x[:, c["nq"] + c["nkv"] :]


def _plain_rows(st):
    """Forward and backward of the rotation, with the head norms where the case has them."""
    c = st["case"]
    cos, sin = _angles(st)
    q, k, v = _heads(st["x"], c)
    dq, dk, dv = _heads(st["dy"], c)
    y, dx, dws = [], [], []
    for x, d, w in ((q, dq, st.get("qw")), (k, dk, st.get("kw"))):
        d = _turn(d, cos, -sin, c)  # the transposed rotation
        if w is None:
            y.append(_turn(x, cos, sin, c))
            dx.append(d)
            continue
        w = w.float()
        r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + _EPS)
        xh = x * r
        y.append(_turn(xh * w, cos, sin, c))
        dws.append((d * xh).sum((0, 1)))
        g = d * w
        dx.append(r * (g - xh * (g * xh).mean(-1, keepdim=True)))
    dt = st["x"].dtype
    out = [torch.cat([*y, v], dim=1).flatten(1).to(dt), torch.cat([*dx, dv], dim=1).flatten(1).to(dt)]
    return out + [w.to(dt) for w in dws]


def _plain_cache(st):
    c = st["case"]
    cos, sin = _angles(st)
    x, dt = st["x"], _DTYPES[c["dtype"]]
    if x.dim() == 3:
        x = x.sum(0).to(dt)  # the projection's own output type
    q, k, v = _heads(x, c)
    y = []
    for h, w in ((q, st.get("qw")), (k, st.get("kw"))):
        if w is not None:
            h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + _EPS) * w.float()
        y.append(_turn(h, cos, sin, c).to(dt))
    v = v.to(dt)
    keep = st["slots"] >= 0
    # a row without a slot is written to a spare row behind the cache
    for cache, rows in ((st["k_cache"], y[1]), (st["v_cache"], v)):
        flat = cache.view(-1, c["nkv"], c["D"])
        slot = torch.where(keep, st["slots"], torch.zeros_like(st["slots"])).long()
        wide = torch.cat([flat, flat[:1]])
        wide[torch.where(keep, slot, torch.full_like(slot, flat.shape[0]))] = rows
        flat.copy_(wide[:-1])
    return [torch.cat([y[0], y[1], v], dim=1).flatten(1), st["k_cache"], st["v_cache"]]


def _plain_layout(st):
    lens, starts, tables, bs = st["lens"].long(), st["starts"].long(), st["tables"], st["case"]["block"]
    n = (lens - starts).clamp_min(0)
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    cu, cu_all = torch.cat([zero, n.cumsum(0)]), torch.cat([zero, lens.cumsum(0)])
    at = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(cu[1:], at, right=True)
    inside = seq < lens.shape[0]
    seq = seq.clamp_max(lens.shape[0] - 1)
    pos = torch.where(inside, at - cu[seq] + starts[seq], torch.zeros_like(at))
    slot = tables[seq, pos // bs].long() * bs + pos % bs
    none = torch.full_like(at, -1)
    i32 = torch.int32
    return [cu.to(i32), pos.to(i32), torch.where(inside, slot, none).to(i32),
            torch.where(inside, cu_all[seq] + pos, none).to(i32)]


def _plain_moe(st):
    c = st["case"]
    T, k, H, F = c["T"], c["k"], c["H"], c["F"]
    # 64 bits for the logits alone: experts that lie next to one another are told apart by them
    logits = st["h"].double() @ st["router"].double().t()
    top, idx = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k]
    ref = top if c["norm"] else logits
    w = torch.exp(top - top[:, :1]) / torch.exp(ref - top[:, :1]).sum(-1, keepdim=True)
    w = w.float()
    if st["live"] is not None:
        on = st["live"][:, None] > 0
        w = torch.where(on, w, torch.zeros_like(w))
    flat = idx.reshape(-1)
    x = st["h"].float().repeat_interleave(k, dim=0)
    y = []
    step = max(1, int(4e8) // (H * F))  # weights of so many pairs are copied at a time
    for s in range(0, T * k, step):
        e = flat[s : s + step]
        gu = torch.bmm(st["wgu"][e].float(), x[s : s + step, :, None])[..., 0]
        act = gu[:, :F] * torch.sigmoid(gu[:, :F]) * gu[:, F:]
        y.append(torch.bmm(st["wd"][e].float(), act[..., None])[..., 0])
    out = (torch.cat(y).view(T, k, H) * w[..., None]).sum(1).to(st["h"].dtype)
    if st["live"] is not None:
        idx = torch.where(on, idx, torch.full_like(idx, -1))
    return [out, w, idx.to(torch.int32)]


def _own_pass(st):
    from skyrl_b200.ops import attention, moe_few, rotary

    c = st["case"]
    if c["op"] == "layout":
        lay = attention.paged_layout(st["tables"], st["lens"], c["block"], st["total"], starts=st["starts"])
        return [lay.cu_seqlens, lay.positions, lay.slots, lay.rows]
    if c["op"] == "moe":
        w, idx = moe_few.route_few(st["h"], st["router"], c["k"], c["norm"], live=st["live"])
        return [moe_few.expert_ffn_few(st["h"], w, idx, st["wgu"], st["wd"]), w, idx]
    if c["op"] == "cache":
        out = rotary.qk_rope_cache(st["x"], st["pos"], st["table"], st["k_cache"], st["v_cache"], st["slots"], c["nq"],
                                   c["nkv"], c["D"], q_norm=st.get("qw"), k_norm=st.get("kw"), eps=_EPS,
                                   interleaved=c["interleaved"])
        return [out, st["k_cache"], st["v_cache"]]
    x = st["x"].detach().requires_grad_()
    if c["op"] == "rotary":
        y = rotary.rotary(x, st["pos"], st["table"], c["nq"] + c["nkv"], c["D"], interleaved=c["interleaved"])
        return [y.detach(), *torch.autograd.grad(y, (x,), st["dy"])]
    qw, kw = st["qw"].detach().requires_grad_(), st["kw"].detach().requires_grad_()
    y = rotary.qk_norm_rope(x, qw, kw, st["pos"], st["table"], c["nq"], c["nkv"], c["D"], _EPS,
                            interleaved=c["interleaved"])
    return [y.detach(), *torch.autograd.grad(y, (x, qw, kw), st["dy"])]


def run(state):
    if own:
        return _own_pass(state)
    op = state["case"]["op"]
    return {"rotary": _plain_rows, "norm": _plain_rows, "cache": _plain_cache, "layout": _plain_layout,
            "moe": _plain_moe}[op](state)


# ----------------------------------------------------------------------------- from the definitions, in 64 bits
def _exact_angles(case, pos):
    """Angle of every pair at every position and the factor on the rotation, from the scaling rules one pair at a time."""
    R, base, f, L = case["R"], case["theta"], case["factor"], case["original"]
    freq, gain = [], 1.0
    for i in range(R // 2):
        w = base ** (-2.0 * i / R)
        if case["scaling"] == "linear":
            w /= f
        elif case["scaling"] == "llama3":
            turns = L * w / (2 * math.pi)
            s = min(max((turns - 1.0) / (4.0 - 1.0), 0.0), 1.0)
            w = s * w + (1 - s) * w / f
        elif case["scaling"] == "yarn":
            edge = [R * math.log(L / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (32.0, 1.0)]
            lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), R - 1)
            s = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            w = s * w / f + (1 - s) * w
            gain = 0.1 * math.log(f) + 1.0
        freq.append(w)
    w = torch.tensor(freq, dtype=torch.float64, device=pos.device)
    return pos.double()[:, None, None] * w, gain


def _exact_matrix_pairs(case, device):
    """Element indices (first, second) of every rotated pair."""
    i = torch.arange(case["R"] // 2, device=device)
    return (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + case["R"] // 2)


def _exact_rotate(x, ang, gain, case, back=False):
    z = torch.complex(gain * torch.cos(ang), gain * torch.sin(ang))
    first, second = _exact_matrix_pairs(case, x.device)
    p = torch.complex(x[..., first], x[..., second]) * (z.conj() if back else z)
    out = x.clone()
    out[..., first], out[..., second] = p.real, p.imag
    return out


def _exact_rows(case, seed):
    st = _rows(case, seed)
    nq, nkv, D, T = case["nq"], case["nkv"], case["D"], case["T"]
    ang, gain = _exact_angles(case, st["pos"])
    x, d = st["x"].double().view(T, -1, D), st["dy"].double().view(T, -1, D)
    y, dx = x.clone(), d.clone()
    grads = []
    for lo, hi, key in ((0, nq, "qw"), (nq, nq + nkv, "kw")):
        a, g = x[:, lo:hi], _exact_rotate(d[:, lo:hi], ang, gain, case, back=True)
        if key not in st:
            y[:, lo:hi], dx[:, lo:hi] = _exact_rotate(a, ang, gain, case), g
            continue
        w = st[key].double()
        rms = torch.sqrt((a * a).sum(-1, keepdim=True) / D + _EPS)
        y[:, lo:hi] = _exact_rotate(a / rms * w, ang, gain, case)
        grads.append(torch.einsum("thd,thd->d", g, a / rms))
        # d(a_i / rms) / d a_j = (delta_ij - a_i a_j / (D rms^2)) / rms
        along = ((g * w) * a).sum(-1, keepdim=True) / (D * rms * rms)
        dx[:, lo:hi] = (g * w - a * along) / rms
    return [y.reshape(T, -1), dx.reshape(T, -1), *grads]


def _exact_cache(case, seed):
    st = _rows(case, seed)
    nq, nkv, D, T = case["nq"], case["nkv"], case["D"], case["T"]
    ang, gain = _exact_angles(case, st["pos"])
    x = st["x"]
    if x.dim() == 3:
        x = x.double().sum(0).to(_DTYPES[case["dtype"]])  # the projection's output is held in this type
    out = x.double().view(T, -1, D).clone()
    for lo, hi, key in ((0, nq, "qw"), (nq, nq + nkv, "kw")):
        a = out[:, lo:hi]
        if key in st:
            a = a / torch.sqrt((a * a).sum(-1, keepdim=True) / D + _EPS) * st[key].double()
        out[:, lo:hi] = _exact_rotate(a, ang, gain, case)
    caches = []
    live = torch.nonzero(st["slots"] >= 0)[:, 0]
    for lo in (nq, nq + nkv):
        cache = st["k_cache"].double().view(-1, nkv, D)
        cache[st["slots"][live].long()] = out[live, lo : lo + nkv]
        caches.append(cache.view(st["k_cache"].shape))
    return [out.reshape(T, -1), *caches]


def _exact_moe(case, seed):
    st = _moe_inputs(case, seed)
    T, k, H, F = case["T"], case["k"], case["H"], case["F"]
    h = st["h"].double()
    z = (h[:, None, :] * st["router"].double()[None]).sum(-1) if T * case["E"] * H < 1 << 26 else None
    if z is None:
        z = torch.stack([(h[t] * st["router"].double()).sum(-1) for t in range(T)])
    p = torch.softmax(z, dim=-1)
    out = torch.zeros(T, H, dtype=torch.float64, device=h.device)
    W = torch.zeros(T, k, dtype=torch.float64, device=h.device)
    mass = torch.zeros(T, dtype=torch.float64, device=h.device)
    left = p.clone()
    pick = []
    for s in range(k):  # the largest that is left
        pick.append(left.argmax(-1))
        W[:, s] = p.gather(1, pick[s][:, None])[:, 0]
        mass += W[:, s]
        left.scatter_(1, pick[s][:, None], -1.0)
    if case["norm"]:
        W /= mass[:, None]
    if st["live"] is not None:
        W *= (st["live"] > 0).double()[:, None]
    choice = torch.stack(pick, 1)
    for e in choice.unique().tolist():
        t, s = torch.nonzero(choice == e, as_tuple=True)
        up = h[t] @ st["wgu"][e].double().t()
        act = up[:, :F] / (1 + torch.exp(-up[:, :F])) * up[:, F:]
        out.index_add_(0, t, (act @ st["wd"][e].double().t()) * W[t, s][:, None])
    return [out, W, None]


def _exact_layout(case, seed):
    """Request after request, on the host."""
    st, bs = _layout_inputs(case, seed), case["block"]
    tables = st["tables"].cpu().long()
    pos, slots, rows, cu, whole = [], [], [], [0], 0
    for i, (n, c) in enumerate(zip(st["lens"].tolist(), st["starts"].tolist())):
        p = torch.arange(c, max(n, c))
        pos.append(p)
        slots.append(tables[i].repeat_interleave(bs)[p] * bs + p.remainder(bs))
        rows.append(p + whole)
        cu.append(cu[-1] + len(p))
        whole += n
    spare = st["total"] - cu[-1]
    pos.append(torch.zeros(spare, dtype=torch.long))
    for out in (slots, rows):
        out.append(torch.full((spare,), -1, dtype=torch.long))
    return [t.cuda() for t in (torch.tensor(cu), torch.cat(pos), torch.cat(slots), torch.cat(rows))]


def exact(case, seed):
    if case["op"] == "layout":
        return _exact_layout(case, seed)
    if case["op"] == "moe":
        return _exact_moe(case, seed)
    return _exact_cache(case, seed) if case["op"] == "cache" else _exact_rows(case, seed)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "layout":
        # lengths, starts and the offsets; the table entries that are used and three numbers a row
        rows = sum(n - c for n, c in _layout_lengths(case))
        return {"bytes": 12 * case["B"] + rows * (12 + 4 / case["block"]), "flops": 0}
    if op == "moe":
        T, E, k, H, F = (case[n] for n in ("T", "E", "k", "H", "F"))
        rows = T * (1 - case["dead"])
        used = E * (1 - (1 - k / E) ** rows)  # experts that some row picks, in the mean
        return {"bytes": 2 * (used * 3 * F * H + E * H + 2 * T * H) + 8 * T * k, "flops": 2 * rows * k * 3 * F * H + 2 * T * E * H}
    size = 4 if case["dtype"] == "fp32" else 2
    T, W = case["T"], (case["nq"] + 2 * case["nkv"]) * case["D"]
    turned = (case["nq"] + case["nkv"]) * case["D"]
    angles = T * (4 * case["R"] + 4)
    if op == "cache":
        src = case["parts"] * 4 if case["parts"] else size
        kv = 2 * case["nkv"] * case["D"] * size * (1 - case["hole"])
        return {"bytes": T * (W * (src + size) + kv + 4) + angles, "flops": T * turned * 8}
    # rows and their gradients in and out once; the backward pass of the norm needs the heads that it normalised
    again = T * turned * size if op == "norm" else 0
    return {"bytes": 4 * T * W * size + again + 2 * angles, "flops": T * turned * (24 if op == "norm" else 6)}
