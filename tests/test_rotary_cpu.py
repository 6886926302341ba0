"""Rotary tables and the CPU formulation of rotary / head norms / cache rows against 64-bit definitions; refusals."""
import math

import pytest
import torch

from skyrl_b200.ops import attention, rotary
from skyrl_b200.ops import elementwise as ew

SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
}


def angles64(pos, R, theta, scaling):
    """[T, R/2] fp64 angles and the factor on the rotation, pair by pair from the scaling rules."""
    freq, gain = [], 1.0
    kind = (scaling or {}).get("rope_type") or (scaling or {}).get("type")
    for i in range(R // 2):
        w = theta ** (-2.0 * i / R)
        if kind == "linear":
            w /= scaling["factor"]
        elif kind == "llama3":
            L, lo, hi = scaling["original_max_position_embeddings"], scaling["low_freq_factor"], scaling["high_freq_factor"]
            wave = 2 * math.pi / w
            if wave > L / lo:
                w /= scaling["factor"]
            elif wave >= L / hi:
                s = (L / wave - lo) / (hi - lo)
                w = (1 - s) * w / scaling["factor"] + s * w
        elif kind == "yarn":
            L, f = scaling["original_max_position_embeddings"], scaling["factor"]
            edge = [R * math.log(L / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (32.0, 1.0)]
            lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), R - 1)
            s = min(max((i - lo) / (hi - lo), 0.0), 1.0)
            w = s * w / f + (1 - s) * w
            gain = 0.1 * math.log(f) + 1.0
        freq.append(w)
    return pos.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=pos.device), gain


def rows64(x, qw, kw, ang, gain, nq, nk, D, eps, interleaved):
    """The definition in fp64 (differentiable): norm and rotation of the first nq + nk heads of rows ``x`` [T, W]."""
    T = x.shape[0]
    h = x.double().view(T, x.shape[1] // D, D)
    z = torch.polar(torch.full_like(ang, gain), ang)[:, None]
    half = ang.shape[1]
    out = []
    for lo, hi, w in ((0, nq, qw), (nq, nq + nk, kw)):
        p = h[:, lo:hi]
        if w is not None:
            p = p / torch.sqrt((p * p).sum(-1, keepdim=True) / D + eps) * w.double()
        rot, rest = p[..., : 2 * half], p[..., 2 * half :]
        pair = rot.unflatten(-1, (half, 2)) if interleaved else rot.unflatten(-1, (2, half)).transpose(-1, -2)
        c = torch.complex(pair[..., 0].contiguous(), pair[..., 1].contiguous()) * z
        rot = torch.stack([c.real, c.imag], -1 if interleaved else -2).flatten(-2)
        out.append(torch.cat([rot, rest], -1))
    return torch.cat([*out, h[:, nq + nk :]], 1).flatten(1)


@pytest.mark.parametrize("kind", sorted(SCALINGS))
@pytest.mark.parametrize("R,theta", [(128, 1e6), (32, 1e4), (20, 5e5)])
def test_table_matches_the_scaling_rules(kind, R, theta):
    pos = torch.tensor([0, 1, 77, 4095, 40000])
    ang, gain = angles64(pos, R, theta, SCALINGS[kind])
    tab = ew.build_rope_table(40001, R, theta, "cpu", scaling=SCALINGS[kind])
    want = torch.cat([ang.cos(), ang.sin()], -1) * gain
    # one fp32 rounding of a value of at most gain, and fp64 angles of up to 4e4 that two orders of operations form
    assert (tab[pos].double() - want).abs().max() <= gain * (2.0**-24 + 4e4 * 2.0**-50)


def test_unscaled_table_is_the_one_without_scaling():
    a, b = ew.build_rope_table(300, 64, 1e4, "cpu"), ew.build_rope_table(300, 64, 1e4, "cpu", scaling={"rope_type": "default"})
    assert torch.equal(a, b)


def test_table_refusals():
    for bad in ({"rope_type": "spiral", "factor": 2.0}, {"type": "linear", "factor": 0.5},
                {"rope_type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
                 "original_max_position_embeddings": 1024}):
        with pytest.raises(ValueError):
            ew.build_rope_table(8, 8, 1e4, "cpu", scaling=bad)


CASES = [  # T, nq, nkv, D, R, interleaved
    (7, 2, 1, 16, 16, False), (7, 2, 1, 16, 8, False), (5, 3, 1, 10, 6, True), (4, 4, 2, 24, 24, True), (1, 1, 1, 8, 2, False),
    (0, 2, 1, 16, 16, False),
]


@pytest.mark.parametrize("T,nq,nkv,D,R,inter", CASES)
@pytest.mark.parametrize("normed", [False, True])
def test_rows_and_gradients_match_64_bits(T, nq, nkv, D, R, inter, normed):
    g = torch.Generator().manual_seed(T * 100 + D)
    W = (nq + 2 * nkv) * D
    x = torch.randn(T, W, generator=g)
    qw, kw = (1 + 0.2 * torch.randn(D, generator=g) for _ in range(2))
    dy = torch.randn(T, W, generator=g)
    pos = torch.randint(0, 500, (T,), generator=g).to(torch.int32)
    table = ew.build_rope_table(500, R, 1e4, "cpu")
    ang, gain = angles64(pos, R, 1e4, None)
    leaves = [t.clone().requires_grad_() for t in (x, qw, kw)]
    if normed:
        y = rotary.qk_norm_rope(*leaves, pos, table, nq, nkv, D, 1e-6, interleaved=inter)
    else:
        y = rotary.rotary(leaves[0], pos, table, nq + nkv, D, interleaved=inter)
    l64 = [t.double().requires_grad_() for t in (x, qw, kw)]
    y64 = rows64(l64[0], l64[1] if normed else None, l64[2] if normed else None, ang, gain, nq, nkv, D, 1e-6, inter)
    # about 64 fp32 roundings of values below 16
    assert (y.double() - y64).abs().max().item() <= 2.0**-14 if T else y.shape == (0, W)
    n = 3 if normed else 1
    got, want = torch.autograd.grad(y, leaves[:n], dy), torch.autograd.grad(y64, l64[:n], dy.double())
    for a, b in zip(got, want):
        assert a.dtype == torch.float32 and (T == 0 or (a.double() - b).abs().max() <= 2.0**-14 * max(1, b.abs().max()))
    if T == 0:
        assert all(float(a.abs().sum()) == 0 for a in got)
        return
    # the formula's gradient against differences of the definition, along one direction
    v = torch.randn(x.shape, generator=g, dtype=torch.float64)
    f = lambda e: (rows64(x.double() + e * v, l64[1].detach() if normed else None, l64[2].detach() if normed else None,  # noqa: E731
                          ang, gain, nq, nkv, D, 1e-6, inter) * dy.double()).sum()
    diff = (f(1e-6) - f(-1e-6)) / 2e-6
    assert abs(float(diff - (got[0].double() * v).sum())) <= 1e-4 * (1 + float((got[0].double() * v).abs().sum()))


def test_weight_gradients_go_to_main_grad_and_accumulate():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 48, generator=g, requires_grad=True)
    qw, kw = (torch.nn.Parameter(1 + 0.1 * torch.randn(16, generator=g)) for _ in range(2))
    pos, table = torch.arange(6, dtype=torch.int32), ew.build_rope_table(6, 16, 1e4, "cpu")
    call = lambda: rotary.qk_norm_rope(x, qw, kw, pos, table, 1, 1, 16, 1e-6).square().sum().backward()  # noqa: E731
    call()
    want = qw.grad.clone(), kw.grad.clone()
    qw.grad = kw.grad = None
    qw.main_grad, kw.main_grad = torch.ones(16), torch.zeros(16)
    call()
    call()
    assert qw.grad is None and kw.grad is None
    assert torch.allclose(qw.main_grad, 1 + 2 * want[0], atol=1e-5) and torch.allclose(kw.main_grad, 2 * want[1], atol=1e-5)


def test_one_weight_for_queries_and_keys():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(6, 48, generator=g), torch.nn.Parameter(1 + 0.1 * torch.randn(16, generator=g))
    pos, table = torch.arange(6, dtype=torch.int32), ew.build_rope_table(6, 16, 1e4, "cpu")
    call = lambda: rotary.qk_norm_rope(x, w, w, pos, table, 1, 1, 16, 1e-6).square().sum().backward()  # noqa: E731
    call()
    want, w.grad = w.grad.clone(), None
    w.main_grad = torch.zeros(16)
    call()
    assert w.grad is None and torch.allclose(w.main_grad, want, atol=1e-5)


def test_cache_rows_partial_sums_and_empty_slots():
    g = torch.Generator().manual_seed(1)
    T, nq, nkv, D, bs = 9, 3, 2, 16, 4
    W = (nq + 2 * nkv) * D
    part = torch.randn(3, T, W, generator=g)
    x = part.double().sum(0).float()
    qw, kw = (1 + 0.2 * torch.randn(D, generator=g) for _ in range(2))
    pos, table = torch.arange(T, dtype=torch.int32) * 3, ew.build_rope_table(64, D, 1e4, "cpu")
    slots = torch.tensor([5, -1, 0, 19, 20, 7, -5, 2, 11], dtype=torch.int32)  # 20 lies behind the cache
    kc, vc = torch.full((5, bs, nkv, D), 9.0), torch.full((5, bs, nkv, D), 7.0)
    y = rotary.qk_rope_cache(part, pos, table, kc, vc, slots, nq, nkv, D, q_norm=qw, k_norm=kw)
    want = rotary.qk_norm_rope(x, qw, kw, pos, table, nq, nkv, D, 1e-6)
    assert torch.equal(y, want)
    ek, ev = torch.full((20, nkv * D), 9.0), torch.full((20, nkv * D), 7.0)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < 20:
            ek[s], ev[s] = want[t, nq * D : (nq + nkv) * D], want[t, (nq + nkv) * D :]
    assert torch.equal(kc.view(20, -1), ek) and torch.equal(vc.view(20, -1), ev)
    rows = x.clone()
    same = rotary.qk_rope_cache(rows, pos, table, kc, vc, slots, nq, nkv, D, q_norm=qw, k_norm=kw, out=rows)
    assert same is rows and torch.equal(rows, want)


def test_position_outside_the_table_is_nan_in_the_rotated_part_only():
    pos, table = torch.tensor([0, -1, 8], dtype=torch.int32), ew.build_rope_table(8, 4, 1e4, "cpu")
    y = rotary.rotary(torch.ones(3, 24), pos, table, 2, 8)
    nan = torch.isnan(y.view(3, 3, 8))
    assert not nan[0].any() and nan[1:, :2, :4].all() and not nan[1:, :2, 4:].any() and not nan[1:, 2].any()


def test_refusals():
    x, pos, table = torch.randn(4, 48), torch.arange(4, dtype=torch.int32), ew.build_rope_table(8, 16, 1e4, "cpu")
    w = torch.ones(16)
    ok = dict(x=x, pos=pos, table=table, n=2, D=16)
    for bad in (dict(x=x.view(2, 2, 48)), dict(x=x.long()), dict(pos=pos.long()), dict(pos=pos[:3]), dict(pos=torch.arange(8, dtype=torch.int32)[::2]),
                dict(table=table.half()), dict(table=table[:, :3]), dict(table=table[:, ::2]), dict(n=4), dict(D=20), dict(n=0),
                dict(D=8), dict(x=torch.randn(4, 2048), D=1024)):
        a = {**ok, **bad}
        with pytest.raises(ValueError):
            rotary.rotary(a["x"], a["pos"], a["table"], a["n"], a["D"])
    for qw, kw in ((w, None), (w, w[:8]), (w, w.double()), (torch.ones(32)[::2], w)):
        with pytest.raises(ValueError):
            rotary.qk_norm_rope(x, qw, kw, pos, table, 1, 1, 16, 1e-6)
    kc, vc, slots = torch.zeros(2, 4, 1, 16), torch.zeros(2, 4, 1, 16), torch.arange(4, dtype=torch.int32)
    ok = dict(x=x, kc=kc, vc=vc, slots=slots, out=None, nq=1)
    for bad in (dict(x=x.half()), dict(x=x[None].half()), dict(x=x.clone().requires_grad_()), dict(kc=kc.transpose(0, 1)), dict(vc=vc[:1]),
                dict(vc=vc.half()), dict(slots=slots.long()), dict(slots=slots[:2]), dict(out=torch.empty(4, 64)), dict(nq=2),
                dict(out=torch.empty(4, 48).half()), dict(x=x[0])):
        a = {**ok, **bad}
        with pytest.raises(ValueError):
            rotary.qk_rope_cache(a["x"], pos, table, a["kc"], a["vc"], a["slots"], a["nq"], 1, 16, out=a["out"])


def test_cache_rows_refuse_weights_with_gradients_and_overlapping_rows():
    buf = torch.randn(8, 112)
    x, pos, table = buf[:4, :48], torch.arange(4, dtype=torch.int32), ew.build_rope_table(8, 16, 1e4, "cpu")
    kc, vc, slots, w = torch.zeros(2, 4, 1, 16), torch.zeros(2, 4, 1, 16), torch.arange(4, dtype=torch.int32), torch.ones(16)

    def run(out, x=x, q_norm=None, k_norm=None):
        return rotary.qk_rope_cache(x, pos, table, kc, vc, slots, 1, 1, 16, q_norm=q_norm, k_norm=k_norm, out=out)

    for q, k in ((w.clone().requires_grad_(), w), (w, w.clone().requires_grad_())):
        with pytest.raises(ValueError, match="gradient"):
            run(None, q_norm=q, k_norm=k)
        with torch.no_grad():
            run(None, q_norm=q, k_norm=k)
    part = torch.randn(3, 4, 48)
    for out in (buf[1:5, :48], buf[:4, 16:64], buf.view(-1)[: 4 * 56].view(4, 56)[:, :48]):
        with pytest.raises(ValueError, match="lies on"):
            run(out)
    with pytest.raises(ValueError, match="lies on"):
        run(part[1], x=part)
    want = run(None)
    for out in (buf[4:, :48], buf[:4, 48:96], buf[1:5, 64:]):  # other rows; columns beside
        assert torch.equal(run(out), want)
    assert torch.equal(run(x), want)


# ----------------------------------------------------------------------------- paged layout
def layout_oracle(tables, lens, starts, bs, total):
    cu, pos, slots, rows, whole = [0], [], [], [], 0
    for b, n in enumerate(lens):
        n = max(n, 0)
        s = min(max(starts[b], 0), n) if starts else 0
        for p in range(s, n):
            e = tables[b][p // bs] if p // bs < len(tables[b]) else -1
            pos.append(p)
            slots.append(e * bs + p % bs if e >= 0 else -1)
            rows.append(whole + p)
        cu.append(cu[-1] + n - s)
        whole += n
    pad = max(0, total - len(pos))
    return cu, (pos + [0] * pad)[:total], (slots + [-1] * pad)[:total], (rows + [-1] * pad)[:total]


LAYOUTS = [  # lens, starts, block size, table width, rows more or less than there are
    ([1], None, 4, 1, 0), ([5, 0, 3], [4, 0, 0], 4, 2, 3), ([9, 9, 9], [9, 0, 8], 4, 3, 0), ([0, 0], None, 2, 1, 2),
    ([7, 2], [0, 2], 4, 1, 0), ([12], [3], 5, 3, -4), ([3, -2, 4], [-1, 0, 9], 2, 2, 1), ([], None, 8, 1, 2), ([4, 4], None, 8, 0, 0),
]


def layout_case(lens, starts, bs, width, extra, device="cpu"):
    g = torch.Generator().manual_seed(len(lens) + bs)
    B = len(lens)
    tables = torch.randperm(B * width + 5, generator=g)[: B * width].view(B, width).to(torch.int32)
    if B * width > 2:
        tables[0, -1] = -1
    n = len(layout_oracle(tables.tolist(), lens, starts, bs, 0)[0]) and layout_oracle(tables.tolist(), lens, starts, bs, 0)[0][-1]
    total = max(0, n + extra)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    got = attention.paged_layout(tables.to(device), i32(lens), bs, total, starts=None if starts is None else i32(starts))
    want = layout_oracle(tables.tolist(), lens, starts, bs, total)
    return got, want


@pytest.mark.parametrize("lens,starts,bs,width,extra", LAYOUTS)
def test_layout(lens, starts, bs, width, extra):
    got, want = layout_case(lens, starts, bs, width, extra)
    for g, w in zip(got, want):
        assert g.dtype == torch.int32 and g.tolist() == w


def test_layout_refusals():
    t, n = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for a in ((t.long(), n, 4, 2), (t[0], n, 4, 2), (t, n.long(), 4, 2), (t, n[:1], 4, 2), (t, n, 0, 2), (t, n, 4, -1), (t, n, 4, 2**31),
              (t.t(), torch.ones(3, dtype=torch.int32), 4, 2)):
        with pytest.raises(ValueError):
            attention.paged_layout(*a)
    with pytest.raises(ValueError):
        attention.paged_layout(t, n, 4, 2, starts=n.long())
