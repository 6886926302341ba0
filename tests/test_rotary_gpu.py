"""Rotary / head-norm / cache-row / layout kernels against 64-bit definitions on the device."""
import pytest
import torch
from test_rotary_cpu import LAYOUTS, SCALINGS, angles64, layout_case, layout_oracle, rows64

from skyrl_b200.ops import _lib, attention, rotary
from skyrl_b200.ops import elementwise as ew

pytestmark = pytest.mark.gpu


def half_step(t, dtype):
    """Bound on one rounding to ``dtype``: half a step of the value, or half the smallest step."""
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    return torch.finfo(dtype).eps / 2 * t.abs() + tiny


def head_max(t, D):
    """Largest magnitude of every head, on all its elements."""
    h = t.abs().view(t.shape[0], -1, D)
    return h.max(-1, keepdim=True).values.expand_as(h).reshape(t.shape)


def head_sum(t, D):
    h = t.abs().view(t.shape[0], -1, D)
    return h.sum(-1, keepdim=True).expand_as(h).reshape(t.shape)


def make(T, nq, nkv, D, R, dtype, seed=0, theta=1e4, scaling=None, max_pos=3000, layout="plain"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    W = (nq + 2 * nkv) * D
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731

    def rows():
        if layout == "plain":
            return rnd(T, W).to(dtype)
        if layout == "strided":  # columns of a wider row
            return rnd(T, W + 64).to(dtype)[:, 32 : 32 + W]
        if layout == "odd":  # no 16-byte alignment
            return rnd(T, W + 3).to(dtype)[:, 1 : 1 + W]
        return rnd(W, T).to(dtype).t()  # transposed

    x, dy = rows(), rows()
    if T > 2:
        x[1] = 0  # a row without length: the norm divides by sqrt(eps)
        x[2] *= 100
    qw, kw = ((1 + 0.3 * rnd(D)).to(dtype) for _ in range(2))
    pos = torch.randint(0, max_pos, (T,), generator=g, device="cuda").to(torch.int32)
    table = ew.build_rope_table(max_pos, R, theta, "cuda", scaling=scaling)
    return x, dy, qw, kw, pos, table, *angles64(pos, R, theta, scaling)


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
SIZES = [  # T, nq, nkv, D, R, interleaved, dtype, layout, scaling
    (1, 1, 1, 128, 128, False, BF, "plain", "none"), (3, 2, 1, 64, 64, True, BF, "plain", "yarn"),
    (37, 14, 2, 64, 32, False, HF, "plain", "none"), (300, 32, 4, 128, 128, False, BF, "plain", "yarn"),
    (65, 3, 3, 80, 80, True, FP, "plain", "linear"), (130, 5, 1, 96, 48, False, BF, "strided", "llama3"),
    (29, 4, 2, 256, 64, True, HF, "plain", "none"), (17, 2, 2, 512, 512, False, BF, "plain", "none"),
    (33, 4, 1, 128, 96, False, FP, "strided", "none"), (20, 3, 2, 40, 24, False, BF, "plain", "none"),
    (21, 2, 1, 24, 6, True, FP, "plain", "none"), (40, 2, 1, 128, 128, False, BF, "odd", "none"),
    (40, 2, 1, 64, 20, True, HF, "odd", "none"), (50, 2, 1, 128, 64, True, BF, "transposed", "none"),
    (9, 1, 1, 7, 2, False, BF, "plain", "none"), (11, 2, 1, 192, 192, False, BF, "plain", "none"),
    (5000, 32, 4, 128, 128, False, BF, "plain", "none"), (8001, 14, 2, 64, 32, True, HF, "plain", "none"),
    (2500, 16, 8, 128, 64, False, FP, "plain", "none"), (16000, 6, 1, 128, 64, True, BF, "plain", "yarn"),
    (12000, 10, 3, 80, 80, False, HF, "strided", "none"), (10000, 8, 4, 96, 24, False, BF, "plain", "llama3"),
    (4000, 8, 4, 256, 256, True, FP, "plain", "none"), (700, 4, 2, 80, 40, True, BF, "strided", "none"),
    (4001, 2, 1, 24, 8, False, FP, "plain", "none"), (801, 5, 3, 512, 64, False, HF, "plain", "none"),
    (3000, 8, 2, 80, 20, False, BF, "plain", "none"), (2000, 5, 1, 80, 20, True, HF, "plain", "yarn"),
    (1500, 4, 4, 96, 92, False, FP, "strided", "none"), (2500, 3, 1, 8, 4, False, BF, "plain", "none"),
    (3001, 6, 2, 72, 36, False, HF, "plain", "linear"), (1999, 2, 2, 256, 12, True, BF, "plain", "none"),
]


@pytest.mark.parametrize("T,nq,nkv,D,R,inter,dtype,layout,scaling", SIZES)
@pytest.mark.parametrize("normed", [False, True])
def test_rows_and_gradients(T, nq, nkv, D, R, inter, dtype, layout, scaling, normed):
    eps = 1e-6
    x, dy, qw, kw, pos, table, ang, gain = make(T, nq, nkv, D, R, dtype, scaling=SCALINGS[scaling], layout=layout)
    leaves = [x.detach().requires_grad_(), *(w.detach().requires_grad_() for w in ((qw, kw) if normed else ()))]
    if normed:
        y = rotary.qk_norm_rope(*leaves, pos, table, nq, nkv, D, eps, interleaved=inter)
    else:
        y = rotary.rotary(leaves[0], pos, table, nq + nkv, D, interleaved=inter)
    got = torch.autograd.grad(y, leaves, dy)
    l64 = [t.detach().double().requires_grad_() for t in (x, qw, kw)]
    y64 = rows64(l64[0], l64[1] if normed else None, l64[2] if normed else None, ang, gain, nq, nkv, D, eps, inter)
    want = torch.autograd.grad(y64, l64[: len(leaves)], dy.double())
    y64 = y64.detach()
    # forward: about 16 fp32 roundings (statistics, products, table) of values of the head's size, then one of the result
    tol = half_step(y64, dtype) + 2.0**-19 * gain * head_max(y64, D)
    assert ((y.double() - y64).abs() <= tol).all()
    turned = (nq + nkv) * D
    assert torch.equal(y[:, turned:], x[:, turned:]) and torch.equal(got[0][:, turned:], dy[:, turned:])
    if not normed:
        tol = half_step(want[0], dtype) + 2.0**-20 * gain * 2 * head_max(dy.double(), D)
        assert ((got[0].double() - want[0]).abs() <= tol).all()
        return
    # dx = r (g w - xh mean(g w xh)): sums over a head are of D terms (16 in a lane, then a tree): 2^-18 of the terms
    h = x.double().reshape(T, -1, D)[:, : nq + nkv]
    r = torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    w = torch.cat([qw.double().expand(nq, D), kw.double().expand(nkv, D)])[None]
    gmax = 2 * gain * dy.double().reshape(T, -1, D)[:, : nq + nkv].abs().max(-1, keepdim=True).values * w.abs().max()
    xh = (h * r).abs()
    size = (r * gmax * (1 + xh.max(-1, keepdim=True).values * xh.mean(-1, keepdim=True))).expand(T, nq + nkv, D).reshape(T, turned)
    d64 = want[0][:, :turned]
    assert ((got[0][:, :turned].double() - d64).abs() <= half_step(d64, dtype) + 2.0**-18 * size).all()
    # dw: every thread adds up at most 64 heads here before trees over lanes, warps and CTAs (at most 20 rows a step)
    for a, b, lo, hi in ((got[1], want[1], 0, nq), (got[2], want[2], nq, nq + nkv)):
        terms = (xh[:, lo:hi] * gmax[:, lo:hi]).sum((0, 1))
        assert a.dtype == dtype and ((a.double() - b).abs() <= half_step(b, dtype) + 2.0**-16 * terms).all()


def test_weight_gradients_are_repeatable_and_reach_main_grad():
    T, nq, nkv, D = 3001, 8, 2, 128
    x, dy, qw, kw, pos, table, *_ = make(T, nq, nkv, D, D, BF)
    x = x.requires_grad_()

    def grads(q, k):
        y = rotary.qk_norm_rope(x, q, k, pos, table, nq, nkv, D, 1e-6)
        return torch.autograd.grad(y, [t for t in (x, q, k) if t.requires_grad], dy, allow_unused=True)

    q, k = (torch.nn.Parameter(w.clone()) for w in (qw, kw))
    first = grads(q, k)
    for a, b in zip(first, grads(q, k)):
        assert torch.equal(a, b)
    for mg in ((torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")), (None, torch.zeros(D, device="cuda"))):
        q, k = (torch.nn.Parameter(w.clone()) for w in (qw, kw))
        for p, m in zip((q, k), mg):
            if m is not None:
                p.main_grad = m
        for _ in range(2):
            out = grads(q, k)
        assert torch.equal(out[0], first[0]) and out[2] is None
        # two equal fp32 sums on top of what was there, against one sum that was rounded to bf16
        assert ((mg[1] / 2 - first[2].float()).abs() <= 2.0**-8 * first[2].float().abs() + 1e-6).all()
        if mg[0] is None:
            assert torch.equal(out[1], first[1])
        else:
            assert out[1] is None and (((mg[0] - 1) / 2 - first[1].float()).abs() <= 2.0**-8 * first[1].float().abs() + 2.0**-20).all()
    frozen = grads(qw, kw)  # weights without gradients
    assert len(frozen) == 1 and torch.equal(frozen[0], first[0])


CACHE = [  # T, parts, nq, nkv, D, R, interleaved, dtype, normed
    (1, 1, 2, 1, 128, 128, False, BF, True), (64, 4, 32, 4, 128, 128, False, BF, True), (77, 0, 32, 4, 128, 128, False, BF, True),
    (50, 3, 4, 2, 64, 32, True, BF, False), (33, 0, 3, 3, 96, 96, True, HF, False), (20, 2, 2, 1, 40, 24, False, BF, True),
    (19, 0, 2, 1, 24, 10, True, FP, True), (4100, 0, 32, 4, 128, 128, False, BF, True), (600, 8, 4, 4, 256, 128, False, HF, True),
    (14001, 0, 6, 1, 128, 128, True, BF, False), (9001, 0, 14, 3, 96, 96, False, HF, True),
]


@pytest.mark.parametrize("T,parts,nq,nkv,D,R,inter,dtype,normed", CACHE)
def test_cache_rows(T, parts, nq, nkv, D, R, inter, dtype, normed):
    x, _, qw, kw, pos, table, ang, gain = make(T, nq, nkv, D, R, dtype, seed=3)
    if not normed:
        qw = kw = None
    W, bs = x.shape[1], 16
    g = torch.Generator(device="cuda").manual_seed(5)
    src = x
    if parts:
        src = torch.randn(parts, T, W, generator=g, device="cuda")
        x = src.double().sum(0).float().to(dtype)  # a sum that has lost nothing, in fp32 and then in the rows' type
    blocks = T // bs + 2
    slots = torch.randperm(blocks * bs, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 4:
        slots[1], slots[3], slots[4] = -1, -7, blocks * bs  # none, none, behind the cache
    kc, vc = (torch.full((blocks, bs, nkv, D), v, device="cuda", dtype=dtype) for v in (3.0, 5.0))
    y = rotary.qk_rope_cache(src, pos, table, kc, vc, slots, nq, nkv, D, q_norm=qw, k_norm=kw, eps=1e-6, interleaved=inter)
    y64 = rows64(x, qw, kw, ang, gain, nq, nkv, D, 1e-6, inter)
    assert ((y.double() - y64).abs() <= half_step(y64, dtype) + 2.0**-19 * head_max(y64, D)).all()
    ek, ev = (torch.full((blocks * bs, nkv * D), v, device="cuda", dtype=dtype) for v in (3.0, 5.0))
    on = (slots >= 0) & (slots < blocks * bs)
    ek[slots[on].long()], ev[slots[on].long()] = y[on, nq * D : (nq + nkv) * D], y[on, (nq + nkv) * D :]
    assert torch.equal(kc.view(blocks * bs, -1), ek) and torch.equal(vc.view(blocks * bs, -1), ev)
    if not parts:  # the same in place
        kc2, vc2 = (torch.full((blocks, bs, nkv, D), v, device="cuda", dtype=dtype) for v in (3.0, 5.0))
        rows = x.clone()
        back = rotary.qk_rope_cache(rows, pos, table, kc2, vc2, slots, nq, nkv, D, q_norm=qw, k_norm=kw, eps=1e-6,
                                    interleaved=inter, out=rows)
        assert back is rows and torch.equal(rows, y) and torch.equal(kc2, kc) and torch.equal(vc2, vc)
    assert _lib.status_read_clear() == 0


def test_long_cache_offsets_pass_32_bits():
    """A slot whose byte and element offsets lie beyond 2^32 and 2^31."""
    nkv, D, bs = 8, 128, 32
    blocks = (1 << 31) // (nkv * D * bs) + 2  # elements: just above 2^31
    kc = torch.zeros(blocks, bs, nkv, D, device="cuda", dtype=BF)
    vc = torch.zeros_like(kc)
    x, _, _, _, pos, table, *_ = make(2, 8, nkv, D, D, BF)
    slots = torch.tensor([blocks * bs - 1, 1], device="cuda", dtype=torch.int32)
    y = rotary.qk_rope_cache(x, pos, table, kc, vc, slots, 8, nkv, D)
    assert torch.equal(kc.view(-1, nkv * D)[slots.long()], y[:, 8 * D : 16 * D])
    assert torch.equal(vc.view(-1, nkv * D)[slots.long()], y[:, 16 * D :])
    kc.view(-1, nkv * D)[slots.long()] = 0
    assert not kc.any()


def test_one_weight_for_queries_and_keys():
    """Both gradients go to one buffer: to its fp32 main_grad and through the rows' type."""
    T, nq, nkv, D = 2000, 4, 4, 64
    x, dy, w, _, pos, table, *_ = make(T, nq, nkv, D, D, BF)
    q, k = w.clone().requires_grad_(), w.clone().requires_grad_()
    dq, dk = torch.autograd.grad(rotary.qk_norm_rope(x, q, k, pos, table, nq, nkv, D, 1e-6), (q, k), dy)
    one = torch.nn.Parameter(w.clone())
    one.main_grad = torch.zeros(D, device="cuda")
    rotary.qk_norm_rope(x, one, one, pos, table, nq, nkv, D, 1e-6).backward(dy)
    # the two sums are fp32 in the buffer and were rounded to bf16 above, half a step each
    assert one.grad is None
    assert ((one.main_grad - dq.float() - dk.float()).abs() <= 2.0**-8 * (dq.float().abs() + dk.float().abs()) + 2.0**-20).all()


@pytest.mark.parametrize("D", [64, 24])
def test_infinite_partial_sums_stay_infinite(D):
    x, _, _, _, pos, table, *_ = make(4, 2, 1, D, D, BF)
    part = torch.stack([x.float(), torch.ones(4, 4 * D, device="cuda"), torch.zeros(4, 4 * D, device="cuda")])
    part[1, 1, 3 * D + 2], part[1, 2, 3 * D + 5] = float("inf"), float("-inf")  # value heads
    part[1, 3, 3 * D + 7], part[2, 3, 3 * D + 7] = float("inf"), float("-inf")
    kc, vc = (torch.zeros(1, 4, 1, D, device="cuda", dtype=BF) for _ in range(2))
    slots = torch.arange(4, device="cuda", dtype=torch.int32)
    y = rotary.qk_rope_cache(part, pos, table, kc, vc, slots, 2, 1, D)
    assert y[1, 3 * D + 2] == float("inf") and y[2, 3 * D + 5] == float("-inf") and torch.isnan(y[3, 3 * D + 7])
    assert torch.isfinite(y).sum() == y.numel() - 3 and torch.equal(vc.view(4, D).view(torch.int16), y[:, 3 * D :].view(torch.int16))


@pytest.mark.parametrize("D,R", [(64, 32), (24, 10)])
def test_position_outside_the_table(D, R):
    x, dy, qw, kw, pos, table, *_ = make(6, 2, 1, D, R, BF, max_pos=16)
    pos[1], pos[4] = -1, 16
    x = x.requires_grad_()
    y = rotary.rotary(x, pos, table, 3, D)
    (d,) = torch.autograd.grad(y, x, dy)
    for t in (y, d):
        nan = torch.isnan(t.view(6, 4, D))
        assert nan[[1, 4], :3, :R].all() and not nan[[1, 4], :3, R:].any() and not nan[:, 3].any() and not nan[[0, 2, 3, 5]].any()


@pytest.mark.parametrize("T,D,R,inter", [(4, 40, 12, False), (9000, 40, 12, False), (9000, 40, 12, True), (9000, 64, 32, False)])
def test_infinities_behind_the_rotated_part_stay_where_they_are(T, D, R, inter):
    x, _, _, _, pos, table, *_ = make(T, 3, 1, D, R, BF)
    at = torch.zeros_like(x, dtype=torch.bool).view(T, 5, D)
    at[::2, :4, R], at[1::2, :4, R + 3] = True, True
    x.view(T, 5, D)[at] = float("inf")
    y = rotary.rotary(x, pos, table, 4, D, interleaved=inter)
    assert torch.equal(y.view(T, 5, D)[..., R:], x.view(T, 5, D)[..., R:]) and torch.isfinite(y.view(T, 5, D)[..., :R]).all()


def test_empty_batch_and_infinities_pass_through():
    x, dy, qw, kw, pos, table, *_ = make(4, 2, 1, 64, 32, BF)
    e = x[:0].detach().requires_grad_()
    q, k = (w.detach().requires_grad_() for w in (qw, kw))
    y = rotary.qk_norm_rope(e, q, k, pos[:0], table, 2, 1, 64, 1e-6)
    gs = torch.autograd.grad(y, (e, q, k), dy[:0])
    assert y.shape == x[:0].shape and not gs[1].any() and not gs[2].any()
    x[0, 40] = float("inf")  # behind the rotated part of head 0
    x[1, 200] = float("nan")  # a value head
    y = rotary.rotary(x, pos, table, 3, 64)
    assert torch.isinf(y[0, 40]) and torch.isfinite(y[0, :40]).all() and torch.isnan(y[1, 200]) and torch.isfinite(y[1, :200]).all()


def test_capture_replays_on_new_data_beside_other_streams():
    T, nq, nkv, D = 333, 8, 2, 128
    x, dy, qw, kw, pos, table, *_ = make(T, nq, nkv, D, D, BF)
    kc, vc = (torch.zeros(32, 16, nkv, D, device="cuda", dtype=BF) for _ in range(2))
    slots = torch.arange(T, device="cuda", dtype=torch.int32)
    xs = x.clone().requires_grad_()
    q, k = (w.clone().requires_grad_() for w in (qw, kw))

    def step():
        y = rotary.qk_norm_rope(xs, q, k, pos, table, nq, nkv, D, 1e-6)
        gs = torch.autograd.grad(y, (xs, q, k), dy)
        with torch.no_grad():
            z = rotary.qk_rope_cache(xs.detach(), pos, table, kc, vc, slots, nq, nkv, D, q_norm=qw, k_norm=kw)
        return [y.detach(), *gs, z]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    new = torch.randn(T, x.shape[1], device="cuda").to(BF)
    with torch.no_grad():
        xs.copy_(new)
    graph.replay()
    got = [o.clone() for o in out] + [kc.clone(), vc.clone()]
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.current_stream())
        want = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want + [kc, vc]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lens,starts,bs,width,extra", LAYOUTS)
def test_layout(lens, starts, bs, width, extra):
    got, want = layout_case(lens, starts, bs, width, extra, device="cuda")
    for g, w in zip(got, want):
        assert g.dtype == torch.int32 and g.tolist() == w


@pytest.mark.parametrize("B,longest,bs", [(700, 90, 16), (3, 20000, 32), (1, 5000, 8)])
def test_layout_of_many_and_long_sequences(B, longest, bs):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    lens[0] = longest
    starts = [int(n * float(torch.rand((), generator=g))) if i % 2 else 0 for i, n in enumerate(lens)]
    width = longest // bs + 1
    tables = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32)
    total = sum(n - s for n, s in zip(lens, starts)) + 7
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    wide = torch.cat([tables, tables], 1).cuda()[:, :width]  # rows of a wider table
    got = attention.paged_layout(wide, i32(lens), bs, total, starts=i32(starts))
    for a, b in zip(got, layout_oracle(tables.tolist(), lens, starts, bs, total)):
        assert a.tolist() == b
