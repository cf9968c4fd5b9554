"""bq_lora against the definition in 64 bits.

Tolerance.  Products are exact (bf16 adapters times int8 codes, or times parts that sum to all
24 bits of an fp32 value), sums fp32.  An addition is off by at most 2^-24 of the running sum,
which is at most S = sum |a_k x_k|; n additions of independent roundings stay within
8 sqrt(n) 2^-24 S (eight standard deviations of roundings uniform in half a step would be less).
With n = K for t and 3 rank for B t:
  |y - ref| <= |scale| sum_j |b_j| (8 sqrt(K) 2^-24 S_j + 8 sqrt(3 rank) 2^-24 |t_j|) + 2^-23 (|base| + |ref|)
"""
import ctypes
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
NAN = float("nan")
EPS = 2.0 ** -24


def _rand(seed, *shape):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal(shape).astype(np.float32))


def _rows_of(kind, x):
    """What the call takes of x (fp32, CPU), and what it stands for in 64 bits."""
    if kind == "q8":
        g = x.reshape(x.shape[0], -1, 32)
        d = g.abs().amax(-1) * (1 / 127)
        inv = torch.where(d > 0, 1 / d, torch.zeros(()))
        q = (g * inv[..., None]).round().clamp(-127, 127).to(torch.int8).reshape(x.shape)
        return (q.cuda(), d.cuda()), q.double() * d.double().repeat_interleave(32, 1)
    x = x.to(torch.bfloat16 if kind == "bf16" else torch.float32)
    return x.cuda(), x.double()


def _reference(x, a, b, base, adapter, scale, n):
    """(y, tolerance) of one part, fp64."""
    K, rank = x.shape[1], a.shape[1]
    y = torch.zeros((x.shape[0], b.shape[1]), dtype=torch.float64) if base is None else base.double().clone()
    tol = 2.0 ** -23 * y.abs()
    for i in range(n):
        at = torch.nonzero(adapter == i)[:, 0]
        if len(at) == 0:
            continue
        A, B, s = a[i].double(), b[i].double(), 1.0 if scale is None else float(scale[i].double())
        t, S = x[at] @ A.T, x[at].abs() @ A.abs().T
        d = s * (t @ B.T)
        y[at] += d
        tol[at] += abs(s) * ((8 * math.sqrt(K) * EPS * S + 8 * math.sqrt(3 * rank) * EPS * t.abs()) @ B.abs().T) + 2.0 ** -23 * y[at].abs()
    return y, tol


def _lora(bq, rows, K, Ns, rank, n, kind, seed=1, adapter=None, scaled=True, base="y", pad=0, run=None):
    rng = np.random.default_rng(seed)
    if adapter is None:
        adapter = rng.integers(0, n, rows)
    adapter = torch.as_tensor(np.asarray(adapter), dtype=torch.int32)
    print(f"lora rows {rows} K {K} N {Ns} rank {rank} adapters {n} {kind} base {base} pad {pad}", flush=True)
    x = _rand(seed, rows, K)
    if pad and kind != "q8":
        wide = torch.full((rows, K + pad), NAN)
        wide[:, :K] = x
        gx, rx = _rows_of(kind, wide)
        gx, rx = gx[:, :K], rx[:, :K]
    else:
        gx, rx = _rows_of(kind, x)
    scale = _rand(seed + 1, n) if scaled else None
    parts, want = [], []
    for i, N in enumerate(Ns):
        a, b = (_rand(seed + 10 + i, n, rank, K) / K ** 0.5).bfloat16(), _rand(seed + 20 + i, n, N, rank).bfloat16()
        y0 = _rand(seed + 30 + i, rows, N)
        y = torch.full((rows, N + pad), NAN, device="cuda")
        if base == "y":
            y[:, :N] = y0.cuda()
            part = (a.cuda(), b.cuda(), y[:, :N])
        elif base == "other":
            z = torch.full((rows, N + 2 * pad), NAN, device="cuda")
            z[:, :N] = y0.cuda()
            part = (a.cuda(), b.cuda(), y[:, :N], z[:, :N])
        else:
            part = (a.cuda(), b.cuda(), y[:, :N], None)
        parts.append(part)
        want.append((y, y0, _reference(rx, a, b, y0 if base else None, adapter, scale, n)))
    op = bq.Lora(gx, adapter.cuda(), parts, scale=None if scale is None else scale.cuda())
    op.work.view(torch.float32).fill_(NAN)
    op.run()
    torch.cuda.synchronize()
    for i, (y, y0, (ref, tol)) in enumerate(want):
        N = Ns[i]
        got = y[:, :N].cpu().double()
        if pad:
            assert torch.isnan(y[:, N:]).all()
        assert torch.isfinite(got).all()
        err = (got - ref).abs()
        print(f"  part {i}: worst error / tolerance {(err / tol.clamp(min=1e-30)).max().item():.3f}", flush=True)
        assert (err <= tol).all(), i
        none = (adapter < 0) | (adapter >= n)
        if none.any():  # what has no adapter is the base, bit for bit
            assert torch.equal(y[:, :N].cpu()[none], y0[none] if base else torch.zeros_like(y0[none]))
    return op, parts


@pytest.mark.parametrize("kind", ["q8", "f32", "bf16"])
@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 72, 256])
def test_ranks(bq, kind, rank):
    _lora(bq, 5, 256, [48], rank, 3, kind, seed=rank)


@pytest.mark.parametrize("kind", ["q8", "f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 33, 255, 256, 257, 300, 1000])
def test_rows(bq, kind, rows):
    """One row to several tiles, either side of where the rows of an adapter are found otherwise; adapters anywhere."""
    _lora(bq, rows, 96, [272, 16], 16, 5, kind, seed=rows)


@pytest.mark.parametrize("rows", [40, 400])
def test_rows_of_one_adapter_and_of_none(bq, rows):
    """All rows with one adapter; none with any; runs; slots outside the pool are none."""
    for adapter in (np.full(rows, 2), np.full(rows, -1), np.repeat([3, -1, 0, 7, 1], rows // 5), np.arange(rows) % 9 - 3):
        for base in ("y", "other", None):
            _lora(bq, rows, 64, [80, 32], 8, 4, "q8", seed=rows, adapter=adapter, base=base)


@pytest.mark.parametrize("kind", ["q8", "f32", "bf16"])
@pytest.mark.parametrize("K", [32, 64, 160, 1056, 9216])
def test_widths(bq, kind, K):
    _lora(bq, 9, K, [16, 4096, 528, 240], 16, 4, kind, seed=K)
    _lora(bq, 270, K, [1040], 32, 2, kind, seed=K + 1, adapter=np.repeat([1, 0], 135))


@pytest.mark.parametrize("kind", ["q8", "f32", "bf16"])
def test_strides_and_bases(bq, kind):
    for rows in (7, 290):
        for base in ("y", "other", None):
            _lora(bq, rows, 128, [64, 144], 24, 3, kind, seed=rows, base=base, pad=8)
    _lora(bq, 7, 128, [64], 24, 3, kind, scaled=False)


def test_values_of_any_size(bq):
    """fp32 rows whose values are 2^40 apart, and rows of NaN beside others: each row is its own."""
    for rows in (20, 300):
        K, N, rank, n = 128, 64, 16, 2
        x = _rand(3, rows, K) * torch.exp2(torch.arange(rows, dtype=torch.float32)[:, None] % 41 - 20)
        x[:, ::7] *= 2.0 ** 20
        bad = torch.arange(rows) % 9 == 4
        x[bad] = NAN
        a, b = (_rand(4, n, rank, K)).bfloat16(), _rand(5, n, N, rank).bfloat16()
        adapter = torch.arange(rows) % 2
        y = torch.zeros((rows, N), device="cuda")
        bq.Lora(x.cuda(), adapter.int().cuda(), [(a.cuda(), b.cuda(), y)]).run()
        ref, tol = _reference(x.double(), a, b, None, adapter, None, n)
        got = y.cpu().double()
        assert torch.isnan(got[bad]).all()
        assert ((got - ref).abs() <= tol)[~bad].all()


def test_offsets_past_32_bits(bq):
    """An adapter more than 2^32 bytes into its pool."""
    K, N, rank, n = 8192, 64, 256, 1030
    a = torch.zeros((n, rank, K), dtype=torch.bfloat16, device="cuda")
    b = torch.zeros((n, N, rank), dtype=torch.bfloat16, device="cuda")
    a[n - 1], b[n - 1] = 1.0, 2.0
    x = torch.ones((3, K), device="cuda")
    y = torch.zeros((3, N), device="cuda")
    bq.Lora(x, torch.tensor([n - 1, 0, n - 2], dtype=torch.int32, device="cuda"), [(a, b, y)]).run()
    assert (y[0] == 2.0 * rank * K).all() and (y[1:] == 0).all()   # powers of two: exact


def test_captured_and_replayed(bq):
    """The rows' adapters, the rows and the scales change between replays of one graph; equal calls give equal bits."""
    for rows in (12, 300):
        K, N, rank, n = 256, 96, 16, 6
        a, b = (_rand(6, n, rank, K) / 16).bfloat16(), _rand(7, n, N, rank).bfloat16()
        x, base = torch.zeros((rows, K), device="cuda"), torch.zeros((rows, N), device="cuda")
        adapter = torch.zeros(rows, dtype=torch.int32, device="cuda")
        scale, y, z = torch.zeros(n, device="cuda"), torch.zeros((rows, N), device="cuda"), torch.zeros((rows, N), device="cuda")
        ga, gb = a.cuda(), b.cuda()
        op = bq.Lora(x, adapter, [(ga, gb, y, base)], scale=scale)
        again = bq.Lora(x, adapter, [(ga, gb, z, base)], scale=scale)
        op.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            op.run()
        for step in range(4):
            hx, hb, hs = _rand(40 + step, rows, K), _rand(50 + step, rows, N), _rand(60 + step, n)
            ha = torch.from_numpy(np.random.default_rng(step).integers(-1, n, rows).astype(np.int32))
            for g, h in ((x, hx), (base, hb), (scale, hs), (adapter, ha)):
                g.copy_(h)
            y.fill_(NAN)
            op.work.view(torch.float32).fill_(NAN)
            graph.replay()
            again.run()
            torch.cuda.synchronize()
            ref, tol = _reference(hx.double(), a, b, hb, ha, hs, n)
            assert ((y.cpu().double() - ref).abs() <= tol).all(), (rows, step)
            assert torch.equal(y, z)


def test_two_calls_on_two_streams(bq):
    jobs = []
    for i in range(2):
        a, b = (_rand(70 + i, 4, 16, 512) / 20).bfloat16(), _rand(72 + i, 4, 256, 16).bfloat16()
        x, base = _rand(74 + i, 200, 512), _rand(76 + i, 200, 256)
        adapter = torch.arange(200) * (3 + i) % 4
        y = torch.zeros((200, 256), device="cuda")
        jobs.append((bq.Lora(x.cuda(), adapter.int().cuda(), [(a.cuda(), b.cuda(), y, base.cuda())]), y,
                     _reference(x.double(), a, b, base, adapter, None, 4), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        for op, _, _, st in jobs:
            with torch.cuda.stream(st):
                op.run()
    torch.cuda.synchronize()
    for _, y, (ref, tol), _ in jobs:
        assert ((y.cpu().double() - ref).abs() <= tol).all()


def test_refusals(bq):
    rows, K, N, rank, n = 4, 64, 32, 8, 2
    y = torch.full((rows, N), 7.0, device="cuda")
    x, a = torch.zeros((rows, K), device="cuda"), torch.zeros((n, rank, K), dtype=torch.bfloat16, device="cuda")
    b = torch.zeros((n, N, rank), dtype=torch.bfloat16, device="cuda")
    adapter = torch.zeros(rows, dtype=torch.int32, device="cuda")
    op = bq.Lora(x, adapter, [(a, b, y)], scale=torch.ones(n, device="cuda"))
    L, s = bq.load(), op.struct
    call = lambda: L.bq_lora(ctypes.byref(s), None)

    def refused(code, where, **fields):
        keep = {f: getattr(where, f) for f in fields}
        for f, v in fields.items():
            setattr(where, f, v)
        assert call() == code, (fields, call())
        for f, v in keep.items():
            setattr(where, f, v)
    E, U = bq.BQ_EINVAL, bq.BQ_UNSUPPORTED
    for f in (dict(rows=-1), dict(K=0), dict(rank=0), dict(n_adapters=0), dict(n_parts=0), dict(n_parts=5), dict(x_type=13), dict(x=None),
              dict(x=s.x + 4), dict(adapter=None), dict(ldx=K - 4), dict(ldx=K + 2), dict(work=None), dict(work_bytes=s.work_bytes - 4),
              dict(work=s.work + 8), dict(x_type=bq.TYPE_Q8_0), dict(x_type=bq.TYPE_BF16, ldx=K + 4)):
        refused(E, s, **f)
    for f in (dict(K=48), dict(rank=12), dict(rank=264)):
        refused(U, s, **f)
    p = s.parts[0]
    for f in (dict(a=None), dict(b=None), dict(y=None), dict(a=p.a + 2), dict(y=p.y + 4), dict(base=p.base + 4), dict(ldy=N - 4), dict(ldy=N + 2),
              dict(ldbase=N - 4), dict(ldbase=N + 4), dict(N=0)):
        refused(E, p, **f)
    refused(U, p, N=24)
    refused(U, p, N=1 << 26, ldy=1 << 26, ldbase=1 << 26)
    refused(U, s, rows=(1 << 20) + 1)
    s.parts[1] = p
    refused(E, s, n_parts=2)   # two parts that add to the same y
    assert L.bq_lora(None, None) == E
    s.rows = 0
    assert call() == bq.BQ_OK
    torch.cuda.synchronize()
    assert (y == 7.0).all()
    W = L.bq_lora_workspace_bytes
    assert W(rows, rank, 1) == s.work_bytes and W(0, 8, 1) == W(1, 0, 1) == W(1, 264, 1) == W(1, 8, 5) == W(1, 8, 0) == 0


@pytest.mark.parametrize("reader", [0, 1])
def test_base_that_another_part_writes(bq, reader):
    """The parts run side by side: one whose base is another's output would read it before or after it was written."""
    rows, K, N, rank, n = 3, 64, 32, 8, 2
    x, a = torch.zeros((rows, K), device="cuda"), torch.zeros((n, rank, K), dtype=torch.bfloat16, device="cuda")
    b = torch.zeros((n, N, rank), dtype=torch.bfloat16, device="cuda")
    ys = [torch.full((rows, N), 7.0, device="cuda") for _ in range(2)]
    op = bq.Lora(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), [(a, b, ys[0]), (a, b, ys[1])])
    call = lambda: bq.load().bq_lora(ctypes.byref(op.struct), None)
    part, own = op.struct.parts[reader], op.struct.parts[reader].base
    part.base = op.struct.parts[1 - reader].y
    assert call() == bq.BQ_EINVAL
    part.base = own
    assert call() == bq.BQ_OK
    torch.cuda.synchronize()


def _q5(bq, seed, K, N):
    import synth
    raw = torch.from_numpy(synth.quantize_q5k(_rand(seed, N, K).numpy() * 0.05)).cuda()
    rep, rep_min = bq.repack_q5k(raw, K, N)
    return bq.make_weight(raw, bq.TYPE_Q5_K, K, N, rep=rep, rep_min=rep_min)


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_decode_step(bq, rows):
    """The step's projection hook: at every projection of an attention and an FFN block, what the library's hook adds to
    the outputs is the definition's, of the q8 rows that the projection read; behind a step that was captured too."""
    E, A, F, n, rank = 256, 256, 512, 3, 16
    f32 = lambda *s: torch.zeros(s, device="cuda")
    wide = max(E, A, F)
    qkv_n = [A, 128, A]
    weights = [_q5(bq, 80 + i, E, v) for i, v in enumerate(qkv_n)]   # (they hold the tensors, the array does not)
    qkv = (bq.Weight * 3)(*weights)
    o, gate, up, down = _q5(bq, 84, A, E), _q5(bq, 85, E, F), _q5(bq, 86, E, F), _q5(bq, 87, F, E)
    q8 = (torch.zeros(rows * wide, dtype=torch.int8, device="cuda"), f32(rows * wide // 32), torch.zeros(rows * wide // 32, dtype=torch.int32, device="cuda"))
    x, proj, g, u = f32(rows, E), f32(rows, E), f32(rows, F), f32(rows, F)
    outs = [f32(rows, v) for v in qkv_n]
    attn = _rand(88, rows, A).cuda()
    vec = lambda v: torch.full((v,), 0.7, device="cuda")
    vecs = [vec(E), vec(A), vec(F), vec(F)]
    ptr = lambda t: t.data_ptr()
    ys = (ctypes.c_void_p * 3)(*[ptr(t) for t in outs])
    ba, bf = bq.DecodeBlock(), bq.DecodeBlock()
    ba.kind, ba.alpha, ba.qkv, ba.n_qkv, ba.qkv_out = bq.BLOCK_ATTN, ptr(vecs[0]), qkv, 3, ys
    ba.attn_out, ba.attn_gate, ba.sgate, ba.n_attn, ba.o = ptr(attn), ptr(outs[2]), ptr(vecs[1]), A, ctypes.pointer(o)
    bf.kind, bf.alpha, bf.gate, bf.up, bf.down, bf.n_ff = bq.BLOCK_FFN, ptr(vecs[0]), ctypes.pointer(gate), ctypes.pointer(up), ctypes.pointer(down), F
    bf.s_gate, bf.s_up = ptr(vecs[2]), ptr(vecs[3])
    blocks = (bq.DecodeBlock * 2)(ba, bf)
    st = bq.DecodeStep()
    st.n_blocks, st.blocks, st.n_embd, st.rows, st.x, st.proj, st.ffn_g, st.ffn_u = 2, blocks, E, rows, ptr(x), ptr(proj), ptr(g), ptr(u)
    st.xq, st.xd, st.xsum = (ptr(t) for t in q8)
    xdh = torch.zeros((rows, wide // 32), dtype=torch.int16, device="cuda")
    st.xdh = ptr(xdh)

    adapter = torch.from_numpy(np.random.default_rng(90).integers(-1, n, rows).astype(np.int32))
    ga = adapter.cuda()

    def lora(seed, K, targets):
        xq, xd = q8[0][: rows * K].view(rows, K), q8[1][: rows * K // 32].view(rows, K // 32)
        return bq.Lora((xq, xd), ga, [((_rand(seed + i, n, rank, K) / 16).bfloat16().cuda(), _rand(seed + 5 + i, n, y.shape[1], rank).bfloat16().cuda(), y)
                                      for i, y in enumerate(targets)])
    ops = {(0, bq.PROJ_QKV): lora(100, E, outs), (0, bq.PROJ_O): lora(120, A, [proj]), (1, bq.PROJ_GATE_UP): lora(140, E, [g, u]),
           (1, bq.PROJ_DOWN): lora(160, F, [proj])}
    plan = bq.LoraPlan([{k[1]: v for k, v in ops.items() if k[0] == b} for b in (0, 1)])
    L, seen = bq.load(), []

    def hook(user, block, proj_, stream):
        op = ops[block, proj_]
        xq, xd = op._keep[0], op._keep[1]
        before = [p[2].clone() for p in op._keep[3]]
        seen.append((op, xq.cpu().double() * xd.cpu().double().repeat_interleave(32, 1), [t.cpu() for t in before]))
        L.bq_lora_hook(user, block, proj_, stream)
        seen[-1] += ([p[2].cpu().double() for p in op._keep[3]],)
    cb = bq.PROJ_HOOK(hook)
    st.projected, st.projected_user = cb, ctypes.addressof(plan.struct)
    start = _rand(89, rows, E).cuda()

    def run(f):
        x.copy_(start)
        bq.norm_q8("norm", rows, E, out=x, a=x, q8=q8)
        f()
        torch.cuda.synchronize()
        plan.check()
        return x.clone()
    first = run(lambda: bq.decode_enqueue(st))
    assert [id(s[0]) for s in seen] == [id(ops[k]) for k in ((0, bq.PROJ_QKV), (0, bq.PROJ_O), (1, bq.PROJ_GATE_UP), (1, bq.PROJ_DOWN))]
    for op, xr, before, after in seen:
        for (a, b, _), y0, y1 in zip(op._keep[3], before, after):
            ref, tol = _reference(xr, a.cpu(), b.cpu(), y0, adapter, None, n)
            worst = ((y1 - ref).abs() / tol).max().item()
            assert worst <= 1, worst
    # the library's hook by itself, eager and captured
    plan.install(st)
    assert torch.equal(run(lambda: bq.decode_enqueue(st)), first)
    graph = bq.DecodeGraph(st)
    for _ in range(3):
        assert torch.equal(run(graph.launch), first)
    # without adapters the step gives something else; with adapters of none what it gives without the hook
    ga.fill_(-1)
    none = run(lambda: bq.decode_enqueue(st))
    st.projected = bq.PROJ_HOOK()
    assert torch.equal(run(lambda: bq.decode_enqueue(st)), none) and (not (adapter >= 0).any() or not torch.equal(none, first))
    plan.install(st)
    if rows == 1:
        st.fold = 1
        with pytest.raises(bq.BqError) as e:
            bq.decode_enqueue(st)
        assert e.value.code == bq.BQ_UNSUPPORTED
    bad = bq.LoraPlanStruct(1, plan._blocks, 0)
    L.bq_lora_hook(ctypes.byref(bad), 1, 0, None)
    assert bad.status == bq.BQ_EINVAL
