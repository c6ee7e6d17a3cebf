"""The token-transformer operators (musev_amd.token_ops): refusals and plans on the CPU; with -m gpu every kernel against its definition in
64 bits.  u below is the half step of the output type (fp16 2^-11, bf16 2^-8, relative); the bounds are elementwise and derived beside
each oracle."""
import math
import os
import random
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]
IDS = ["fp16", "bf16"]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def subnormal(dt):
    """absolute half step below the normal range"""
    return torch.finfo(dt).tiny * torch.finfo(dt).eps / 2


def rnd(shape, seed, dt, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dt).to(DEV)


def within(got, want, bound, what=""):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.numel():
        return
    assert bool(torch.isfinite(got).all()), (what, "not finite")
    over = (got - want).abs() - bound
    at = int(over.argmax())
    assert over.max().item() <= 0, (what, f"element {at}: got {got.flatten()[at].item()}, want {want.flatten()[at].item()}, "
                                    f"bound {bound.flatten()[at].item()}, {int((over > 0).sum())} over")


# ---- on the CPU: the ABI, plans and refusals -----------------------------------------------------------------------------------
def test_every_declared_symbol_is_exported_and_bound():
    from musev_amd import _lib
    lib = _lib.load()
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "musev_tokens.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(mv_[a-z0-9_]+)\s*\(", hdr))
    assert names == set(_lib.TOKEN_SIGNATURES)
    for n in names:
        assert hasattr(lib, n), n
    assert lib.mv_tokens_abi_version() == _lib.MV_TOKENS_ABI_VERSION


def test_operators_are_public():
    from musev_amd import ops, token_ops
    for n in token_ops.__all__:
        assert getattr(ops, n) is getattr(token_ops, n) and n in ops.__all__


def test_entry_points_refuse_without_a_gpu():
    import ctypes as C
    from musev_amd import _lib
    lib = _lib.load()

    def refused(rc, text):
        assert rc == -1 and text in lib.mv_last_error(), (rc, lib.mv_last_error())
    for fn in (lib.mv_attention_packed, lib.mv_rotary_axes, lib.mv_gated_residual_norm, lib.mv_gemm_i8, lib.mv_linear_i8):
        refused(fn(None, None), b"null descriptor")
    a = _lib.AttnPackedDesc()
    a.q = a.k = a.v = a.out = a.items = 16
    a.n_items, a.heads, a.kv_heads, a.d, a.scale = 1, 4, 2, 64, 0.125
    a.ldq = a.ldo = 256
    a.ldk = a.ldv = 128
    for name, bad, text in (("d", 12, b"head dim"), ("d", 136, b"head dim"), ("kv_heads", 3, b"heads"), ("dtype", 2, b"element type"),
                            ("n_items", -1, b"items"), ("q", 0, b"null"), ("k", 8, b"aligned"), ("ldv", 132, b"aligned"), ("ldk", 1 << 24, b"stride"),
                            ("n_joins", 1, b"workspace"), ("scale", float("nan"), b"scale"), ("scale", 2e6, b"scale")):
        old = getattr(a, name)
        setattr(a, name, bad)
        refused(lib.mv_attention_packed(C.byref(a), None), text)
        setattr(a, name, old)
    assert lib.mv_attention_packed_workspace_bytes(-1, 1, 64) == -1 and lib.mv_attention_packed_workspace_bytes(3, 2, 64) == 3 * 2 * 66 * 4
    r = _lib.RotaryDesc()
    r.q = r.out_q = r.positions = r.turns = r.axis = 16
    r.tokens, r.heads, r.kv_heads, r.d, r.pairs, r.axes = 4, 2, 2, 64, 32, 1
    for name, bad, text in (("pairs", 33, b"pairs"), ("heads", 0, b"heads"), ("dtype", 7, b"element type"), ("turns", 0, b"null")):
        old = getattr(r, name)
        setattr(r, name, bad)
        refused(lib.mv_rotary_axes(C.byref(r), None), text)
        setattr(r, name, old)
    n = _lib.GatedNormDesc()
    n.x = n.f = n.stream_out = 16
    n.rows, n.groups, n.c = 4, 1, 64
    for name, bad, text in (("c", 0, b"columns"), ("c", 16385, b"columns"), ("groups", 0, b"groups"), ("rows", -1, b"rows"), ("x", 0, b"null")):
        old = getattr(n, name)
        setattr(n, name, bad)
        refused(lib.mv_gated_residual_norm(C.byref(n), None), text)
        setattr(n, name, old)
    g = _lib.GemmI8Desc()
    g.a = g.w = g.a_scale = g.w_scale = g.out = 16
    g.M, g.N, g.kp, g.lda, g.ldw, g.ldo = 4, 8, 128, 128, 128, 8
    for name, bad, text in (("kp", 64, b"kp"), ("kp", 131200, b"kp"), ("lda", 64, b"lda"), ("N", 0, b"N 0"), ("act", 5, b"activation"), ("w", 8, b"aligned")):
        old = getattr(g, name)
        setattr(g, name, bad)
        refused(lib.mv_gemm_i8(C.byref(g), None), text)
        setattr(g, name, old)
    ln = _lib.LinearI8Desc()
    ln.x = ln.w = ln.w_scale = ln.out = ln.workspace = 16
    ln.M, ln.N, ln.K, ln.kp, ln.ldx, ln.ldw, ln.ldo = 4, 8, 100, 128, 100, 128, 8
    for name, bad, text in (("kp", 256, b"kp"), ("K", 0, b"K 0"), ("x", 0, b"null"), ("w", 8, b"aligned"), ("act", 3, b"activation"), ("dtype", 2, b"element type"),
                            ("ldw", 64, b"ldw"), ("N", 0, b"N 0")):
        old = getattr(ln, name)
        setattr(ln, name, bad)
        refused(lib.mv_linear_i8(C.byref(ln), None), text)
        setattr(ln, name, old)
    ln.M, ln.workspace = 17, 0
    refused(lib.mv_linear_i8(C.byref(ln), None), b"workspace")
    refused(lib.mv_quantize_rows_i8(16, 64, 4, 64, 0, 16, 64, 16, None), b"code rows")
    refused(lib.mv_quantize_rows_i8(16, 64, 4, 0, 0, 16, 128, 16, None), b"131071")


def _cover(items, joins, ws_rows, ql, kl, group, causal):
    """every packed row's every visible key is walked by exactly one item, the parts of a row are joined for exactly that row, and no two
    parts share workspace rows"""
    want, q_at, k_at = set(), 0, 0
    for q, kv in zip(ql, kl):
        for m0 in range(0, q * group, 128):
            want.add((q_at, q, k_at, kv, m0))
        q_at, k_at = q_at + q, k_at + kv
    tiles = {}
    for it in items:
        tiles.setdefault(tuple(it[:5]), []).append(it)
    assert set(tiles) == want
    joined = {(j[0], j[1], j[2], j[3]): j for j in joins}
    assert len(joined) == len(joins)
    used = set()
    for key, items in tiles.items():
        q_row, q, k_row, kv, m0 = key
        rows = min(128, q * group - m0)
        last = (m0 + rows - 1) // group
        vis = kv if not causal else max(0, min(kv, last + kv - q + 1))
        items.sort(key=lambda i: i[5])
        assert items[0][5] == 0 and items[-1][6] == vis and all(a[6] == b[5] for a, b in zip(items, items[1:]))
        if len(items) == 1:
            assert items[0][7] == -1 and (q_row, q, kv, m0) not in joined
            continue
        j = joined.pop((q_row, q, kv, m0))
        assert j[5] == len(items) and j[6] == rows
        for s, it in enumerate(items):
            assert it[7] == j[4] + s * rows and it[5] < it[6] and it[5] % 64 == 0
            mine = set(range(it[7], it[7] + rows))
            assert not (mine & used)
            used |= mine
    assert not joined and used == set(range(ws_rows))


@pytest.mark.parametrize("seed", range(12))
def test_plan_covers_every_visible_key_once(seed):
    r = random.Random(seed)
    from musev_amd import token_ops as to
    for causal in (False, True):
        n = r.randint(1, 12)
        one = r.random() < 0.4
        ql = [1 if one else r.choice([0, 1, 2, 31, 33, 127, 128, 129, 700]) for _ in range(n)]
        kl = [r.choice([0, 1, 63, 64, 65, 500, 5000, 20000]) for _ in range(n)]
        kvh, group = r.choice([1, 2, 8]), r.choice([1, 3, 4, 8])
        plan = to.attention_plan(ql, kl, heads=kvh * group, kv_heads=kvh, d=64, causal=causal, device="cpu")
        items, joins = (t.tolist() for t in plan._tensors)
        d = plan
        assert len(items) == d.n_items and len(joins) == d.n_joins and d.join_rows == max((j[6] for j in joins), default=0)
        _cover(items, joins, d.ws_rows, ql, kl, group, causal)
        from musev_amd import _lib
        assert plan._workspace == _lib.load().mv_attention_packed_workspace_bytes(d.ws_rows, kvh, 64)


@pytest.mark.parametrize("ql,kl,group,kvh,d,split", [([300] * 4, [300] * 4, 1, 8, 64, False), ([700] * 3, [700] * 3, 4, 2, 64, False), ([1], [8192], 4, 8, 128, True),
                                                     ([128], [8192], 1, 8, 128, True), ([1500], [1500], 4, 1, 128, True), ([16] * 8, [2000] * 8, 4, 2, 128, True),
                                                     ([1], [100], 1, 1, 64, False), ([0, 3], [50, 0], 1, 1, 64, False)])
@pytest.mark.parametrize("causal", [False, True])
def test_plan_splits_where_the_parts_pay(ql, kl, group, kvh, d, split, causal):
    from musev_amd import token_ops as to
    items, joins, ws = to._plan_items(ql, kl, group, kvh, causal, d)
    assert bool(joins) == split
    _cover(items, joins, ws, ql, kl, group, causal)


LATE = {   # lengths, heads per key / value head, key / value heads, causal -> tiles that are split
    "few_late": ([6000], [6000], 1, 12, False, 5),
    "many_late": ([13312], [13312], 1, 8, False, 40),
    "two_lengths": ([13312, 5121], [13312, 5121], 1, 16, False, 8),
    "one_key_head": ([1100], [9000], 64, 1, False, 38),
    "late_but_short": ([3000] * 4, [3000] * 4, 1, 8, False, 0),
    "balanced": ([16384], [16384], 4, 4, True, 0),
    "too_many_rounds": ([70000], [3000], 1, 8, False, 0),
    "heads_beyond_the_blocks": ([200], [2100], 1, 600, False, 0),
}


@pytest.mark.parametrize("name", list(LATE))
def test_plan_splits_the_blocks_that_would_run_late(name):
    """the parts cover every key once; the longest items come first"""
    from musev_amd import token_ops as to
    ql, kl, group, kvh, causal, split = LATE[name]
    items, joins, ws = to._plan_items(ql, kl, group, kvh, causal)
    assert len(joins) == split
    _cover(items, joins, ws, ql, kl, group, causal)
    assert all(a[6] - a[5] >= b[6] - b[5] for a, b in zip(items, items[1:]))


def test_plan_refusals():
    from musev_amd import ops
    ok = dict(heads=4, kv_heads=2, d=64, device="cpu")
    for bad, match in ((dict(ok, heads=5), "heads"), (dict(ok, kv_heads=0), "heads"), (dict(ok, d=60), "head dim"), (dict(ok, d=136), "head dim"),
                       (dict(ok, scale=float("inf")), "scale")):
        with pytest.raises(ValueError, match=match):
            ops.attention_plan([3], **bad)
    for q, kv, match in (([], None, "length"), ([-1], None, "length"), ([1, 2], [3], "lengths"), ([2 ** 31], None, "rows"), ([2 ** 30], None, "rows")):
        with pytest.raises(ValueError, match=match):
            ops.attention_plan(q, kv, **ok)
    with pytest.raises(ValueError, match="sections"):
        ops.rotary_table([3], device="cpu")
    with pytest.raises(ValueError, match="theta"):
        ops.rotary_table([4], theta=0.0, device="cpu")


def test_tensors_off_the_gpu_are_refused():
    from musev_amd import ops
    x = torch.zeros(4, 64, dtype=torch.float16)
    plan = ops.attention_plan([4], heads=1, d=64, device="cpu")
    table = ops.rotary_table([64], device="cpu")
    for call in (lambda: ops.attention_packed(plan, x, x, x), lambda: ops.rotary_axes(x, None, torch.zeros(4, 1), table, heads=1, d=64),
                 lambda: ops.gated_residual_norm(x, x), lambda: ops.quantize_rows_i8(x),
                 lambda: ops.pack_weight_i8(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_plan_takes_integers_only():
    import numpy as np
    from musev_amd import ops
    ok = dict(heads=2, d=64, device="cpu")
    assert ops.attention_plan(np.array([3, 4]), torch.tensor([5, 6]), **ok).kv_lens == (5, 6)
    with pytest.raises(TypeError):
        ops.attention_plan([3.5], **ok)


@pytest.fixture
def on_cpu(monkeypatch):
    """argument checks alone: CPU tensors pass for device memory and no launch may follow"""
    from musev_amd import token_ops as to
    monkeypatch.setattr(to, "_on_gpu", lambda t: True)

    class Launched(Exception):
        pass

    def load():
        raise Launched
    monkeypatch.setattr(to._lib, "load", load)

    monkeypatch.setattr(to, "_current_device", lambda: -1)    # (what get_device() says of a CPU tensor)
    monkeypatch.setattr(to, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(to._Held, "_use", lambda self, s: None)
    return Launched


def test_refusals_of_attention(on_cpu):
    from musev_amd import ops
    plan = ops.attention_plan([3, 5], heads=4, kv_heads=2, d=16, device="cpu")
    q, kv = torch.zeros(8, 64, dtype=torch.float16), torch.zeros(8, 32, dtype=torch.float16)
    with pytest.raises(on_cpu):
        ops.attention_packed(plan, q, kv, kv)
    big = torch.zeros(8, 256, dtype=torch.float16)
    with pytest.raises(on_cpu):   # (columns of one matrix, apart)
        ops.attention_packed(plan, big[:, :64], big[:, 64:96], big[:, 96:128], out=big[:, 128:192])
    for args, kw, match in (((q[:7], kv, kv), {}, "q"), ((q, kv[:7], kv), {}, "k"), ((q, kv, kv[:, :16]), {}, "v"), ((q[:, :32], kv, kv), {}, "q"),
                            ((q, kv.bfloat16(), kv), {}, "k"), ((q.float(), kv, kv), {}, "q"), ((q.t().contiguous().t(), kv, kv), {}, "unit inner"),
                            ((q, kv, kv), {"out": q}, "overlaps"), ((big[:, :64], kv, kv), {"out": big[:, 32:96]}, "overlaps"),
                            ((q, kv, kv), {"out": torch.zeros(7, 64, dtype=torch.float16)}, "out"),
                            ((big[:, 4:68], kv, kv), {}, "16"), ((q, kv, kv), {"out": torch.zeros(8, 300, dtype=torch.float16)[:, 8:72]}, "16"), ((q, torch.zeros(8, 36, dtype=torch.float16)[:, :32], kv), {}, "16")):
        with pytest.raises(ValueError, match=match):
            ops.attention_packed(plan, *args, **kw)


def test_tensors_that_require_gradients_are_refused(on_cpu):
    from musev_amd import ops
    x = torch.zeros(6, 64, dtype=torch.float16)
    p = torch.zeros(64, dtype=torch.float16, requires_grad=True)
    r = torch.zeros(6, 64, dtype=torch.float16, requires_grad=True)
    plan, table = ops.attention_plan([6], heads=1, d=64, device="cpu"), ops.rotary_table([64], device="cpu")
    w = ops.Int8Rows(torch.zeros(64, 128, dtype=torch.int8), torch.ones(64), 64)
    pos = torch.zeros(6, 1)
    for call in (lambda: ops.attention_packed(plan, x, r, x), lambda: ops.rotary_axes(r, None, pos, table, heads=1, d=64),
                 lambda: ops.gated_residual_norm(x, r), lambda: ops.gated_residual_norm(x, x, pre=(p, None, 1e-6)), lambda: ops.linear_i8(r, w),
                 lambda: ops.linear_i8(x, w, bias=p)):
        with pytest.raises(ValueError, match="gradients"):
            call()
        with torch.no_grad(), pytest.raises(on_cpu):
            call()


def test_refusals_of_rotary(on_cpu):
    from musev_amd import ops
    table = ops.rotary_table([8, 8], device="cpu")
    q, k, pos = torch.zeros(6, 64, dtype=torch.bfloat16), torch.zeros(6, 32, dtype=torch.bfloat16), torch.zeros(6, 2, dtype=torch.int32)
    kw = dict(heads=4, kv_heads=2, d=16)
    with pytest.raises(on_cpu):
        ops.rotary_axes(q, k, pos, table, **kw, out_q=q, out_k=k)
    for args, more, match in (((q, k, pos.long(), table), {}, "int32"), ((q, k, pos[:5], table), {}, "positions"), ((q, k, pos[:, :1], table), {}, "positions"),
                              ((q, k[:5], pos, table), {}, "k"), ((q, k, pos, ops.rotary_table([20], device="cpu")), {}, "elements"),
                              ((q, k, pos, table), {"pairing": "x"}, "pairing"), ((q, k, pos, table), {"heads": 3}, "q"),
                              ((q, None, pos, table), {"out_k": k}, "out_k"), ((q, k, pos, table), {"out_q": q[:5]}, "out_q"),
                              ((q, q[:, :32], pos, table), {"out_k": q[:, 16:48]}, "overlaps")):
        with pytest.raises(ValueError, match=match):
            ops.rotary_axes(*args, **{**kw, **more})


def test_refusals_of_the_gated_norm(on_cpu):
    from musev_amd import ops
    x, f, g = torch.zeros(6, 40, dtype=torch.float16), torch.zeros(6, 40, dtype=torch.float16), torch.zeros(3, 40, dtype=torch.float16)
    pre = (None, None, 1e-6)
    for kw in (dict(pre=pre, gate=g, rows_per_group=2), dict(out=x, pre=pre, norm_out=f), dict(gate=g[:1])):
        with pytest.raises(on_cpu):
            ops.gated_residual_norm(x, f, **kw)
    idx = torch.zeros(6, dtype=torch.int32)
    for kw, match in ((dict(kind="batch"), "kind"), (dict(scale=g, rows_per_group=2), "pre"), (dict(gate=g), "groups"), (dict(gate=g, rows_per_group=1), "cover"),
                      (dict(gate=g, rows_per_group=2, group_index=idx), "both"), (dict(gate=g, group_index=idx.long()), "int32"),
                      (dict(group_index=idx), "without"), (dict(gate=g[:, :8]), "gate"), (dict(gate=g, pre=pre, scale=g[:2], rows_per_group=3), "scale"),
                      (dict(pre=(x[0, :8], None, 1e-6)), "gamma"), (dict(pre=pre, out=x, norm_out=x), "overlaps"), (dict(out=g), "out")):
        with pytest.raises(ValueError, match=match):
            ops.gated_residual_norm(x, f, **kw)
    with pytest.raises(ValueError, match="f"):
        ops.gated_residual_norm(x, f[:5])
    wide = torch.zeros(1, 16385, dtype=torch.float16)
    with pytest.raises(ValueError, match="columns"):
        ops.gated_residual_norm(wide, wide)


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["pre", "post"])
def test_the_gated_norm_refuses_an_eps_that_is_none(on_cpu, which, eps):
    from musev_amd import ops
    x, f = torch.zeros(6, 40, dtype=torch.float16), torch.zeros(6, 40, dtype=torch.float16)
    with pytest.raises(ValueError, match="eps"):
        ops.gated_residual_norm(x, f, **{which: (None, None, eps)})


def test_refusals_of_the_int8_projection(on_cpu):
    from musev_amd import ops
    w = ops.pack_weight_i8(torch.ones(24, 40, dtype=torch.int8), torch.ones(24))
    assert w.codes.shape == (24, 128) and int(w.codes[:, 40:].abs().sum()) == 0 and w.k == 40
    a = ops.Int8Rows(torch.zeros(6, 128, dtype=torch.int8), torch.ones(6), 40)
    b, r = torch.zeros(24, dtype=torch.float16), torch.zeros(6, 24, dtype=torch.float16)
    with pytest.raises(on_cpu):
        ops.gemm_i8(a, w, bias=b, residual=r, out=r)
    for kw, match in ((dict(bias=b[:8]), "bias"), (dict(residual=r[:5]), "residual"), (dict(dtype=torch.float32), "dtype"), (dict(act=9), "activation"),
                      (dict(out=r[:, :8]), "out"), (dict(bias=b.bfloat16()), "bias")):
        with pytest.raises(ValueError, match=match):
            ops.gemm_i8(a, w, **kw)
    with pytest.raises(ValueError, match="rows of"):
        ops.gemm_i8(ops.Int8Rows(a.codes, a.scale, 41), w)
    for codes, scale, k in ((a.codes, a.scale, 129), (a.codes[:, :64], a.scale, 40), (a.codes, a.scale[:5], 40), (a.codes.int(), a.scale, 40)):
        with pytest.raises(ValueError, match="Int8Rows"):
            ops.Int8Rows(codes, scale, k)
    x = torch.zeros(6, 40, dtype=torch.float16)
    with pytest.raises(ValueError, match="weight of"):
        ops.linear_i8(x[:, :39], w)
    sq = ops.pack_weight_i8(torch.ones(40, 40, dtype=torch.int8), torch.ones(40))
    with pytest.raises(ValueError, match="overlaps"):
        ops.linear_i8(x, sq, out=x)
    with pytest.raises(ValueError, match="131071"):
        ops.pack_weight_i8(torch.zeros(1, 131072, dtype=torch.int8), torch.ones(1))
    for codes, scale, match in ((w.codes.int(), w.scale, "codes"), (w.codes, w.scale[:3], "scale"), (w.codes, w.scale.double(), "scale")):
        with pytest.raises(ValueError, match=match):
            ops.pack_weight_i8(codes, scale)


# ---- packed attention -------------------------------------------------------------------------------------------------------------
def attention_oracle(q, k, v, ql, kl, heads, kv_heads, d, causal, scale=None):
    """(out, bound): out in fp64.  Bound: with P_j = exp(s_j - m) rounded to the type once (u relative; fp16 below 2^-14: 2^-25 absolute,
    and the largest P of a row is at least 1), the scores' fp32 error e <= (d + 8) 2^-24 scale sum|q||k| turning into e relative on P, exp
    and the fp32 sums 2^-20, and one rounding of the result:
        |err| <= u |o| + (u + 2 e + 2^-19) sum p |v| + [fp16] 2^-25 sum |v| + half a subnormal step"""
    scale = d ** -0.5 if scale is None else scale
    u = half_step(q.dtype)
    out = torch.zeros(sum(ql), heads * d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    q0 = k0 = 0
    for lq, lk in zip(ql, kl):
        for h in range(heads):
            kvh = h // (heads // kv_heads)
            qq = q[q0:q0 + lq, h * d:(h + 1) * d].double()
            kk, vv = k[k0:k0 + lk, kvh * d:(kvh + 1) * d].double(), v[k0:k0 + lk, kvh * d:(kvh + 1) * d].double()
            for r in range(0, lq, 1024):
                e = min(lq, r + 1024)
                see = torch.ones(e - r, lk, dtype=torch.bool, device=q.device)
                if causal:
                    see = torch.arange(lk, device=q.device)[None] <= torch.arange(r, e, device=q.device)[:, None] + lk - lq
                any_seen = see.any(1, keepdim=True)
                s = (qq[r:e] @ kk.t()).nan_to_num() * scale
                s = s.masked_fill(~see, -math.inf)
                m = s.amax(1, keepdim=True).masked_fill(~any_seen, 0.0) if lk else torch.zeros(e - r, 1, dtype=torch.float64, device=q.device)
                p = torch.exp(s - m)
                p = p / p.sum(1, keepdim=True).masked_fill(~any_seen, 1.0)
                vz = vv.nan_to_num(nan=0.0, posinf=0.0, neginf=0.0)
                o = p @ vz
                err = (d + 8) * 2.0 ** -24 * abs(scale) * (qq[r:e].abs() @ kk.abs().nan_to_num(0.0, 0.0, 0.0).t()).masked_fill(~see, 0.0).amax(1, keepdim=True) \
                    if lk else torch.zeros(e - r, 1, dtype=torch.float64, device=q.device)
                b = u * o.abs() + (u + 2 * err + 2.0 ** -19) * (p @ vz.abs()) + subnormal(q.dtype)
                if q.dtype == torch.float16:
                    b = b + 2.0 ** -25 * (see.double() @ vz.abs())
                out[q0 + r:q0 + e, h * d:(h + 1) * d] = o
                bound[q0 + r:q0 + e, h * d:(h + 1) * d] = b * any_seen
        q0, k0 = q0 + lq, k0 + lk
    return out, bound


def attention_inputs(ql, kl, heads, kv_heads, d, dt, seed, fused=False, scale=1.0):
    if fused:
        qkv = rnd((sum(ql) + 3, (heads + 2 * kv_heads) * d), seed, dt, scale)
        return qkv[:, :heads * d], qkv[:, heads * d:(heads + kv_heads) * d], qkv[:, (heads + kv_heads) * d:]
    return rnd((sum(ql), heads * d), seed, dt, scale), rnd((sum(kl), kv_heads * d), seed + 1, dt, scale), rnd((sum(kl), kv_heads * d), seed + 2, dt)


ATTN = {
    "one": ([1], None, 1, 1, 64, True),
    "lengths_zero_to_long": ([0, 1, 2, 63, 64, 65, 127, 128, 129, 300, 0], None, 2, 2, 64, True),
    "bidirectional": ([5, 0, 64, 200, 129], None, 3, 3, 128, False),
    "grouped": ([130, 1, 77], None, 8, 2, 128, True),
    "grouped_three": ([50, 43], None, 6, 2, 40, True),
    "one_kv_head": ([70, 9], None, 7, 1, 24, False),
    "chunks": ([7, 1, 64, 129], [300, 4097, 64, 1000], 8, 2, 80, True),
    "more_queries_than_keys": ([40, 200, 5], [3, 100, 0], 4, 4, 64, True),
    "cross": ([40, 200, 5], [77, 0, 1], 4, 2, 64, False),
    "one_token": ([1] * 9, [1, 2, 63, 64, 65, 129, 1000, 5000, 0], 32, 8, 128, True),
    "one_token_no_groups": ([1, 1], [3000, 77], 4, 4, 104, True),
    "one_token_wide_group": ([1, 2], [700, 9000], 32, 1, 128, True),
    "few_rows_long_keys": ([3, 2], [16500, 12001], 4, 2, 64, True),
    "d8": ([33, 70], None, 2, 1, 8, True),
    "d16": ([33, 70], [100, 71], 2, 1, 16, False),
    "d32": ([129, 65], None, 2, 2, 32, True),
    "d48": ([65], [190], 4, 2, 48, True),
    "d112": ([150], None, 2, 2, 112, True),
    "d72": ([33, 150], None, 2, 2, 72, False),
    "d96": ([200], None, 2, 2, 96, True),
    "d120": ([100], [333], 2, 1, 120, True),
    "long": ([2500], None, 2, 1, 128, True),
    "many_short": ([(i * 7) % 23 for i in range(150)], None, 2, 2, 64, True),
}


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("name", list(ATTN))
def test_attention(name, dt):
    from musev_amd import ops
    ql, kl, heads, kvh, d, causal = ATTN[name]
    fused = kl is None
    kl = ql if kl is None else kl
    q, k, v = attention_inputs(ql, kl, heads, kvh, d, dt, 11, fused)
    plan = ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d, causal=causal)
    got = ops.attention_packed(plan, q, k, v)
    torch.cuda.synchronize()
    within(got, *attention_oracle(q, k, v, ql, kl, heads, kvh, d, causal), what=name)


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("seed", range(6))
def test_attention_of_drawn_lengths(seed, dt):
    from musev_amd import ops
    r = random.Random(1000 + seed)
    kvh, d, causal = r.choice([1, 2, 4]), 8 * r.randint(1, 16), r.random() < 0.6
    heads = kvh * r.choice([1, 2, 5, 8])
    kl = [r.choice([0, 1, r.randint(2, 64), r.randint(65, 1500)]) for _ in range(r.randint(1, 8))]
    ql = [r.choice([0, 1, kv, r.randint(1, 200)]) for kv in kl]
    q, k, v = attention_inputs(ql, kl, heads, kvh, d, dt, seed)
    got = ops.attention_packed(ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d, causal=causal), q, k, v)
    torch.cuda.synchronize()
    within(got, *attention_oracle(q, k, v, ql, kl, heads, kvh, d, causal), what=(ql, kl, heads, kvh, d, causal))


@gpu
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_blocks_that_would_run_late(causal):
    """a little more than a round of blocks: the last tiles' keys are split"""
    from musev_amd import ops
    ql, kl, heads, kvh, d = [2176, 3], [4100, 900], 32, 4, 32
    q, k, v = attention_inputs(ql, kl, heads, kvh, d, torch.float16, 21)
    plan = ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d, causal=causal)
    assert plan.n_joins > 0 or causal
    got = ops.attention_packed(plan, q, k, v)
    torch.cuda.synchronize()
    within(got, *attention_oracle(q, k, v, ql, kl, heads, kvh, d, causal), what=causal)


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_attention_of_peaked_and_of_growing_scores(dt):
    """scores up to some hundreds (the running maximum moves a lot), keys that grow along the sequence, another scale"""
    from musev_amd import ops
    ql, heads, kvh, d = [300, 77], 4, 2, 64
    q, k, v = attention_inputs(ql, ql, heads, kvh, d, dt, 5, scale=4.0)
    k = (k.float() * torch.linspace(0.1, 3.0, k.shape[0], device=DEV)[:, None]).to(dt)
    for scale in (None, 0.03, -0.2):
        got = ops.attention_packed(ops.attention_plan(ql, heads=heads, kv_heads=kvh, d=d, scale=scale), q, k, v)
        torch.cuda.synchronize()
        within(got, *attention_oracle(q, k, v, ql, ql, heads, kvh, d, True, scale), what=scale)


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("scale", [0.0, 1e-30])
def test_attention_of_a_vanishing_scale(scale, dt):
    """every key a query sees weighs the same; keys split over many parts and not"""
    from musev_amd import ops
    ql, kl = [130, 1, 0, 2], [130, 3000, 7, 64]
    q, k, v = attention_inputs(ql, kl, 4, 2, 64, dt, 31)
    got = ops.attention_packed(ops.attention_plan(ql, kl, heads=4, kv_heads=2, d=64, scale=scale), q, k, v)
    torch.cuda.synchronize()
    within(got, *attention_oracle(q, k, v, ql, kl, 4, 2, 64, True, scale), what=scale)


@gpu
@pytest.mark.parametrize("dt,big,step", [(torch.bfloat16, 2.0 ** 55, 2.0 ** 50), (torch.float16, 2.0 ** 15, 2.0 ** 4)], ids=["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [([200], [200]), ([1, 3], [5000, 70])], ids=["prompt", "split"])
def test_attention_of_scores_far_below_zero(lens, d, dt, big, step):
    """the best score a query sees is -d big step, the others lower by at least as much: its output is that key's value, exactly"""
    from musev_amd import ops
    ql, kl = lens
    q = torch.full((sum(ql), d), big, device=DEV).to(dt)
    rank = torch.cat([torch.arange(n) % 200 + 1 + (torch.arange(n) > 0) for n in kl])
    k = (rank[:, None].float() * -step).expand(-1, d).contiguous().to(DEV).to(dt)   # (multiples of a power of two up to 201: exact)
    v = rnd((sum(kl), d), 3, dt)
    got = ops.attention_packed(ops.attention_plan(ql, kl, heads=1, d=d, scale=1.0), q, k, v)
    first = torch.tensor([sum(kl[:i]) for i, n in enumerate(ql) for _ in range(n)], device=DEV)
    assert torch.equal(got, v[first])


@gpu
@pytest.mark.parametrize("one", [False, True], ids=["prompt", "one_token"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=["nan", "inf", "-inf"])
def test_what_is_not_seen_does_not_reach_the_output(bad, one):
    """later tokens of the same tile, the next sequence in the same tile, rows behind the last sequence"""
    from musev_amd import ops
    dt, heads, kvh, d = torch.float16, 4, 2, 64
    ql, kl = ([1, 1], [70, 300]) if one else ([40, 200], [70, 200])
    q, k, v = attention_inputs(ql, kl, heads, kvh, d, dt, 9)
    pad = torch.zeros(40, kvh * d, dtype=dt, device=DEV)
    k, v = torch.cat([k, pad]), torch.cat([v, pad])
    # (the bound is attention_oracle's: the order in which a row's sum is formed is not part of the definition and may differ beside such values)
    clean, bound = attention_oracle(q, k, v, ql, kl, heads, kvh, d, True)
    k2, v2 = k.clone(), v.clone()
    k2[sum(kl):], v2[sum(kl):] = bad, bad
    if one:
        first_bad = 1                     # the second sequence's keys: seen by the second query only
        k2[70:], v2[70:] = bad, bad
    else:
        first_bad = 40 + 150              # a later token of the second sequence
        k2[70 + 150], v2[70 + 150] = bad, bad
    got = ops.attention_packed(ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d), q, k2, v2)
    torch.cuda.synchronize()
    within(got[:first_bad], clean[:first_bad], bound[:first_bad])
    if not one:   # V alone: a visible infinity is an infinity, a visible NaN is NaN, in its own columns only
        v3 = v.clone()
        v3[70 + 150, 5] = bad
        got = ops.attention_packed(ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d), q, k, v3)
        torch.cuda.synchronize()
        seen = got[40 + 150:].view(-1, heads, d)[:, :2, 5]
        assert bool((torch.isnan(seen) if math.isnan(bad) else seen == bad).all())
        rest = torch.ones_like(got, dtype=torch.bool)
        rest.view(-1, heads, d)[40 + 150:, :2, 5] = False
        within(got[rest], clean[rest], bound[rest])


@gpu
def test_attention_leaves_rows_behind_the_last_sequence_and_other_columns():
    from musev_amd import ops
    dt, heads, d, ql = torch.bfloat16, 2, 64, [5, 140]
    q, k, v = attention_inputs(ql, ql, heads, heads, d, dt, 3, fused=True)
    wide = torch.full((160, 304), 7.0, dtype=dt, device=DEV)
    out = wide[:, 8:8 + heads * d]
    res = ops.attention_packed(ops.attention_plan(ql, heads=heads, d=d), q, k, v, out=out)
    torch.cuda.synchronize()
    assert res is out
    within(out[:145], *attention_oracle(q, k, v, ql, ql, heads, heads, d, True))
    assert bool((wide[145:] == 7).all()) and bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + heads * d:] == 7).all())


@gpu
def test_attention_of_no_rows_at_all():
    from musev_amd import ops
    for dt in DTYPES:
        e = torch.empty(0, 128, dtype=dt, device=DEV)
        assert ops.attention_packed(ops.attention_plan([0, 0], heads=2, d=64), e, e, e).shape == (0, 128)
        k = rnd((9, 128), 1, dt)
        assert ops.attention_packed(ops.attention_plan([0, 0], [4, 5], heads=2, d=64), e, k, k).shape == (0, 128)
        q = rnd((7, 128), 2, dt)
        got = ops.attention_packed(ops.attention_plan([3, 4], [0, 0], heads=2, d=64), q, e, e)
        torch.cuda.synchronize()
        assert bool((got == 0).all())


@gpu
def test_attention_far_into_a_large_matrix():
    """key rows whose byte offsets pass 2^32, and rows 8 MB apart"""
    from musev_amd import ops
    dt, d = torch.float16, 64
    ld = 1 << 20
    big = torch.zeros(3000 * ld + 512, dtype=dt, device=DEV)     # 6 GB
    k = big[:3000 * ld].view(3000, ld)[:, 8:8 + d]
    v = big[:3000 * ld].view(3000, ld)[:, 128:128 + d]
    k.copy_(rnd((3000, d), 3, dt))
    v.copy_(rnd((3000, d), 4, dt))
    q = rnd((131, d), 5, dt)
    ql, kl = [1, 130], [100, 2900]
    got = ops.attention_packed(ops.attention_plan(ql, kl, heads=1, d=d), q, k, v)
    torch.cuda.synchronize()
    within(got, *attention_oracle(q, k.contiguous(), v.contiguous(), ql, kl, 1, 1, d, True))


# ---- rotary positions ---------------------------------------------------------------------------------------------------------------
def rotary_oracle(x, pos, sections, theta, shared, heads, d, pairing):
    """(out, bound): angle and turn in fp64.  Bound: u |y| for the rounding, 2^-20 hypot(a, b) for the fp32 sine, cosine and products"""
    rotary = sum(sections)
    ang = []
    for a, n in enumerate(sections):
        for i in range(n // 2):
            e = 2.0 * len(ang) / rotary if shared else 2.0 * i / n
            ang.append(pos[:, a].double() * theta ** -e)
    ang = torch.stack(ang, 1)[:, None]
    y = x.double().view(-1, heads, d).clone()
    size = torch.zeros_like(y)
    p = torch.arange(rotary // 2, device=x.device)
    ia, ib = (2 * p, 2 * p + 1) if pairing == "adjacent" else (p, p + rotary // 2)
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    size[..., ia] = size[..., ib] = torch.hypot(a, b)
    bound = (half_step(x.dtype) * y.abs() + 2.0 ** -20 * size + subnormal(x.dtype)) * (size > 0)
    return y.reshape(x.shape), bound.reshape(x.shape)


ROT = {
    # tokens, heads, kv_heads, d, sections, theta, shared, pairing, position kind, last position
    "one_token": (1, 32, 8, 128, [128], 10000.0, False, "halves", "int", 131072),
    "video": (300, 4, 4, 128, [32, 48, 48], 10000.0, False, "adjacent", "int", 64),
    "video_halves": (77, 6, 2, 128, [32, 48, 48], 10000.0, False, "halves", "int", 64),
    "shared_ladder": (65, 4, 1, 128, [32, 48, 48], 1000000.0, True, "halves", "int", 40000),
    "pass_through": (33, 3, 3, 80, [8, 24, 24], 10000.0, False, "adjacent", "float", 50),
    "pass_through_halves": (33, 3, 3, 80, [8, 24, 26], 10000.0, False, "halves", "float", 50),
    "odd_pairs": (29, 5, 5, 50, [6, 10, 30], 500.0, False, "adjacent", "int", 900),
    "odd_pairs_halves": (29, 5, 5, 50, [6, 10, 30], 500.0, False, "halves", "int", 900),
    "odd_head": (17, 3, 1, 21, [2, 18], 10000.0, False, "adjacent", "float", 100),
    "odd_head_halves": (17, 3, 1, 21, [2, 18], 10000.0, True, "halves", "float", 100),
    "far": (64, 2, 2, 64, [64], 10000.0, False, "adjacent", "int", 2 ** 31 - 1),
    "far_float": (64, 2, 2, 64, [64], 10000.0, False, "halves", "float", 1.0e6),
    "four_axes": (100, 2, 1, 40, [8, 8, 8, 16], 10000.0, False, "adjacent", "int", 1000),
    "many_tokens": (5000, 8, 8, 64, [16, 24, 24], 10000.0, False, "halves", "int", 64),
}


def rotary_inputs(name, dt):
    n, heads, kvh, d, sec, theta, shared, pairing, kind, top = ROT[name]
    qk = rnd((n, (heads + kvh) * d), 21, dt)
    g = torch.Generator().manual_seed(22)
    if kind == "int":
        pos = torch.randint(-(top // 4), top, (n, len(sec)), generator=g, dtype=torch.int64).to(torch.int32).to(DEV)
    else:
        pos = ((torch.rand((n, len(sec)), generator=g) - 0.2) * top).to(DEV)
    return qk[:, :heads * d], qk[:, heads * d:], pos


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("name", list(ROT))
def test_rotary(name, dt):
    from musev_amd import ops
    n, heads, kvh, d, sec, theta, shared, pairing, kind, top = ROT[name]
    q, k, pos = rotary_inputs(name, dt)
    table = ops.rotary_table(sec, theta, shared=shared)
    oq, ok = ops.rotary_axes(q, k, pos, table, heads=heads, kv_heads=kvh, d=d, pairing=pairing)
    only, none = ops.rotary_axes(q, None, pos, table, heads=heads, d=d, pairing=pairing)
    torch.cuda.synchronize()
    assert none is None and torch.equal(only, oq)
    for got, x, h in ((oq, q, heads), (ok, k, kvh)):
        within(got, *rotary_oracle(x, pos, sec, theta, shared, h, d, pairing), what=name)
    q2, k2 = q.clone(), k.clone()   # in place
    rq, rk = ops.rotary_axes(q2, k2, pos, table, heads=heads, kv_heads=kvh, d=d, pairing=pairing, out_q=q2, out_k=k2)
    torch.cuda.synchronize()
    assert rq is q2 and rk is k2 and torch.equal(q2, oq) and torch.equal(k2, ok)


@gpu
@pytest.mark.parametrize("off", [1, 4, 8])
def test_rotary_of_unaligned_slices(off):
    from musev_amd import ops
    dt, heads, d, sec = torch.float16, 3, 64, [16, 24, 24]
    big = rnd((70, off + heads * d + 5), 31, dt)
    pos = torch.randint(0, 64, (70, 4), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).to(DEV)[:, 1:]
    q = big[:, off:off + heads * d]
    keep = big.clone()
    want, bound = rotary_oracle(q, pos, sec, 10000.0, False, heads, d, "adjacent")
    ops.rotary_axes(q, None, pos, ops.rotary_table(sec), heads=heads, d=d, out_q=q)
    torch.cuda.synchronize()
    within(q, want, bound)
    assert torch.equal(big[:, :off], keep[:, :off]) and torch.equal(big[:, off + heads * d:], keep[:, off + heads * d:])


# ---- gated residual norm ------------------------------------------------------------------------------------------------------------
def norm_oracle(x, f, kind, alpha, post, pre, gate, scale, shift, of):
    """((s, bound), (h, bound)).  fp32 sums over C terms in trees and short runs: a statistic is off by at most 2^-19 of its terms' mean
    size; a product or sum adds 2^-23 of what it joins.  Bounds: u |result| + 2^-18 (sum of the sizes of what the result was formed from)"""
    u, c = half_step(x.dtype), 2.0 ** -18

    def stats(v, size, aff):
        mean = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
        r = 1.0 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + aff[2])
        n, sz = (v - mean) * r, (size + (size.mean(1, keepdim=True) if kind == "layer" else 0.0)) * r
        sz = sz + n.abs() * (r ** 2 * (size ** 2).mean(1, keepdim=True))    # (the statistic's own error, relative, on every element)
        if aff[0] is not None:
            n, sz = n * aff[0].double(), sz * aff[0].double().abs()
        if aff[1] is not None:
            n, sz = n + aff[1].double(), sz + aff[1].double().abs()
        return n, sz
    xd, y = x.double(), f.double()
    ysz = y.abs()
    if post is not None:
        y, ysz = stats(y, ysz, post)
    if gate is not None:
        y, ysz = y * gate.double()[of], ysz * gate.double()[of].abs()
    s, ssz = alpha * xd + y, (alpha * xd).abs() + ysz
    first = (s, u * s.abs() + c * ssz + subnormal(x.dtype))
    if pre is None:
        return first, None
    h, hsz = stats(s, ssz, pre)
    if scale is not None:
        m = 1 + scale.double()[of]
        h, hsz = h * m, hsz * (1 + scale.double()[of].abs())
    if shift is not None:
        h, hsz = h + shift.double()[of], hsz + shift.double()[of].abs()
    return first, (h, u * h.abs() + c * hsz + subnormal(x.dtype))


NORM_C = [1, 7, 8, 40, 64, 320, 500, 520, 640, 1000, 1001, 1280, 2048, 2056, 4096, 5000, 8192, 16384]


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("c", NORM_C)
def test_gated_norm(c, kind, dt):
    from musev_amd import ops
    rows, groups = (37, 5) if c < 4096 else (9, 2)
    if c in (640, 1001, 1280):
        rows = 2049   # (the form for many rows)
    x, f = rnd((rows, c), 41, dt), rnd((rows, c), 42, dt, 0.7)
    x[:, ::13] *= 20
    gate, scale, shift = (rnd((groups, c), 43 + i, dt, 0.5) for i in range(3))
    vec = [rnd((c,), 50 + i, dt, 0.3) + (1 if i % 2 == 0 else 0) for i in range(4)]
    per = -(-rows // groups)
    byrow = torch.arange(rows, device=DEV) // per
    idx = torch.randint(0, groups, (rows,), generator=torch.Generator().manual_seed(3), dtype=torch.int32).to(DEV)
    for post, pre, g, mod, index in (((vec[0], vec[1], 1e-5), (vec[2], vec[3], 1e-6), True, True, True), (None, (vec[2], None, 1e-6), True, True, False),
                                     ((vec[0], None, 1e-5), None, True, False, False), (None, (None, None, 1e-5), False, False, False),
                                     (None, None, True, False, True), (None, (None, vec[3], 1e-5), False, True, True)):
        of = (idx.long() if index else byrow) if (g or mod) else torch.zeros(rows, dtype=torch.long, device=DEV)
        kw = dict(kind=kind, alpha=0.75, post=post, pre=pre, gate=gate if g else None, scale=scale if mod else None, shift=shift if mod else None)
        how = {} if not (g or mod) else dict(group_index=idx) if index else dict(rows_per_group=per)
        s, h = ops.gated_residual_norm(x, f, **kw, **how)
        torch.cuda.synchronize()
        ws, wh = norm_oracle(x, f, kind, 0.75, post, pre, kw["gate"], kw["scale"], kw["shift"], of)
        within(s, *ws, what=("s", c, kind))
        assert (h is None) == (pre is None)
        if pre is not None:
            within(h, *wh, what=("h", c, kind))


@gpu
@pytest.mark.parametrize("kind,dt", [("layer", torch.float16), ("rms", torch.bfloat16)], ids=["layer-fp16", "rms-bf16"])
@pytest.mark.parametrize("rows", [35, 16389])
@pytest.mark.parametrize("c", [3, 100, 128, 129, 250, 256, 257, 384, 385, 511, 512])
def test_gated_norm_of_rows_that_share_a_wave(c, rows, kind, dt):
    """narrow rows side by side in a wave, some of no group (NaN) between those that have one; in place"""
    from musev_amd import ops
    x, f = rnd((rows, c), 41, dt), rnd((rows, c), 42, dt, 0.7)
    gate, scale, shift = (rnd((5, c), 43 + i, dt, 0.5) for i in range(3))
    post, pre = (rnd((c,), 50, dt, 0.3) + 1, rnd((c,), 51, dt, 0.3), 1e-5), (rnd((c,), 52, dt, 0.3) + 1, None, 1e-6)
    idx = torch.randint(-1, 6, (rows,), generator=torch.Generator().manual_seed(3), dtype=torch.int32).to(DEV)
    has = (idx >= 0) & (idx < 5)
    want = norm_oracle(x, f, kind, 0.75, post, pre, gate, scale, shift, idx.long().clamp(0, 4))
    s, h = ops.gated_residual_norm(x, f, kind=kind, alpha=0.75, post=post, pre=pre, gate=gate, scale=scale, shift=shift, group_index=idx, out=x, norm_out=f)
    torch.cuda.synchronize()
    for got, (w, b) in zip((s, h), want):
        assert bool(got[~has].isnan().all())
        within(got[has], w[has], b[has], what=(c, rows, kind))


@gpu
@pytest.mark.parametrize("c", [40, 320, 1001, 4100])
def test_gated_norm_in_place_strided_and_unaligned(c):
    from musev_amd import ops
    dt, rows = torch.bfloat16, 50
    big = rnd((rows, 2 * c + 11), 61, dt)
    x, f = big[:, 3:3 + c], big[:, 5 + c:5 + 2 * c]
    gate = rnd((1, c + 1), 62, dt)[:, 1:]
    pre = (None, None, 1e-6)
    keep = big.clone()
    ws, wh = norm_oracle(x.clone(), f.clone(), "layer", 1.0, None, pre, gate, None, None, torch.zeros(rows, dtype=torch.long, device=DEV))
    s, h = ops.gated_residual_norm(x, f, pre=pre, gate=gate, out=x, norm_out=f)
    torch.cuda.synchronize()
    assert s is x and h is f
    within(s, *ws)
    within(h, *wh)
    mask = torch.ones(2 * c + 11, dtype=torch.bool)
    mask[3:3 + c] = mask[5 + c:5 + 2 * c] = False
    assert torch.equal(big[:, mask.to(DEV)], keep[:, mask.to(DEV)])


@gpu
def test_gated_norm_rows_of_no_group_zero_rows_and_constant_rows():
    from musev_amd import ops
    dt, c = torch.float16, 320
    x, f, gate = rnd((6, c), 71, dt), rnd((6, c), 72, dt), rnd((3, c), 73, dt)
    idx = torch.tensor([0, 3, -1, 2, 2 ** 31 - 1, 1], dtype=torch.int32, device=DEV)
    s, h = ops.gated_residual_norm(x, f, gate=gate, pre=(None, None, 1e-6), group_index=idx)
    torch.cuda.synchronize()
    bad = torch.tensor([False, True, True, False, True, False], device=DEV)
    assert bool(torch.isnan(s[bad]).all()) and bool(torch.isnan(h[bad]).all())
    ws, wh = norm_oracle(x[~bad], f[~bad], "layer", 1.0, None, (None, None, 1e-6), gate, None, None, idx[~bad].long())
    within(s[~bad], *ws)
    within(h[~bad], *wh)
    s, h = ops.gated_residual_norm(x[:0], f[:0], pre=(None, None, 1e-6))
    assert s.shape == (0, c) and h.shape == (0, c)
    z = torch.zeros(2, c, dtype=dt, device=DEV)   # a constant row has no spread: 0 (layer), a zero row 0 (rms)
    for kind in ("layer", "rms"):
        s, h = ops.gated_residual_norm(z + (3 if kind == "layer" else 0), z, kind=kind, pre=(None, None, 1e-6))
        torch.cuda.synchronize()
        assert bool((h == 0).all())


# ---- int8 projection ------------------------------------------------------------------------------------------------------------------
def quantized(x):
    """exact codes (fp64 quotients of short numbers round like the exact ones) and the fp32 scale"""
    top = x.double().abs().amax(1, keepdim=True)
    codes = torch.round(127 * x.double() / top.masked_fill(top == 0, 1))
    return codes, (top / 127).float().double()


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("k", [1, 7, 8, 127, 128, 129, 320, 1000, 1280, 5120, 9000])
def test_quantize_rows(k, dt):
    from musev_amd import ops
    x = rnd((19, k), 81, dt)
    x[3] = 0
    x[4] *= 1e-4
    x[5] = (torch.arange(k, device=DEV) % 128).to(dt)          # top 127 (where k allows): codes are the values
    x[6] = ((torch.arange(k, device=DEV) % 254).float() / 2).to(dt)
    x[6, 0] = 127                                              # ties: halves round to even
    x[7, 0] = torch.finfo(dt).max
    x[8] = torch.finfo(dt).tiny
    big = torch.zeros(19, k + 3, dtype=dt, device=DEV)
    big[:, 1:k + 1] = x
    for t in (x, big[:, 1:k + 1]):
        got = ops.quantize_rows_i8(t)
        torch.cuda.synchronize()
        codes, scale = quantized(x)
        assert got.k == k and got.codes.shape == (19, -(-k // 128) * 128)
        assert torch.equal(got.codes[:, :k].double(), codes), (got.codes[:, :k].double() - codes).abs().amax(1)
        assert bool((got.codes[:, k:] == 0).all())
        assert torch.equal(got.scale.double(), scale[:, 0])


def linear_oracle(x, codes, w_scale, bias, residual, silu):
    """(out, bound): the sum of products is exact, then a handful of fp32 operations (2^-20 of every size joined; SiLU's exp and reciprocal
    included) and one rounding"""
    c, s = quantized(x)
    y = (c @ codes.double().t()) * s * w_scale.double()
    size = y.abs()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    if silu:
        size = size + y.abs()
        y = y * torch.sigmoid(y)
    if residual is not None:
        y, size = y + residual.double(), size + residual.double().abs()
    return y, half_step(x.dtype) * y.abs() + 2.0 ** -19 * size + subnormal(x.dtype)


LIN = [(1, 16384, 40), (1, 16385, 40), (3, 5000, 100), (4, 4096, 33), (4, 4097, 33), (8, 1024, 64), (8, 1025, 64), (16, 512, 48), (16, 513, 48), (5, 1600, 20), (1, 1, 1), (4, 3, 5), (1, 128, 128), (1, 1280, 5120), (1, 1000, 1111), (2, 64, 7), (3, 40, 1), (5, 5120, 640), (8, 129, 33), (16, 1280, 320), (17, 1280, 320), (31, 384, 257),
       (33, 256, 96), (64, 640, 640), (65, 1000, 255), (127, 128, 256), (128, 256, 128), (129, 320, 129), (255, 2560, 320), (300, 1152, 1000),
       (1001, 1000, 1111), (1000, 5120, 1280), (4100, 640, 512), (513, 16, 513), (2, 9000, 48), (33, 16, 33), (40, 130, 1000), (100, 700, 130), (513, 2050, 1000), (400, 3000, 1000), (25, 2100, 90), (700, 128, 260)]


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("mkn", LIN, ids=[f"{m}x{k}x{n}" for m, k, n in LIN])
def test_linear_i8(mkn, dt):
    from musev_amd import ops
    m, k, n = mkn
    x = rnd((m, k), 91, dt)
    x[:, ::61] *= 8
    g = torch.Generator().manual_seed(92)
    codes = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8).to(DEV)
    ws = ((0.5 + torch.rand(n, generator=g)) / (73 * math.sqrt(k))).to(DEV)
    bias, res = rnd((n,), 93, dt), rnd((m, n + 5), 94, dt)[:, 3:3 + n]
    w = ops.pack_weight_i8(codes, ws)
    for b, r, act in ((None, None, 0), (bias, res, 0), (bias, None, ops.MV_ACT_SILU), (None, res, ops.MV_ACT_SILU)):
        got = ops.linear_i8(x, w, bias=b, residual=r, act=act)
        torch.cuda.synchronize()
        within(got, *linear_oracle(x, codes, ws, b, r, act == ops.MV_ACT_SILU), what=(mkn, act))
        assert torch.equal(got, ops.gemm_i8(ops.quantize_rows_i8(x), w, bias=b, residual=r, act=act, dtype=dt))
    wide = torch.full((m, n + 9), 3.0, dtype=dt, device=DEV)   # a strided result that is the residual itself
    out = wide[:, 1:1 + n]
    out.copy_(res)
    ops.linear_i8(x, w, residual=out, out=out)
    torch.cuda.synchronize()
    within(out, *linear_oracle(x, codes, ws, None, res, False))
    assert bool((wide[:, :1] == 3).all()) and bool((wide[:, 1 + n:] == 3).all())


@gpu
@pytest.mark.parametrize("m,k,n,dt", [(8200, 300, 8197, torch.float16), (26624, 200, 5121, torch.bfloat16)], ids=["ragged", "residual_past_the_cache"])
def test_linear_i8_large(m, k, n, dt):
    """the largest tiles, ragged on every side"""
    from musev_amd import ops
    x = rnd((m, k), 1, dt)
    g = torch.Generator().manual_seed(2)
    codes = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8).to(DEV)
    ws = ((0.5 + torch.rand(n, generator=g)) / (73 * math.sqrt(k))).to(DEV)
    bias, w = rnd((n,), 3, dt), ops.pack_weight_i8(codes, ws)
    res = torch.randn((m, n + 3), generator=torch.Generator(DEV).manual_seed(4), device=DEV).to(dt)[:, 1:1 + n]
    for r, act in ((None, ops.MV_ACT_SILU), (res, 0)):
        got = ops.linear_i8(x, w, bias=bias, residual=r, act=act)
        torch.cuda.synchronize()
        for a in range(0, m, 4096):
            want, bound = linear_oracle(x[a:a + 4096], codes, ws, bias, None if r is None else r[a:a + 4096], act == ops.MV_ACT_SILU)
            within(got[a:a + 4096], want, bound, what=(m, k, n, a))


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("k", [2600, 2817, 4096])
def test_linear_i8_long_k_in_two_groups(k, dt):
    """an even and an odd number of steps of K shared by two groups of waves"""
    from musev_amd import ops
    m, n = 701, 1501
    x = rnd((m, k), 1, dt)
    codes = torch.randint(-127, 128, (n, k), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(torch.int8).to(DEV)
    ws = ((0.5 + torch.rand(n, generator=torch.Generator().manual_seed(3))) / (73 * math.sqrt(k))).to(DEV)
    res, w = rnd((m, n), 4, dt), ops.pack_weight_i8(codes, ws)
    got = ops.linear_i8(x, w, residual=res)
    torch.cuda.synchronize()
    within(got, *linear_oracle(x, codes, ws, None, res, False), what=k)


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1900, 100, 3989), (2048, 1300, 2100), (5848, 260, 4000)], ids=["one_round", "long_k", "left_over"])
def test_linear_i8_one_round_of_middle_tiles(m, k, n, dt):
    """tiles of 128 x 128, ragged, alone and for the rows that the largest tiles leave"""
    from musev_amd import ops
    x = rnd((m, k), 1, dt)
    codes = torch.randint(-127, 128, (n, k), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(torch.int8).to(DEV)
    ws = ((0.5 + torch.rand(n, generator=torch.Generator().manual_seed(3))) / (73 * math.sqrt(k))).to(DEV)
    bias, w = rnd((n,), 3, dt), ops.pack_weight_i8(codes, ws)
    res = torch.randn((m, n + 3), generator=torch.Generator(DEV).manual_seed(4), device=DEV).to(dt)[:, 1:1 + n]
    for r, act in ((None, ops.MV_ACT_SILU), (res, 0)):
        got = ops.linear_i8(x, w, bias=bias, residual=r, act=act)
        torch.cuda.synchronize()
        for a in range(0, m, 4096):
            want, bound = linear_oracle(x[a:a + 4096], codes, ws, bias, None if r is None else r[a:a + 4096], act == ops.MV_ACT_SILU)
            within(got[a:a + 4096], want, bound, what=(m, k, n, a))


@gpu
@pytest.mark.parametrize("m,k,n,dt", [(8200, 300, 8190, torch.float16), (8300, 140, 8190, torch.bfloat16)])
def test_linear_i8_rows_left_over_by_whole_rounds(m, k, n, dt):
    """the rows behind the last whole round of the largest tiles, added to a residual in place; columns beside the result stay as they were"""
    from musev_amd import ops
    x = rnd((m, k), 1, dt)
    codes = torch.randint(-127, 128, (n, k), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(torch.int8).to(DEV)
    ws = ((0.5 + torch.rand(n, generator=torch.Generator().manual_seed(3))) / (73 * math.sqrt(k))).to(DEV)
    bias, w = rnd((n,), 3, dt), ops.pack_weight_i8(codes, ws)
    wide = torch.randn((m, n + 4), generator=torch.Generator(DEV).manual_seed(4), device=DEV).to(dt)
    before = wide.clone()
    got = ops.linear_i8(x, w, bias=bias, residual=wide[:, 1:1 + n], out=wide[:, 1:1 + n])
    torch.cuda.synchronize()
    assert torch.equal(wide[:, :1], before[:, :1]) and torch.equal(wide[:, 1 + n:], before[:, 1 + n:])
    for a in range(0, m, 4096):
        want, bound = linear_oracle(x[a:a + 4096], codes, ws, bias, before[a:a + 4096, 1:1 + n], False)
        within(got[a:a + 4096], want, bound, what=(m, k, n, a))


@gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_i8_extreme_codes_zero_and_nonfinite_rows(m):
    """the largest possible sum (K = 131072 would reach 2^31) stays exact; a row that is not finite gives NaN, the others do not notice"""
    from musev_amd import ops
    dt, k, n = torch.bfloat16, 65536, 130
    x = torch.full((m, k), -1.0, dtype=dt, device=DEV)
    codes = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w = ops.pack_weight_i8(codes, torch.full((n,), 2.0 ** -20, device=DEV))
    if m > 2:
        x[1] = 0
        x[2, 77] = float("inf")
        x[3, 78] = float("nan")
    got = ops.linear_i8(x, w)
    torch.cuda.synchronize()
    want = torch.full((m, n), 128.0 * k * 2.0 ** -20, dtype=torch.float64, device=DEV)
    rows = torch.ones(m, dtype=torch.bool, device=DEV)
    if m > 2:
        want[1] = 0
        rows[2:4] = False
        assert bool(torch.isnan(got[2:4]).all())
    within(got[rows], want[rows], half_step(dt) * want[rows].abs() + 2.0 ** -20 * want[rows])


@gpu
def test_no_rows():
    from musev_amd import ops
    w = ops.pack_weight_i8(torch.ones(8, 40, dtype=torch.int8, device=DEV), torch.ones(8, device=DEV))
    for dt in DTYPES:
        x = torch.empty(0, 40, dtype=dt, device=DEV)
        assert ops.linear_i8(x, w).shape == (0, 8) and ops.quantize_rows_i8(x).codes.shape == (0, 128)
        assert ops.gemm_i8(ops.quantize_rows_i8(x), w, dtype=dt).shape == (0, 8)
        assert ops.rotary_axes(x, None, torch.empty(0, 1, device=DEV), ops.rotary_table([40]), heads=1, d=40)[0].shape == (0, 40)


@gpu
@pytest.mark.parametrize("m", [1, 20, 200])
def test_linear_of_columns_of_a_wide_matrix(m):
    """x a column slice with an odd offset, the result another matrix's slice, two results side by side"""
    from musev_amd import ops
    dt, k, n = torch.bfloat16, 300, 133
    big = rnd((m, k + 9), 5, dt)
    x = big[:, 3:3 + k]
    g = torch.Generator().manual_seed(6)
    codes = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8).to(DEV)
    ws = torch.full((n,), 0.01, device=DEV)
    w = ops.pack_weight_i8(codes.t().contiguous().t(), ws)     # (any strides)
    wide = torch.zeros(m, 2 * n, dtype=dt, device=DEV)
    ops.linear_i8(x, w, out=wide[:, :n])
    ops.linear_i8(x, w, out=wide[:, n:], residual=wide[:, :n])
    torch.cuda.synchronize()
    want, bound = linear_oracle(x.contiguous(), codes, ws, None, None, False)
    within(wide[:, :n], want, bound)
    within(wide[:, n:], *linear_oracle(x.contiguous(), codes, ws, None, wide[:, :n], False))


# ---- together, on other streams, in graphs ----------------------------------------------------------------------------------------------
class Block:
    """one transformer block's attention half as it is served: int8 q/k/v projection -> rotary positions -> packed attention -> int8 output
    projection -> gated residual norm"""

    def __init__(self, ql, dt, heads=4, kvh=2, d=64, seed=100):
        from musev_amd import ops
        self.ops, self.dt, self.ql, self.heads, self.kvh, self.d, self.c = ops, dt, ql, heads, kvh, d, heads * d
        g = torch.Generator().manual_seed(seed)
        def weight(n, k):
            codes = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8).to(DEV)
            return codes, ((0.5 + torch.rand(n, generator=g)) / (73 * math.sqrt(k))).to(DEV)
        self.wqkv, self.wo = weight((heads + 2 * kvh) * d, self.c), weight(self.c, self.c)
        self.pq, self.po = ops.pack_weight_i8(*self.wqkv), ops.pack_weight_i8(*self.wo)
        self.sec = [16, 24, 24]
        self.table = ops.rotary_table(self.sec)
        self.plan = ops.attention_plan(ql, heads=heads, kv_heads=kvh, d=d)
        rows = sum(ql)
        self.pos = torch.randint(0, 64, (rows, 3), generator=g, dtype=torch.int32).to(DEV)
        self.of = torch.repeat_interleave(torch.arange(len(ql)), torch.tensor(ql)).to(torch.int32).to(DEV)
        self.gate, self.scale, self.shift = (rnd((len(ql), self.c), seed + i, dt, 0.3) for i in range(3))
        self.pre = (rnd((self.c,), seed + 5, dt, 0.1) + 1, None, 1e-6)

    def __call__(self, x, trace=None):
        o, h, kv, d = self.ops, self.heads, self.kvh, self.d
        qkv = o.linear_i8(x, self.pq)
        q, k, v = qkv[:, :h * d], qkv[:, h * d:(h + kv) * d], qkv[:, (h + kv) * d:]
        raw = qkv.clone() if trace is not None else None
        o.rotary_axes(q, k, self.pos, self.table, heads=h, kv_heads=kv, d=d, out_q=q, out_k=k)
        a = o.attention_packed(self.plan, q, k, v)
        f = o.linear_i8(a, self.po)
        s, n = o.gated_residual_norm(x, f, gate=self.gate, pre=self.pre, scale=self.scale, shift=self.shift, group_index=self.of)
        if trace is not None:
            trace.update(raw=raw, qkv=qkv, a=a, f=f)
        return s, n


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("ql", [[77, 5, 140], [1]], ids=["prompts", "one_token"])
def test_operators_together(ql, dt):
    """every stage against its definition on what the stage before handed over"""
    b = Block(ql, dt)
    x = rnd((sum(ql), b.c), 7, dt)
    t = {}
    s, n = b(x, t)
    torch.cuda.synchronize()
    h, kv, d = b.heads, b.kvh, b.d
    within(t["raw"], *linear_oracle(x, *b.wqkv, None, None, False), what="qkv")
    for lo, cnt in ((0, h), (h * d, kv)):
        sl = slice(lo, lo + cnt * d)
        within(t["qkv"][:, sl], *rotary_oracle(t["raw"][:, sl].contiguous(), b.pos, b.sec, 10000.0, False, cnt, d, "adjacent"), what="rotary")
    q, k, v = t["qkv"][:, :h * d], t["qkv"][:, h * d:(h + kv) * d], t["qkv"][:, (h + kv) * d:]
    assert torch.equal(v, t["raw"][:, (h + kv) * d:])
    within(t["a"], *attention_oracle(q, k, v, ql, ql, h, kv, d, True), what="attention")
    within(t["f"], *linear_oracle(t["a"], *b.wo, None, None, False), what="out")
    ws, wn = norm_oracle(x, t["f"], "layer", 1.0, None, b.pre, b.gate, b.scale, b.shift, b.of.long())
    within(s, *ws, what="stream")
    within(n, *wn, what="norm")


@gpu
def test_two_captured_graphs_and_eager_calls_agree():
    """two graphs of the same plan, table and weights, replayed in turn with eager work between: each replay gives the eager result"""
    b1, dt = Block([3, 40, 1000], torch.float16), torch.float16
    b2 = Block([1, 1, 1], dt, seed=200)
    b2.plan = b2.ops.attention_plan([1, 1, 1], [1, 1, 1], heads=4, kv_heads=2, d=64)
    xs = [rnd((sum(b.ql), b.c), 300 + i, dt) for i, b in enumerate((b1, b2))]
    long_q, long_k, long_v = attention_inputs([1, 2], [9000, 7001], 8, 2, 128, dt, 17)
    plan = b1.ops.attention_plan([1, 2], [9000, 7001], heads=8, kv_heads=2, d=128)   # (joined partial sums: a workspace per graph)

    deep = b1.ops.pack_weight_i8(torch.randint(-127, 128, (640, 3000), generator=torch.Generator().manual_seed(4), dtype=torch.int32).to(torch.int8).to(DEV),
                                 torch.full((640,), 0.001, device=DEV))
    rows = rnd((300, 3000), 18, dt)   # (K in groups of waves: more LDS than a launch has by default)

    def work(b, x):
        return (*b(x), b.ops.attention_packed(plan, long_q, long_k, long_v), b.ops.linear_i8(rows, deep))
    want = [[t.clone() for t in work(b, x)] for b, x in zip((b1, b2), xs)]
    torch.cuda.synchronize()
    graphs, outs, ins = [], [], [x.clone() for x in xs]
    side = torch.cuda.Stream()
    for b, x in zip((b1, b2), ins):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(b, x)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(b, x))
        graphs.append(g)
    for rep in range(4):
        order = (0, 1) if rep % 2 else (1, 0)
        for i in order:
            for t in outs[i]:
                t.fill_(float("nan"))
            graphs[i].replay()
            work(b1, xs[0])        # eager work of its own in between
        torch.cuda.synchronize()
        for i in (0, 1):
            for got, w in zip(outs[i], want[i]):
                assert torch.equal(got, w), (rep, i)
    new = rnd(ins[0].shape, 999, dt)   # a replay reads its inputs' new contents
    ins[0].copy_(new)
    graphs[0].replay()
    torch.cuda.synchronize()
    for got, w in zip(outs[0], work(b1, new)):
        assert torch.equal(got, w)


@gpu
def test_two_streams_at_once():
    """the same plan and weights on two streams at once: nothing is shared between the calls"""
    b = Block([200, 77, 1, 900], torch.bfloat16)
    plan = b.ops.attention_plan([1] * 3, [5000, 9000, 333], heads=8, kv_heads=2, d=128)
    qkv = [attention_inputs([1] * 3, [5000, 9000, 333], 8, 2, 128, torch.bfloat16, 400 + i) for i in range(2)]
    xs = [rnd((sum(b.ql), b.c), 500 + i, torch.bfloat16) for i in range(2)]
    want = [(*b(x), b.ops.attention_packed(plan, *t)) for x, t in zip(xs, qkv)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append((*b(xs[i]), b.ops.attention_packed(plan, *qkv[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            for a, w in zip(res, want[i]):
                assert torch.equal(a, w)


@gpu
def test_calls_are_bit_reproducible():
    b = Block([513, 33], torch.float16)
    x = rnd((546, b.c), 1, torch.float16)
    first = [t.clone() for t in b(x)]
    for _ in range(3):
        assert all(torch.equal(a, w) for a, w in zip(b(x), first))
