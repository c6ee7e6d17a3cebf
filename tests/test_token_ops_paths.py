"""More of the token-transformer operators (musev_amd.token_ops): the forms that only large, split or unusual calls reach, and the refusals
beside them.  Oracles and bounds are those of test_token_ops; a bound of its own is derived where it stands."""
import copy
import math
import pickle

import pytest
import torch

from test_token_ops import ROOT, DEV, DTYPES, IDS, attention_inputs, attention_oracle, gpu, half_step, linear_oracle, norm_oracle, rnd, rotary_oracle, subnormal, within
from test_token_ops import on_cpu  # noqa: F401  (a fixture)


def randn(shape, seed, dt, scale=1.0):
    """rnd() made on the GPU: large inputs"""
    return (torch.randn(shape, generator=torch.Generator(DEV).manual_seed(seed), device=DEV) * scale).to(dt)


# ---- packed attention: parts of split keys ------------------------------------------------------------------------------------------
SPLIT = {   # q_lens, kv_lens, heads, kv_heads: a join of many parts (shared by eight threads) and of few
    "many_parts": ([1, 3], [8192, 4000], 8, 2),
    "few_parts": ([40, 130], [1500, 1100], 4, 2),
}


def split_plan(name, d, causal=True, scale=None):
    from musev_amd import ops
    ql, kl, heads, kvh = SPLIT[name]
    plan = ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d, causal=causal, scale=scale)
    assert plan.n_joins > 0 and (plan.ws_rows > 16 * plan.n_joins * plan.join_rows) == (name == "many_parts")
    return plan


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("name", list(SPLIT))
def test_what_is_not_seen_does_not_reach_the_output_of_split_keys(name, bad, d, dt):
    """the last key of a sequence (only its last query sees it) and the rows behind the last sequence hold values that are not finite"""
    from musev_amd import ops
    ql, kl, heads, kvh = SPLIT[name]
    plan = split_plan(name, d)
    q, k, v = attention_inputs(ql, kl, heads, kvh, d, dt, 9)
    pad = torch.full((70, kvh * d), bad, dtype=dt, device=DEV)
    clean, bound = attention_oracle(q, k, v, ql, kl, heads, kvh, d, True)
    last = sum(kl) - 1
    k2, v2 = torch.cat([k, pad]), torch.cat([v, pad])
    k2[last], v2[last] = bad, bad
    got = ops.attention_packed(plan, q, k2, v2)
    torch.cuda.synchronize()
    within(got[:-1], clean[:-1], bound[:-1])
    v2 = torch.cat([v, pad])       # V alone: a visible value shows in its own column only
    v2[last, d + 5] = bad          # (of the second key / value head)
    got = ops.attention_packed(plan, q, torch.cat([k, pad]), v2)
    torch.cuda.synchronize()
    rest = torch.ones_like(got, dtype=torch.bool)
    rest.view(-1, heads, d)[-1, heads // 2:, 5] = False
    seen = got[~rest]
    assert bool((torch.isnan(seen) if math.isnan(bad) else seen == bad).all())
    within(got[rest], clean[rest], bound[rest])


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=["nan", "inf", "-inf"])
@pytest.mark.parametrize("name", list(SPLIT))
def test_a_visible_value_that_is_not_finite_shows_however_little_it_weighs(name, bad, dt, monkeypatch):
    """one key outweighs all others by e^512: the others' weights vanish, and 0 x infinity is NaN -- with the keys split into parts as without"""
    from musev_amd import ops, token_ops
    ql, kl, heads, kvh = SPLIT[name]
    d = 64
    q = torch.ones(sum(ql), heads * d, dtype=dt, device=DEV)
    k = torch.zeros(sum(kl), kvh * d, dtype=dt, device=DEV)
    v = rnd((sum(kl), kvh * d), 3, dt)
    k[600], k[kl[0] + 600] = 8, 8
    v[10, 5], v[kl[0] + 10, 5] = bad, bad
    plans = [split_plan(name, d, scale=1.0)]
    monkeypatch.setattr(token_ops, "MIN_PART", 1 << 20)
    plans.append(ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d, scale=1.0))
    assert plans[1].n_joins == 0
    for plan in plans:
        got = ops.attention_packed(plan, q, k, v).view(-1, heads, d)
        torch.cuda.synchronize()
        hit = torch.zeros_like(got, dtype=torch.bool)
        hit[:, :heads // kvh, 5] = True
        assert not bool(torch.isfinite(got[hit]).any()), plan.n_joins
        want = torch.cat([v[600].view(kvh, 1, d).expand(kvh, heads // kvh, d).reshape(1, heads, d).expand(ql[0], -1, -1),
                          v[kl[0] + 600].view(kvh, 1, d).expand(kvh, heads // kvh, d).reshape(1, heads, d).expand(ql[1], -1, -1)])
        assert torch.equal(got[~hit], want[~hit]), plan.n_joins


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("each", [2.0 ** 8, 2.0 ** 12, 2.0 ** 15 - 2.0 ** 7])
@pytest.mark.parametrize("name", list(SPLIT))
def test_parts_of_large_scores_weigh_as_they_should(name, each, dt):
    """Scores are whole numbers 63 each + 0 .. 3, exact in fp32 in any order: only their differences decide.  The keys' values say which score
    a key has.  Bound: the weights' rounding to the type (u; all are at least
    e^-3 of the largest, so none is subnormal), exponents (s - m) c with |s - m| <= 3 (2^-20), the fp32 sums (2^-19), as in
    attention_oracle without its term for the scores' error"""
    from musev_amd import ops
    ql, kl, heads, kvh = SPLIT[name]
    d = 64
    q = torch.ones(sum(ql), heads * d, dtype=dt, device=DEV)
    k = torch.full((sum(kl), kvh, d), each, dtype=dt, device=DEV)
    level = torch.cat([torch.arange(n, device=DEV) // 320 % 4 for n in kl])        # (runs of keys: parts have different maxima)
    k[:, :, -1] = level[:, None].to(dt)
    v = torch.zeros(sum(kl), kvh, d, dtype=dt, device=DEV)
    v[torch.arange(sum(kl), device=DEV), :, level] = 1.0
    plan = split_plan(name, d, causal=False, scale=1.0)
    got = ops.attention_packed(plan, q, k.view(-1, kvh * d), v.view(-1, kvh * d)).view(-1, heads, d)
    torch.cuda.synchronize()
    want = torch.zeros(sum(ql), heads, d, dtype=torch.float64, device=DEV)
    for i in range(2):
        lv = level[sum(kl[:i]):sum(kl[:i + 1])]
        w = torch.exp(lv.double() - 3)
        for x in range(4):
            want[sum(ql[:i]):sum(ql[:i + 1]), :, x] = (w * (lv == x)).sum() / w.sum()
    u = half_step(dt)
    within(got, want, (2 * u + 2.0 ** -18) * want + subnormal(dt), what=each)

# ---- packed attention: making a plan ------------------------------------------------------------------------------------------------
@gpu
def test_a_plan_does_not_wait_for_the_work_queued_on_its_stream():
    """made behind some 30 ms of work that is still running when the call returns; used at once on its own stream and on another"""
    from musev_amd import ops
    heads, kvh, d, ql, kl = 8, 2, 64, [1, 5], [3000, 77]
    q, k, v = attention_inputs(ql, kl, heads, kvh, d, torch.float16, 1)
    want, bound = attention_oracle(q, k, v, ql, kl, heads, kvh, d, True)
    a = randn((8192, 8192), 2, torch.float16)
    b, side = torch.empty_like(a), torch.cuda.Stream()
    for on_side in (False, True):
        ops.attention_packed(ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d), q, k, v)   # (pinned memory, workspaces: allocated)
        torch.cuda.synchronize()
        for _ in range(40):
            torch.matmul(a, a, out=b)
        busy = torch.cuda.Event()
        busy.record()
        plan = ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d)
        assert not busy.query()
        if on_side:
            with torch.cuda.stream(side):
                got = ops.attention_packed(plan, q, k, v)
        else:
            got = ops.attention_packed(plan, q, k, v)
        torch.cuda.synchronize()
        within(got, want, bound, what=on_side)


@gpu
def test_a_plan_is_not_made_while_a_graph_is_captured():
    from musev_amd import ops
    x = torch.zeros(4, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="before the capture"):
            ops.attention_plan([1], [300], heads=1, d=64)
        x += 1
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert bool((x == i + 1).all())


def test_a_plan_during_a_capture_is_refused_before_anything_is_uploaded(monkeypatch):
    from musev_amd import ops
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(ValueError, match="before the capture"):
        ops.attention_plan([1], [300], heads=1, d=64, device="cuda:0")
    assert ops.attention_plan([1], [300], heads=1, d=64, device="cpu").total_kv == 300

def test_first_key_rows_of_a_plan():
    from musev_amd import ops, token_ops
    ok = dict(heads=4, kv_heads=2, d=64, device="cpu")
    ql, kl, first = [1, 3, 0, 2], [700, 0, 5, 300], [1000, 9000, 3, 0]
    plan = ops.attention_plan(ql, kl, kv_first=torch.tensor(first), **ok)
    assert plan.kv_first == (1000, 9000, 3, 0) and plan.total_kv == 1700 and plan.total_q == 6
    packed, placed = (token_ops._plan_items(ql, kl, 2, 2, True, 64, f) for f in (None, first))
    assert packed[1:] == placed[1:]          # (joins know no key rows)
    row = dict(zip([0, 700, 700, 705], first))
    assert [(*i[:2], row[i[2]] if i[3] else 9000, *i[3:]) for i in packed[0]] == placed[0]
    assert ops.attention_plan(ql, kl, **ok).kv_first == (0, 700, 700, 705) and ops.attention_plan(ql, kl, **ok).total_kv == 1005
    assert ops.attention_plan([2], [0], kv_first=[7], **ok).total_kv == 0
    for bad in ([1], [0, 0, 0, -1], [0, 0, 0, 2 ** 31 - 200]):
        with pytest.raises(ValueError, match="kv_first"):
            ops.attention_plan(ql, kl, kv_first=bad, **ok)
    with pytest.raises(TypeError):
        ops.attention_plan(ql, kl, kv_first=[0.5, 0, 0, 0], **ok)


@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
def test_attention_over_a_cache_that_grows(dt):
    """a cache with room for every request: two tokens at once, then one per step, some requests idle; what lies in the room (NaN) is not seen"""
    from musev_amd import ops
    heads, kvh, d, room = 8, 2, 80, [1500, 64, 9, 700]
    first = [sum(room[:i]) + 3 * i for i in range(4)]
    lens = [1490, 0, 1, 600]
    cache = [torch.full((sum(room) + 12, kvh * d), float("nan"), dtype=dt, device=DEV) for _ in range(2)]
    for i, t in enumerate(cache):
        for f, n in zip(first, lens):
            t[f:f + n] = rnd((n, kvh * d), 5 + i, dt)
    for step, new in enumerate(([2, 2, 2, 2], [1, 1, 1, 1], [1, 1, 0, 1], [0, 1, 1, 1], [1, 0, 0, 1])):
        q, k, v = (rnd((sum(new), h * d), 10 * step + i, dt) for i, h in enumerate((heads, kvh, kvh)))
        at = torch.tensor([f + n + j for f, n, m in zip(first, lens, new) for j in range(m)], device=DEV)
        cache[0][at], cache[1][at] = k, v
        lens = [n + m for n, m in zip(lens, new)]
        got = ops.attention_packed(ops.attention_plan(new, lens, heads=heads, kv_heads=kvh, d=d, kv_first=first), q, *cache)
        torch.cuda.synchronize()
        rows = torch.tensor([f + j for f, n in zip(first, lens) for j in range(n)], device=DEV)
        within(got, *attention_oracle(q, cache[0][rows], cache[1][rows], new, lens, heads, kvh, d, True), what=step)


@gpu
def test_requests_that_share_a_prefix_of_keys():
    from musev_amd import ops
    dt, heads, kvh, d = torch.float16, 4, 2, 64
    ql, kl, first = [1, 3, 1], [900, 650, 650], [0, 0, 250]
    q, k, v = rnd((5, heads * d), 1, dt), rnd((900, kvh * d), 2, dt), rnd((900, kvh * d), 3, dt)
    plan = ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d, kv_first=first)
    assert plan.total_kv == 900
    got = ops.attention_packed(plan, q, k, v)
    torch.cuda.synchronize()
    rows = torch.cat([torch.arange(f, f + n) for f, n in zip(first, kl)]).to(DEV)
    within(got, *attention_oracle(q, k[rows], v[rows], ql, kl, heads, kvh, d, True))
    with pytest.raises(ValueError, match="k "):
        ops.attention_packed(plan, q, k[:899], v)

def test_plans_and_tables_do_not_go_by_the_default_device():
    from musev_amd import ops
    with torch.device("meta"):
        plan, table = ops.attention_plan([3, 700], heads=1, d=64, device="cpu"), ops.rotary_table([16, 8], device="cpu")
    assert plan.device.type == table.device.type == "cpu"
    assert [t.tolist() for t in plan._tensors] == [t.tolist() for t in ops.attention_plan([3, 700], heads=1, d=64, device="cpu")._tensors]


@gpu
def test_a_plan_beside_a_default_device():
    from musev_amd import ops
    with torch.device(DEV):
        plan = ops.attention_plan([3, 700], heads=1, d=64)
    q, k, v = attention_inputs([3, 700], [3, 700], 1, 1, 64, torch.float16, 1)
    got = ops.attention_packed(plan, q, k, v)
    torch.cuda.synchronize()
    within(got, *attention_oracle(q, k, v, [3, 700], [3, 700], 1, 1, 64, True))


# ---- rotary positions: several tokens per block, results and inputs past the caches ----------------------------------------------
MANY = {   # tokens, heads, kv_heads, d, sections
    "four_tokens_per_block": (4097, 1, 1, 16, [16]),
    "eight_tokens_per_block": (20003, 2, 1, 24, [8, 14]),
    "two_tokens_per_block": (2049, 6, 3, 40, [8, 8, 16]),
    "results_past_the_caches": (20001, 10, 3, 128, [32, 48, 48]),
    "inputs_past_the_last_cache": (20001, 45, 8, 128, [32, 48, 44]),
}


@gpu
@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
@pytest.mark.parametrize("name", list(MANY))
def test_rotary_of_many_tokens(name, pairing):
    """aligned and one element off it, apart and in place; the last block holds fewer tokens than the others"""
    from musev_amd import ops
    n, heads, kvh, d, sec = MANY[name]
    dt = torch.float16 if pairing == "halves" else torch.bfloat16
    pos = torch.randint(0, 4096, (n, len(sec)), generator=torch.Generator(DEV).manual_seed(1), dtype=torch.int32, device=DEV)
    table = ops.rotary_table(sec)
    wide = randn((n, (heads + kvh) * d + 3), 2, dt)
    for off in (0, 1):
        src = wide[:, off:off + (heads + kvh) * d]
        q, k = src[:, :heads * d], src[:, heads * d:]
        keep = wide.clone()
        oq, ok = ops.rotary_axes(q, k, pos, table, heads=heads, kv_heads=kvh, d=d, pairing=pairing)
        torch.cuda.synchronize()
        for got, x, h in ((oq, q, heads), (ok, k, kvh)):
            for a in range(0, n, 4096):
                within(got[a:a + 4096], *rotary_oracle(x[a:a + 4096], pos[a:a + 4096], sec, 10000.0, False, h, d, pairing), what=(name, off, a))
        ops.rotary_axes(q, k, pos, table, heads=heads, kv_heads=kvh, d=d, pairing=pairing, out_q=q, out_k=k)
        torch.cuda.synchronize()
        assert torch.equal(q, oq) and torch.equal(k, ok)
        cols = slice(off + (heads + kvh) * d, None)
        assert torch.equal(wide[:, :off], keep[:, :off]) and torch.equal(wide[:, cols], keep[:, cols])
        wide = keep


# ---- gated residual norm: inputs past the last-level cache --------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("c,off,dt", [(1001, 3, torch.float16), (1280, 0, torch.bfloat16), (44, 1, torch.float16), (4100, 2, torch.bfloat16)])
def test_gated_norm_of_inputs_past_the_last_cache(c, off, dt):
    """in place, odd widths and columns off their alignment, a row per wave and rows that share one"""
    from musev_amd import ops
    rows = (256 << 20) // (4 * c) + 61
    x, f = (randn((rows, c + 5), s, dt)[:, off:off + c] for s in (1, 2))
    gate, scale, shift = (rnd((7, c), 43 + i, dt, 0.5) for i in range(3))
    pre, per = (rnd((c,), 52, dt, 0.3) + 1, None, 1e-6), -(-rows // 7)
    x0, f0 = x.clone(), f.clone()
    s, h = ops.gated_residual_norm(x, f, alpha=0.75, pre=pre, gate=gate, scale=scale, shift=shift, rows_per_group=per, out=x, norm_out=f)
    torch.cuda.synchronize()
    for a in range(0, rows, 200_000_000 // (8 * c)):
        e = min(rows, a + 200_000_000 // (8 * c))
        ws, wh = norm_oracle(x0[a:e], f0[a:e], "layer", 0.75, None, pre, gate, scale, shift, torch.arange(a, e, device=DEV) // per)
        within(s[a:e], *ws, what=("s", c, a))
        within(h[a:e], *wh, what=("h", c, a))

# ---- int8 projection: narrow and flat results --------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(49152, 200, 64), (49300, 130, 130), (26624, 320, 320), (26700, 100, 264), (25000, 150, 385), (60, 140, 49300), (300, 90, 25700)])
def test_linear_i8_of_few_columns_or_rows(m, k, n, dt):
    """many tiles of the largest size, mostly empty or just not"""
    from musev_amd import ops
    x = randn((m, k), 1, dt)
    codes = torch.randint(-127, 128, (n, k), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(torch.int8).to(DEV)
    ws = ((0.5 + torch.rand(n, generator=torch.Generator().manual_seed(3))) / (73 * math.sqrt(k))).to(DEV)
    bias, w, res = rnd((n,), 3, dt), ops.pack_weight_i8(codes, ws), randn((m, n + 3), 4, dt)[:, 1:1 + n]
    for r, act in ((None, ops.MV_ACT_SILU), (res, 0)):
        got = ops.linear_i8(x, w, bias=bias, residual=r, act=act)
        torch.cuda.synchronize()
        for a in range(0, m, 8192):
            within(got[a:a + 8192], *linear_oracle(x[a:a + 8192], codes, ws, bias, None if r is None else r[a:a + 8192], act == ops.MV_ACT_SILU), what=(m, k, n, a))

# ---- copies of plans, tables and weights --------------------------------------------------------------------------------------------
COPIES = {"deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x)), "copy": copy.copy}


@pytest.mark.parametrize("how", list(COPIES))
def test_copies_hold_addresses_of_their_own_memory(how):
    from musev_amd import ops
    w = ops.Int8Rows(torch.arange(256, dtype=torch.int8).view(2, 128), torch.tensor([1.0, 2.0]), 100)
    table = ops.rotary_table([16, 8], device="cpu")
    plan = ops.attention_plan([1, 3], [5000, 7], kv_first=[9, 0], heads=4, kv_heads=2, d=64, device="cpu", scale=0.5, causal=False)
    w2, table2, plan2 = (COPIES[how](x) for x in (w, table, plan))
    assert (w2._codes, w2._scale) == (w2.codes.data_ptr(), w2.scale.data_ptr()) and torch.equal(w2.codes, w.codes) and torch.equal(w2.scale, w.scale) and w2.k == 100
    assert (table2._turns, table2._axis) == tuple(t.data_ptr() for t in table2._tensors) and (table2.pairs, table2.axes) == (12, 2)
    assert plan2._tables == tuple(t.data_ptr() for t in plan2._tensors)
    skip = {"_tensors", "_tables", "_streams", "_ready"}
    assert {k: v for k, v in vars(plan2).items() if k not in skip} == {k: v for k, v in vars(plan).items() if k not in skip}
    for a, b in ((w, w2), (table, table2), (plan, plan2)):
        assert all(torch.equal(x, y) for x, y in zip(a._tensors, b._tensors))
        if how != "copy":
            assert all(x.data_ptr() != y.data_ptr() for x, y in zip(a._tensors, b._tensors))


@gpu
def test_a_copy_outlives_what_it_was_copied_from():
    from musev_amd import ops
    dt, ql, kl, heads, kvh, d = torch.float16, [1, 3], [5000, 70], 4, 2, 64
    q, k, v = attention_inputs(ql, kl, heads, kvh, d, dt, 1)
    x = rnd((20, 200), 2, dt)
    codes = torch.randint(-127, 128, (64, 200), generator=torch.Generator().manual_seed(3), dtype=torch.int32).to(torch.int8).to(DEV)
    pos = torch.arange(20, dtype=torch.int32, device=DEV).view(20, 1)
    first = [ops.attention_plan(ql, kl, heads=heads, kv_heads=kvh, d=d), ops.pack_weight_i8(codes, torch.full((64,), 0.01, device=DEV)), ops.rotary_table([200])]

    def run(plan, w, table):
        return ops.attention_packed(plan, q, k, v), ops.linear_i8(x, w), ops.rotary_axes(x, None, pos, table, heads=1, d=200)[0]
    want = [t.clone() for t in run(*first)]
    for how in ("deepcopy", "pickle"):
        second = [COPIES[how](t) for t in first]
        torch.cuda.synchronize()
        for t in first[1:]:
            for m in t._tensors:
                m.fill_(0)        # (as another tensor in the freed memory would: no code, no turn)
        assert second[0]._tables == tuple(t.data_ptr() for t in second[0]._tensors)
        got = run(*second)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), how
        first = second


# ---- refusals -----------------------------------------------------------------------------------------------------------------------
def test_tensors_with_a_forward_mode_tangent_are_refused(on_cpu):  # noqa: F811
    import torch.autograd.forward_ad as fw
    from musev_amd import ops
    x, c = torch.zeros(6, 64, dtype=torch.float16), torch.zeros(64, dtype=torch.float16)
    plan, table = ops.attention_plan([6], heads=1, d=64, device="cpu"), ops.rotary_table([64], device="cpu")
    w = ops.Int8Rows(torch.zeros(64, 128, dtype=torch.int8), torch.ones(64), 64)
    pos = torch.zeros(6, 1)
    calls = (lambda x, c, p: ops.attention_packed(plan, x, x, x), lambda x, c, p: ops.rotary_axes(x, None, p, table, heads=1, d=64),
             lambda x, c, p: ops.gated_residual_norm(x, x, pre=(c, None, 1e-6)), lambda x, c, p: ops.linear_i8(x, w, bias=c),
             lambda x, c, p: ops.gemm_i8(w, w, bias=c), lambda x, c, p: ops.linear_i8(x, w, residual=x))
    with fw.dual_level():
        tx, tc, tp = (fw.make_dual(t, torch.ones_like(t)) for t in (x, c, pos))
        for i, call in enumerate(calls):
            with pytest.raises(on_cpu):
                call(x, c, pos.int())
            for args in ([(tx, c, pos)] if i in (0, 5) else [(x, tc, pos)] if i == 4 else [(tx, c, pos), (x, tc, tp)]):
                with pytest.raises(ValueError, match="tangent"):
                    call(*args)
                with torch.no_grad(), pytest.raises(ValueError, match="tangent"):   # (no_grad does not switch forward mode off)
                    call(*args)


def test_int8_scales_that_require_gradients_are_refused(on_cpu):  # noqa: F811
    import torch.autograd.forward_ad as fw
    from musev_amd import ops
    codes, scale = torch.zeros(64, 128, dtype=torch.int8), torch.ones(64)
    learnt = torch.ones(64, requires_grad=True)
    x, plain = torch.zeros(6, 128, dtype=torch.float16), ops.Int8Rows(codes, scale, 128)

    def calls(s):
        w = ops.Int8Rows(codes, s, 128)
        return (lambda: ops.linear_i8(x, w), lambda: ops.gemm_i8(plain, w), lambda: ops.gemm_i8(w, plain))
    for call in calls(learnt):
        with pytest.raises(ValueError, match="scale: requires gradients"):
            call()
        with torch.no_grad(), pytest.raises(on_cpu):
            call()
    with pytest.raises(ValueError, match="scale: requires gradients"):
        ops.pack_weight_i8(codes, learnt)
    with torch.no_grad():
        assert not ops.pack_weight_i8(codes, learnt).scale.requires_grad
    with fw.dual_level():
        dual = fw.make_dual(scale, torch.ones_like(scale))
        for call in (*calls(dual), lambda: ops.pack_weight_i8(codes, dual)):
            with pytest.raises(ValueError, match="tangent"):
                call()


def test_calls_of_more_work_than_a_launch_has_are_refused():
    """a launch has fewer than 2^32 work items: one block more than that is an error of its own, before anything is launched"""
    import ctypes as C
    from musev_amd import _lib
    lib = _lib.load()

    def refused(rc):
        assert rc == -1 and b"2^32 work items" in lib.mv_last_error(), (rc, lib.mv_last_error())
    n = _lib.GatedNormDesc()
    n.x = n.f = n.stream_out = 16
    n.groups = 1
    for c, per_block in ((8, 16), (200, 8), (512, 8), (1280, 4), (2048, 1), (16384, 1)):
        n.c, n.rows = c, ((1 << 24) - 1) * per_block + 1
        refused(lib.mv_gated_residual_norm(C.byref(n), None))
    r = _lib.RotaryDesc()
    r.q = r.out_q = r.positions = r.turns = r.axis = 16
    r.heads, r.d, r.pairs, r.axes, r.tokens = 1, 8, 4, 1, ((1 << 24) - 1) * 8 + 1
    refused(lib.mv_rotary_axes(C.byref(r), None))
    for k, kp, per_block in ((100, 128, 4), (2000, 2048, 1)):
        refused(lib.mv_quantize_rows_i8(16, k, ((1 << 24) - 1) * per_block + 1, k, 0, 16, kp, 16, None))
    a = _lib.AttnPackedDesc()
    a.q = a.k = a.v = a.out = a.items = a.joins = a.workspace = 16
    a.workspace_bytes, a.heads, a.kv_heads, a.d, a.scale = 1 << 50, 4, 2, 64, 0.125
    a.ldq = a.ldo = 256
    a.ldk = a.ldv = 128
    a.n_items = 1 << 23
    refused(lib.mv_attention_packed(C.byref(a), None))
    a.n_items, a.n_joins, a.join_rows = 1, 1 << 20, 128
    refused(lib.mv_attention_packed(C.byref(a), None))
    w = _lib.LinearI8Desc()
    w.x = w.w = w.w_scale = w.out = w.workspace = 16
    w.M, w.N, w.K, w.kp, w.ldx, w.ldw, w.ldo = 1, 2 ** 31 - 1, 100, 128, 100, 128, 8
    refused(lib.mv_linear_i8(C.byref(w), None))
    g = _lib.GemmI8Desc()
    g.a = g.w = g.a_scale = g.w_scale = g.out = 16
    g.M, g.N, g.kp, g.lda, g.ldw, g.ldo = 4, 1 << 27, 128, 128, 128, 8
    refused(lib.mv_gemm_i8(C.byref(g), None))
    g.M, g.N = 2 ** 31 - 1, 2 ** 31 - 1
    refused(lib.mv_gemm_i8(C.byref(g), None))


def test_the_gated_norm_refuses_factors_past_fp32(on_cpu):  # noqa: F811
    from musev_amd import ops
    x = torch.zeros(6, 40, dtype=torch.float16)
    top = torch.finfo(torch.float32).max
    for kw, match in ((dict(pre=(None, None, 1e39)), "eps"), (dict(post=(None, None, 1e300)), "eps"), (dict(alpha=1e39), "alpha"), (dict(alpha=-1e39), "alpha")):
        with pytest.raises(ValueError, match=match):
            ops.gated_residual_norm(x, x, **kw)
    for kw in (dict(pre=(None, None, top)), dict(alpha=-top), dict(alpha=float("inf")), dict(alpha=float("nan"))):
        with pytest.raises(on_cpu):
            ops.gated_residual_norm(x, x, **kw)


def test_operators_are_importable_beside_a_torch_without_a_gpu_build():
    """such a build has no stream handles; the operators need them only when they launch"""
    import subprocess
    import sys
    code = ("import torch\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n    delattr(torch._C, n)\n"
            "from musev_amd import ops\nassert ops.attention_plan([4], heads=1, d=64, device='cpu').total_q == 4")
    assert subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT).returncode == 0
