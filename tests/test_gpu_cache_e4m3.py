"""The 8-bit paged cache: appending with the rotation on the way and attention over it, against the formulas in 64 bits."""
import math

import pytest
import torch

from cajeta_llm_b200.csrc import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
HALF = 2.0 ** -8           # a rounding to bfloat16, half a step


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make_cache(pages, kv, page_tokens, hd, seed=0, spread=3.0):
    """Codes of any value (a few of them zero) and exponents of any size within `spread` octaves; what they stand for."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn((pages, kv, page_tokens, hd), generator=g, device=DEV) * 60
        x[torch.rand(x.shape, generator=g, device=DEV) < 0.01] = 0
        codes = x.clamp(-448, 448).to(torch.float8_e4m3fn)
        e = (torch.rand(x.shape[:-1], generator=g, device=DEV) * 2 * spread - spread - 8).round().to(torch.int32)
        out.append((codes, (e + 127).to(torch.uint8)))
    return out


def stands_for(codes, exponents):
    return codes.to(F64) * torch.exp2(exponents.to(F64) - 127)[..., None]


def tables(lengths, page_tokens, seed=0, extra=3):
    """Pages of requests in mixed order, -1 where a request has none."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page_tokens) for n in lengths]
    order = torch.randperm(sum(need) + extra, generator=g).tolist()
    width, rows, at = max(need + [1]) + 1, [], 0
    for n in need:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return ints(rows), sum(need) + extra


def attention(q, rows, k, v, table, page_tokens, kv, window, scale):
    """Rows [(request, position)] in 64 bits: the result and sum of weight times |value| (what a rounding of weights can move)."""
    T, heads, hd = q.shape
    out, size = torch.zeros((T, heads, hd), dtype=F64, device=DEV), torch.zeros((T, heads, hd), dtype=F64, device=DEV)
    group = heads // kv
    for t, (r, p) in enumerate(rows):
        if r < 0:
            continue
        pages = table[r, :p // page_tokens + 1].long()
        lo = max(0, p + 1 - window) if window else 0
        kk, vv = (x[pages].permute(1, 0, 2, 3).reshape(kv, -1, hd)[:, lo:p + 1] for x in (k, v))
        w = torch.softmax((q[t].to(F64).view(kv, group, hd) @ kk.transpose(1, 2)) * scale, dim=-1)
        out[t], size[t] = (w @ vv).view(heads, hd), (w @ vv.abs()).view(heads, hd)
    return out, size


def close(got, want, size):
    # the result's rounding, the weights' (portions: to bfloat16, 2^-8 of each; single rows: a rest of 2^-4 is rounded to 2^-4 of itself),
    # and 2^-12 for exponentials of float32 scores
    worst = ((got.to(F64) - want).abs() - HALF * want.abs() - (2.0 ** -8 + 2.0 ** -12) * size).max()
    assert float(worst) <= 1e-30, float(worst)


# ---- appending ----------------------------------------------------------------------------------------------------------

def exponent_of(most):
    if most == 0:
        return -100
    return min(max(math.ceil(math.log2(most / 448.0)), -100), 119)


@pytest.mark.parametrize("heads,kv,hd,rot,page_tokens,rows", [
    (4, 2, 128, 128, 16, 5), (16, 16, 128, 64, 16, 1), (28, 4, 128, 128, 32, 37), (14, 2, 64, 64, 16, 300), (3, 1, 64, 6, 5, 9),
    (8, 8, 64, 0, 16, 8), (2, 1, 128, 126, 1, 3)])
def test_append_rotates_and_writes_what_the_formula_says(heads, kv, hd, rot, page_tokens, rows):
    g = torch.Generator(device=DEV)
    g.manual_seed(rows)
    pad = 6
    wide = torch.randn((rows, (heads + 2 * kv) * hd + pad), generator=g, device=DEV) * 3
    wide[0] *= 1e-3
    wide[rows // 2, heads * hd:(heads + 1) * hd] = 0                     # a key of zeros
    start = [max(0, p) for p in (0, 100_003, 31_999)]
    reqs = [i % 3 for i in range(rows)]
    positions = [start[r] + i // 3 for i, r in enumerate(reqs)]
    lengths = [max([p + 1 for p, q in zip(positions, reqs) if q == r] + [1]) for r in range(3)]
    table, pages = tables(lengths, page_tokens)
    sentinel = torch.full((pages, kv, page_tokens, hd), 0x35, dtype=torch.uint8, device=DEV)
    k, v = sentinel.clone().view(torch.float8_e4m3fn), sentinel.clone().view(torch.float8_e4m3fn)
    ke, ve = (torch.full((pages, kv, page_tokens), 200, dtype=torch.uint8, device=DEV) for _ in range(2))
    inv = (10000.0 ** (-torch.arange(0, max(rot, 2), 2, dtype=F64) / max(rot, 2))).to(torch.float32).to(DEV)
    q = torch.empty((rows, heads, hd), dtype=torch.bfloat16, device=DEV)
    K.rope_kv_write_e4m3(wide, pad, pad + heads * hd, pad + (heads + kv) * hd, q, k, v, ke, ve, ints(positions), ints(reqs), table, page_tokens,
                         heads, kv, hd, rot, inv if rot else None, True)
    x = wide[:, pad:].to(F64)
    parts = [t.reshape(rows, -1, hd) for t in x.split([heads * hd, kv * hd, kv * hd], dim=1)]
    if rot:
        a = torch.tensor(positions, dtype=F64, device=DEV)[:, None] * inv.to(F64)
        c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
        for i in (0, 1):
            lo, hi, rest = parts[i].split([rot // 2, rot // 2, hd - rot], dim=-1)
            parts[i] = torch.cat([lo * c - hi * s, lo * s + hi * c, rest], dim=-1)
    # two products of float32 and the angle's cosine (2^-22 of the pair's larger entry), then the rounding
    assert ((q.to(F64) - parts[0]).abs() <= HALF * parts[0].abs() + 2.0 ** -20 * parts[0].abs().amax(-1, keepdim=True)).all()
    seen = torch.zeros(ke.shape, dtype=torch.bool, device=DEV)
    for t in range(rows):
        page, at = int(table[reqs[t], positions[t] // page_tokens]), positions[t] % page_tokens
        seen[page, :, at] = True
        for plane, exps, want in ((k, ke, parts[1][t]), (v, ve, parts[2][t])):
            for h in range(kv):
                e = int(exps[page, h, at]) - 127
                most = float(want[h].abs().max())
                assert e == exponent_of(most) or abs(most / 448 / 2.0 ** round(math.log2(most / 448)) - 1) < 1e-5
                got = plane[page, h, at].to(F64) * 2.0 ** e
                # half a step: 2^-4 of the value, or half the smallest code
                assert ((got - want[h]).abs() <= (2.0 ** -4 * want[h].abs()).clamp(min=2.0 ** (e - 10)) * (1 + 1e-4) + 2.0 ** -20 * most).all()
    for plane, exps in ((k, ke), (v, ve)):
        assert (plane.view(torch.uint8)[~seen] == 0x35).all() and (exps[~seen] == 200).all()      # nothing else was touched


def test_append_of_rows_without_a_place_of_extreme_values_and_of_queries_alone():
    heads, kv, hd, P = 2, 2, 64, 16
    x = torch.zeros((5, 6 * hd), device=DEV)
    x[0, 2 * hd:] = 3.3e38
    x[1, 2 * hd:] = 1e-44
    x[2, 2 * hd:3 * hd] = float("inf")
    x[3, 2 * hd + 1] = float("nan")
    x[4] = 1.0
    table = ints([[0, -1], [1, 2]])
    k, v = (torch.zeros((3, kv, P, hd), device=DEV).to(torch.float8_e4m3fn) for _ in range(2))
    ke, ve = (torch.zeros((3, kv, P), dtype=torch.uint8, device=DEV) for _ in range(2))
    q = torch.empty((5, heads, hd), dtype=torch.bfloat16, device=DEV)

    def go(positions, reqs, write=True):
        K.rope_kv_write_e4m3(x, 0, 2 * hd, 4 * hd, q, k, v, ke, ve, ints(positions), ints(reqs), table, P, heads, kv, hd, 0, None, write)

    go([17, 40, 3, 5, -1], [0, 1, -1, 2, 0])         # no page, past the table, no request, no request, no position
    assert not k.view(torch.uint8).any() and not ke.any() and not ve.any()
    assert (q[4] == 1).all()
    go([0, 1, 2, 3, 4], [0] * 5, write=False)
    assert not ke.any()
    go([0, 1, 2, 3, 4], [0] * 5)
    assert int(ke[0, 0, 0]) == 119 + 127 and (k[0, 0, 0].float() == 448).all()                     # cut to the largest that is held
    assert int(ke[0, 0, 1]) == 27 and not k[0, 0, 1].float().any()                                 # below what is held: zeros
    assert int(ke[0, 0, 2]) == 119 + 127 and (k[0, 0, 2].float() == 448).all()
    assert torch.isnan(k[0, 0, 3].float()[1]) and not k[0, 0, 3].float()[2:].any()
    assert (k[0, 0, 4].float() == 256).all() and int(ke[0, 0, 4]) == 127 - 8


# ---- single rows --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,hd,page_tokens,window,splits", [
    (4, 4, 128, 16, 0, 0), (28, 4, 128, 16, 0, 0), (14, 2, 64, 16, 0, 3), (12, 1, 128, 16, 0, 1), (40, 2, 64, 5, 0, 2), (16, 16, 64, 64, 0, 7),
    (8, 2, 128, 16, 33, 0), (17, 1, 128, 7, 100, 4), (4, 1, 64, 1, 1, 0)])
def test_decoded_rows(heads, kv, hd, page_tokens, window, splits):
    lengths = [1, 2, 31, 32, 33, 64, 127, 128, 129, 300, 777, 1]
    table, pages = tables(lengths, page_tokens, seed=hd)
    (k, ke), (v, ve) = make_cache(pages, kv, page_tokens, hd, seed=heads)
    rows = [(r, n - 1) for r, n in enumerate(lengths)]
    rows[-1] = (-1, 5)                                                          # no request: zeros
    rows.append((9, 250))                                                       # a second row of a request, at an earlier position
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    q = (torch.randn((len(rows), heads, hd), generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    q[2] *= 1e-20
    q[3] = 0
    q[4] *= 1e-3
    scale = 1 / math.sqrt(hd)
    out = torch.full_like(q, 7.0)
    K.decode_attention_e4m3(q, out, k, v, ke, ve, ints([p for _, p in rows]), ints([r for r, _ in rows]), table, page_tokens, heads, kv, hd,
                            window, scale, max(lengths), splits=splits)
    want, size = attention(q, rows, stands_for(k, ke), stands_for(v, ve), table, page_tokens, kv, window, scale)
    close(out, want, size)
    again = torch.empty_like(out)
    K.decode_attention_e4m3(q, again, k, v, ke, ve, ints([p for _, p in rows]), ints([r for r, _ in rows]), table, page_tokens, heads, kv, hd,
                            window, scale, max(lengths), splits=splits)
    assert torch.equal(out, again)


def test_values_of_far_apart_exponents_and_unseen_nan():
    """A first value thousands of octaves above the others' weight, then below it; NaN in keys and values past the row's position."""
    heads, kv, hd, P, n = 4, 2, 128, 16, 200
    table, pages = tables([256], P)
    for order in (1, -1):
        (k, ke), (v, ve) = make_cache(pages, kv, P, hd, seed=5)
        at = torch.arange(256, device=DEV)
        octave = ((at.float() / 255) * 60 - 30).round().to(torch.int32) * order + 127 - 8
        ve[table[0, at // P].long(), :, at % P] = octave.to(torch.uint8)[:, None]
        hidden = at[n:]
        for plane in (k, v):
            plane.view(torch.uint8)[table[0, hidden // P].long(), :, hidden % P] = 0x7f          # NaN
        q = torch.randn((1, heads, hd), device=DEV).to(torch.bfloat16)
        out = torch.empty_like(q)
        K.decode_attention_e4m3(q, out, k, v, ke, ve, ints([n - 1]), ints([0]), table, P, heads, kv, hd, 0, 0.05, 256)
        ks, vs = (torch.nan_to_num(stands_for(c, e)) for c, e in ((k, ke), (v, ve)))
        want, size = attention(q, [(0, n - 1)], ks, vs, table, P, kv, 0, 0.05)
        close(out, want, size)
        many = torch.empty((n, heads, hd), dtype=torch.bfloat16, device=DEV)
        qs = torch.randn((n, heads, hd), device=DEV).to(torch.bfloat16)
        K.prefill_attention_e4m3(qs, many, k, v, ke, ve, ints([0, n]), ints([0]), table, P, heads, kv, hd, 0, 0.05)
        want, size = attention(qs, [(0, p) for p in range(n)], ks, vs, table, P, kv, 0, 0.05)
        close(many, want, size)


# ---- portions of prompts ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv,hd,page_tokens,window,portions", [
    (4, 4, 128, 16, 0, [(0, 300)]),
    (28, 4, 128, 16, 0, [(0, 1), (130, 257), (5, 2)]),
    (14, 2, 64, 16, 0, [(200, 129), (0, 128)]),
    (4, 1, 128, 16, 50, [(0, 300), (333, 64)]),
    (6, 2, 64, 16, 200, [(500, 333), (0, 0), (700, 1)]),
    (3, 3, 128, 5, 0, [(7, 140), (0, 20)]),
    (5, 1, 64, 128, 300, [(1000, 200)]),
    (2, 2, 128, 16, 0, [(2000, 130)]),
    (16, 2, 128, 16, 1, [(0, 150)])])
def test_portions_of_prompts(heads, kv, hd, page_tokens, window, portions):
    lengths = [p + n for p, n in portions]
    table, pages = tables(lengths, page_tokens, seed=heads)
    (k, ke), (v, ve) = make_cache(pages, kv, page_tokens, hd, seed=hd + heads)
    rows = [(r, p + i) for r, (p, n) in enumerate(portions) for i in range(n)]
    start = [0]
    for _, n in portions:
        start.append(start[-1] + n)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    spare = 3
    q = (torch.randn((len(rows) + spare, heads, hd), generator=g, device=DEV) * 1.5).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    scale = 1 / math.sqrt(hd)
    # requests that a layout is filled up with bring no rows and have no pages
    filled = torch.cat([table, torch.full_like(table[:1], -1)])
    K.prefill_attention_e4m3(q, out, k, v, ke, ve, ints(start + start[-1:]), ints([p for p, _ in portions] + [0]), filled, page_tokens, heads, kv,
                             hd, window, scale)
    assert (out[len(rows):] == 7.0).all()                                       # rows of no request are left as they were
    want, size = attention(q[:len(rows)], rows, stands_for(k, ke), stands_for(v, ve), table, page_tokens, kv, window, scale)
    close(out[:len(rows)], want, size)
    assert not K.wait_errors()


def test_a_captured_step_reads_new_inputs_and_two_graphs_share_no_scratch():
    heads, kv, hd, P = 8, 2, 128, 16
    table, pages = tables([700, 900], P)
    (k, ke), (v, ve) = make_cache(pages, kv, P, hd)
    inv = (10000.0 ** (-torch.arange(0, hd, 2, dtype=F64) / hd)).to(torch.float32).to(DEV)
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    ints_01 = ints([0, 1])                     # (the graphs read it: it lives as long as they do)
    for _ in range(2):
        s = dict(x=torch.randn((2, (heads + 2 * kv) * hd), device=DEV), pos=ints([5, 6]), q=torch.empty((2, heads, hd), dtype=torch.bfloat16, device=DEV))

        def step(s=s):
            K.rope_kv_write_e4m3(s["x"], 0, heads * hd, (heads + kv) * hd, s["q"], k, v, ke, ve, s["pos"], ints_01, table, P, heads, kv, hd, hd, inv, True)
            out = torch.empty_like(s["q"])
            K.decode_attention_e4m3(s["q"], out, k, v, ke, ve, s["pos"], ints_01, table, P, heads, kv, hd, 0, 0.09, 900)
            return out

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            s["out"] = step()
        graphs.append((graph, s, step))
    for i, (graph, s, step) in enumerate(graphs):
        s["x"].normal_()
        s["pos"].copy_(ints([600 + i, 850 + i]))
    for graph, _, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    got = [s["out"].clone() for _, s, _ in graphs]
    for (_, s, step), out in zip(graphs, got):
        assert torch.equal(step(), out)


def test_another_stream_than_the_default_one():
    heads, kv, hd, P = 4, 4, 64, 16
    table, pages = tables([100], P)
    (k, ke), (v, ve) = make_cache(pages, kv, P, hd)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        q = torch.randn((40, heads, hd), device=DEV).to(torch.bfloat16)
        out = torch.empty_like(q)
        K.prefill_attention_e4m3(q, out, k, v, ke, ve, ints([0, 40]), ints([60]), table, P, heads, kv, hd, 0, 0.1)
    side.synchronize()
    want, size = attention(q, [(0, 60 + i) for i in range(40)], stands_for(k, ke), stands_for(v, ve), table, P, kv, 0, 0.1)
    close(out, want, size)


@pytest.mark.parametrize("heads,kv,hd,rows,splits", [(16, 16, 128, 1, 8), (20, 1, 64, 3, 2), (8, 2, 128, 2, 5), (16, 16, 128, 9, 8), (8, 8, 64, 70, 3)])
def test_a_rows_blocks_join_in_a_cluster_and_in_a_kernel_alike(heads, kv, hd, rows, splits):
    """Both ways, whichever the sizes choose: of stretches without keys too, and of a row that sees none."""
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + splits)
    pages, page = 8 * rows, 16
    k, v = ((torch.randn((pages, kv, page, hd), generator=g, device=DEV)).to(torch.float8_e4m3fn) for _ in range(2))
    ke, ve = (torch.randint(120, 132, (pages, kv, page), generator=g, device=DEV).to(torch.uint8) for _ in range(2))
    q = torch.randn((rows, heads, hd), generator=g, device=DEV).to(torch.bfloat16)
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(rows, 8)
    positions = (torch.arange(rows, device=DEV) * 37 % 128).to(torch.int32)
    req = torch.arange(rows, device=DEV, dtype=torch.int32)
    req[-1] = -1 if rows > 1 else 0
    got = []
    for cluster in (True, False):
        out = torch.full_like(q, 7.0)
        with pytest.MonkeyPatch.context() as m:
            m.setattr(K, "_e4m3_cluster", lambda *a: cluster)
            K.decode_attention_e4m3(q, out, k, v, ke, ve, positions, req, table, page, heads, kv, hd, 0, hd ** -0.5, 128, splits=splits)
        got.append(out)
    one = torch.empty_like(q)
    K.decode_attention_e4m3(q, one, k, v, ke, ve, positions, req, table, page, heads, kv, hd, 0, hd ** -0.5, 128, splits=1)
    # the same weights; sums in another order and roundings of the last bit
    size = float(one.to(torch.float64).abs().max())
    for out in got:
        assert float((out.to(torch.float64) - one.to(torch.float64)).abs().max()) <= 2.0 ** -7 * size
        if rows > 1:
            assert not out[-1].any()
    assert float((got[0].to(torch.float64) - got[1].to(torch.float64)).abs().max()) <= 2.0 ** -8 * size


@pytest.mark.parametrize("heads,kv,hd,window,portions", [
    (4, 2, 128, 0, [(1500, 300)]), (6, 3, 64, 0, [(700, 130), (0, 90), (2100, 257)]), (2, 1, 128, 400, [(3000, 600)]), (3, 1, 128, 0, [(1023, 1), (1200, 40)])])
def test_portions_whose_keys_blocks_share(heads, kv, hd, window, portions):
    """One, two and four blocks a row block, chosen by how many SMs there are said to be; rows of no request stay as they are."""
    g = torch.Generator(device=DEV)
    g.manual_seed(heads + hd)
    T, page = sum(n for _, n in portions), 16
    per = -(-max(p + n for p, n in portions) // page)
    pages = per * len(portions)
    k, v = ((torch.randn((pages, kv, page, hd), generator=g, device=DEV)).to(torch.float8_e4m3fn) for _ in range(2))
    ke, ve = (torch.randint(122, 130, (pages, kv, page), generator=g, device=DEV).to(torch.uint8) for _ in range(2))
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(len(portions), per)
    q = torch.randn((T + 3, heads, hd), generator=g, device=DEV).to(torch.bfloat16)
    start = [0]
    for _, n in portions:
        start.append(start[-1] + n)
    got = []
    blocks = -(-(T + 3) // 256) - 1 + len(portions)
    for sms in (1, 2 * blocks * heads, 4 * blocks * heads, 148):
        out = torch.full_like(q, 5.0)
        with pytest.MonkeyPatch.context() as m:
            m.setattr(K, "_sm_count", lambda: sms)
            K.prefill_attention_e4m3(q, out, k, v, ke, ve, ints(start), ints([p for p, _ in portions]), table, page, heads, kv, hd, window, hd ** -0.5)
        assert (out[T:] == 5.0).all()
        got.append(out[:T].to(torch.float64))
    # weights rounded to bfloat16 against another reference (2^-8 of a value of at most the largest, twice) and the result's rounding
    most = float((v.to(torch.float64) * torch.exp2(ve.to(torch.float64) - 127)[..., None]).abs().max())
    for out in got[1:]:
        assert float((out - got[0]).abs().max()) <= 2.0 ** -7 * most + 2.0 ** -8 * float(got[0].abs().max())
