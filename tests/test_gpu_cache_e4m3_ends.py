"""The 8-bit cache where a row meets what is not a number, not there, or far apart: every form against the formula in 64 bits."""
import math

import pytest
import torch

from cajeta_llm_b200.csrc import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
HALF = 2.0 ** -8           # a rounding to bfloat16, half a step

# One row by itself, its keys dealt out to a cluster and to blocks that a kernel joins; portions row by row, alone and in a cluster; portions in tiles,
# a block a row block and four.
FORMS = ["one", "cluster", "merge", "rows", "rows in clusters", "tiles", "tiles in clusters"]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make(lengths, kv, hd, page_tokens, seed):
    """Codes and exponents of all pages (a few more than the requests need), and the requests' pages in mixed order."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    need = [-(-n // page_tokens) for n in lengths]
    pages, width = sum(need) + 2, max(need)
    k, v = ((torch.randn((pages, kv, page_tokens, hd), generator=g, device=DEV) * 60).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2))
    ke, ve = (torch.randint(127 - 8, 127 - 4, (pages, kv, page_tokens), generator=g, device=DEV).to(torch.uint8) for _ in range(2))
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    table = [[order.pop() if i < n else -1 for i in range(width)] for n in need]
    return k, v, ke, ve, table


def at(table, r, key, page_tokens):
    return table[r][key // page_tokens], key % page_tokens


def formula(q, rows, k, v, ke, ve, table, page_tokens, window, scale):
    """Rows [(request, position)] in 64 bits: softmax over the keys from position + 1 - window to position whose page is there.  The result, and the
    sum of weight times |value| (what a rounding of weights can move).  No key: zeros."""
    heads, hd = q.shape[1:]
    kv = k.shape[1]
    held = [c.to(F64) * torch.exp2(e.to(F64) - 127)[..., None] for c, e in ((k, ke), (v, ve))]
    out, size = torch.zeros(q.shape, dtype=F64, device=DEV), torch.zeros(q.shape, dtype=F64, device=DEV)
    for t, (r, p) in enumerate(rows):
        keys = torch.arange(max(0, p + 1 - window) if window else 0, max(0, p + 1), device=DEV) if r >= 0 else torch.empty(0, device=DEV, dtype=torch.int64)
        keys = keys[keys < len(table[0]) * page_tokens]
        page = ints(table)[r][keys // page_tokens].long()
        there = (page >= 0) & (page < k.shape[0])
        if not there.any():
            continue
        kk, vv = (x[page[there], :, keys[there] % page_tokens].transpose(0, 1) for x in held)
        w = torch.softmax((q[t].to(F64).view(kv, -1, hd) @ kk.transpose(1, 2)) * scale, dim=-1)
        out[t], size[t] = (w @ vv).view(heads, hd), (w @ vv.abs()).view(heads, hd)
    return out, size


def attend(form, q, rows, k, v, ke, ve, table, page_tokens, window, scale):
    """The rows by one of the forms; those of portions have to be runs of neighbouring positions."""
    heads, hd = q.shape[1:]
    kv, out = k.shape[1], torch.full_like(q, 7.0)
    with pytest.MonkeyPatch.context() as m:
        if form in FORMS[:3]:
            if form != "one":
                m.setattr(K, "_e4m3_cluster", lambda *a: form == "cluster")
            K.decode_attention_e4m3(q, out, k, v, ke, ve, ints([p for _, p in rows]), ints([r for r, _ in rows]), ints(table), page_tokens, heads, kv, hd,
                                    window, scale, max(1, max(p for _, p in rows) + 1), splits={"one": 1, "cluster": 3, "merge": 5}[form])
            return out
        start, prior = [0], []
        for r in range(len(table)):
            mine = [p for s, p in rows if s == r]
            assert mine == list(range(mine[0], mine[0] + len(mine))) if mine else True
            start.append(start[-1] + len(mine))
            prior.append(mine[0] if mine else 0)
        m.setattr(K, "e4m3_portions", lambda *a: {"rows": 1, "rows in clusters": 3}.get(form, 0))
        blocks = -(-len(rows) // 256) - 1 + len(table)
        m.setattr(K, "_sm_count", lambda: 1 if form == "tiles" else 4 * blocks * heads)
        K.prefill_attention_e4m3(q, out, k, v, ke, ve, ints(start), ints(prior), ints(table), page_tokens, heads, kv, hd, window, scale)
    assert not K.wait_errors()
    return out


def agree(got, want, size):
    # the result's rounding, the weights' (2^-8 of each at most: bfloat16 in tiles, f16 for single rows), and 2^-12 for exponentials of float32 scores
    got = got.to(F64)
    assert torch.equal(got.isnan(), want.isnan())
    worst = ((got - want).abs() - HALF * want.abs() - (2.0 ** -8 + 2.0 ** -12) * size).nan_to_num(0.0).max()
    assert float(worst) <= 1e-30, float(worst)


def queries(rows, heads, hd, seed=3):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn((rows, heads, hd), generator=g, device=DEV).to(torch.bfloat16)


@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 128), (20, 1, 64)])
@pytest.mark.parametrize("form", FORMS)
def test_what_is_no_number_and_is_seen_is_in_the_result(form, heads, kv, hd):
    """Queries with an entry that is NaN or infinite: all of the head's result.  A NaN in a key: all heads that share it, for every row that sees it (the
    newest key alone in a warp's share, the first, one in between).  A NaN in a value: that entry."""
    P = 16
    lengths = [33, 65, 97, 300, 700, 1300]
    k, v, ke, ve, table = make(lengths, kv, hd, P, seed=heads)
    rows = [(r, n - 1) for r, n in enumerate(lengths)]
    scale = 1 / math.sqrt(hd)
    for bad in (float("nan"), float("inf"), -float("inf")):
        q = queries(len(rows), heads, hd)
        q[1, 1, 5] = q[3, 0, 0] = q[5, heads - 1, hd - 1] = bad
        agree(attend(form, q, rows, k, v, ke, ve, table, P, 0, scale), *formula(q, rows, k, v, ke, ve, table, P, 0, scale))
    # an infinite entry beside keys that are of one sign there: every score is infinite, of either sign
    signed = k.view(torch.uint8).clone()
    signed[..., 7] = 0xb0
    q = queries(len(rows), heads, hd)
    q[0, 0, 7], q[5, 1, 7] = float("inf"), -float("inf")
    signed = signed.view(torch.float8_e4m3fn)
    agree(attend(form, q, rows, signed, v, ke, ve, table, P, 0, scale), *formula(q, rows, signed, v, ke, ve, table, P, 0, scale))
    q = queries(len(rows), heads, hd)
    for plane in (0, 1):
        c = [x.view(torch.uint8).clone() for x in (k, v)]
        for r, key in ((0, 32), (1, 64), (2, 96), (3, 0), (4, 333), (5, 900)):
            page, i = at(table, r, key, P)
            c[plane][page, kv - 1, i, 3] = 0x7f if r % 2 else 0xff
        kk, vv = (x.view(torch.float8_e4m3fn) for x in c)
        for window in (0, 64):
            agree(attend(form, q, rows, kk, vv, ke, ve, table, P, window, scale), *formula(q, rows, kk, vv, ke, ve, table, P, window, scale))


@pytest.mark.parametrize("page_tokens,hd,window", [(16, 128, 0), (5, 64, 0), (128, 128, 0), (16, 64, 150)])
@pytest.mark.parametrize("form", FORMS)
def test_a_page_that_is_not_there_holds_no_key(form, page_tokens, hd, window):
    """Pages of no number and beyond the pool, at a row's start, in its midst and at its end; a row of which nothing is there."""
    heads, kv = 6, 2
    lengths = [40, 300, 700, 290, 200, 1300]
    k, v, ke, ve, table = make(lengths, kv, hd, page_tokens, seed=page_tokens)
    for r, key, page in ((0, 39, -1), (1, 0, len(k)), (1, 177, -1), (2, 300, -7), (2, 555, 2 ** 31 - 1), (2, 690, len(k)), (3, 130, -1), (5, 40, -1), (5, 1000, -1)):
        table[r][key // page_tokens] = page
    table[4] = [-1] * len(table[4])
    q = queries(len(lengths) * 3, heads, hd)
    rows = [(r, n - 3 + i) for r, n in enumerate(lengths) for i in range(3)]
    scale = 1 / math.sqrt(hd)
    want, size = formula(q, rows, k, v, ke, ve, table, page_tokens, window, scale)
    assert not want[12:15].any()
    agree(attend(form, q, rows, k, v, ke, ve, table, page_tokens, window, scale), want, size)


@pytest.mark.parametrize("form", FORMS[5:])
def test_a_whole_prompt_with_pages_that_are_not_there(form):
    heads, kv, hd, P = 3, 3, 128, 16
    k, v, ke, ve, table = make([420], kv, hd, P, seed=1)
    for i in (0, 3, 4, 11, 25):
        table[0][i] = -1
    q = queries(420, heads, hd)
    rows = [(0, p) for p in range(420)]
    agree(attend(form, q, rows, k, v, ke, ve, table, P, 0, 0.09), *formula(q, rows, k, v, ke, ve, table, P, 0, 0.09))


@pytest.mark.parametrize("below,above,n,where", [
    (40, 25, 200, 0), (40, 25, 200, 77), (40, 25, 200, 199), (20, 30, 200, 5), (100, 90, 200, 40), (12, 60, 130, 129), (30, 0, 200, 0), (-40, -30, 200, 100),
    (-25, -60, 200, 0), (60, 40, 5000, 2500)])
@pytest.mark.parametrize("form", FORMS)
def test_a_large_value_that_a_row_hardly_looks_at_takes_nothing_from_the_others(form, below, above, n, where):
    """One key whose score lies `below` octaves under the others' and whose value `above` octaves over theirs (all of one sign)."""
    heads, kv, hd, P = 4, 2, 128, 16
    k, v, ke, ve, table = make([n], kv, hd, P, seed=n)
    v = (v.float().abs() + 1).to(torch.float8_e4m3fn)
    k = torch.zeros_like(k.float())
    page, i = at(table, 0, where, P)
    k[page, :, i, 0] = -1.0
    k = k.to(torch.float8_e4m3fn)
    ke.fill_(127), ve.fill_(127 - 8)
    ve[page, :, i] += above if above >= 0 else 256 + above
    scale = 0.125
    q = torch.zeros((2, heads, hd), device=DEV)
    q[..., 0] = below / (scale * math.log2(math.e))
    q = q.to(torch.bfloat16)
    rows = [(0, n - 2), (0, n - 1)]
    agree(attend(form, q, rows, k, v, ke, ve, table, P, 0, scale), *formula(q, rows, k, v, ke, ve, table, P, 0, scale))


@pytest.mark.parametrize("form", FORMS)
def test_many_small_weights_beside_a_large_value_and_a_large_weight(form):
    """The largest weight is of a value of nothing, the largest value of a weight of nothing: what is left is most of the result."""
    heads, kv, hd, P, n = 4, 4, 64, 16, 20_000
    k, v, ke, ve, table = make([n], kv, hd, P, seed=6)
    v = (v.float().abs() + 1).to(torch.float8_e4m3fn)
    ve.fill_(127 - 8), ke.fill_(127)
    k = torch.zeros_like(k.float())
    for key, score, e in ((17, 12.0, -60), (2066, -60.0, 13)):
        page, i = at(table, 0, key, P)
        k[page, :, i, 0] = score
        ve[page, :, i] = 127 - 8 + e
    k = k.to(torch.float8_e4m3fn)
    q = torch.zeros((1, heads, hd), device=DEV)
    q[..., 0] = 1.0
    q = q.to(torch.bfloat16)
    scale = 1 / math.log2(math.e)
    rows = [(0, n - 1)]
    agree(attend(form, q, rows, k, v, ke, ve, table, P, 0, scale), *formula(q, rows, k, v, ke, ve, table, P, 0, scale))


@pytest.mark.parametrize("window", [0, 1, 30, 100, 500])
@pytest.mark.parametrize("form", FORMS)
def test_rows_behind_the_tables_last_page_see_the_keys_of_their_window(form, window):
    heads, kv, hd, P = 4, 2, 128, 16
    k, v, ke, ve, table = make([256, 256, 256], kv, hd, P, seed=4)
    rows = [(0, 253), (0, 254), (0, 255), (0, 256), (0, 257), (1, 280), (1, 281), (2, 700), (2, 701)]
    q = queries(len(rows), heads, hd)
    agree(attend(form, q, rows, k, v, ke, ve, table, P, window, 0.1), *formula(q, rows, k, v, ke, ve, table, P, window, 0.1))


@pytest.mark.parametrize("prior,rows,window", [(-300, 150, 0), (-300, 150, 20), (-1000, 400, 0), (-40, 200, 0), (10_000_000, 40, 0), (10_000_000, 40, 1000),
                                               (150, 300, 0), (150, 300, 90)])
@pytest.mark.parametrize("form", FORMS[3:])
def test_rows_outside_the_table_see_the_keys_that_are_there(form, prior, rows, window):
    """Before the first position, behind the last page, and on both sides of it: no key, or those of the table that are in reach."""
    heads, kv, hd, P = 2, 1, 64, 16
    k, v, ke, ve, table = make([200], kv, hd, P, seed=2)
    q = queries(rows, heads, hd)
    at_ = [(0, prior + i) for i in range(rows)]
    agree(attend(form, q, at_, k, v, ke, ve, table, P, window, 0.1), *formula(q, at_, k, v, ke, ve, table, P, window, 0.1))


@pytest.mark.parametrize("prior,rows,window", [(0, 300, 0), (100, 200, 0), (1000, 520, 0), (300, 400, 90), (0, 130, 1)])
@pytest.mark.parametrize("form", FORMS[3:])
def test_a_value_that_is_no_number_reaches_the_rows_that_see_it_alone(form, prior, rows, window):
    """Rows before it, and those whose window has left it behind, share tiles and blocks with the rows that do."""
    heads, kv, hd, P = 4, 2, 128, 16
    k, v, ke, ve, table = make([prior + rows], kv, hd, P, seed=rows)
    c = v.view(torch.uint8).clone()
    for key, head, entry in ((prior + rows // 2, 0, 3), (prior + rows - 1, 1, 127), (prior + rows - 2, 0, 0), (prior + 7, 1, 64), (max(0, prior - 40), 0, 77)):
        page, i = at(table, 0, key, P)
        c[page, head, i, entry] = 0xff
    v = c.view(torch.float8_e4m3fn)
    q = queries(rows, heads, hd)
    where = [(0, prior + i) for i in range(rows)]
    want, size = formula(q, where, k, v, ke, ve, table, P, window, 0.09)
    assert want.isnan().any() and not want[:, 0, 0].isnan()[0]
    agree(attend(form, q, where, k, v, ke, ve, table, P, window, 0.09), want, size)


def test_a_table_of_one_row_is_as_wide_as_it_is():
    """Its stride says nothing: a column turned over, and a row cut out of a wider table."""
    heads, kv, hd, P, n = 4, 2, 128, 16, 100
    k, v, ke, ve, table = make([n], kv, hd, P, seed=9)
    q = queries(3, heads, hd)
    rows = [(0, n - 3 + i) for i in range(3)]
    want, size = formula(q, rows, k, v, ke, ve, table, P, 0, 0.1)
    x = torch.randn((3, (heads + 2 * kv) * hd), device=DEV)
    row = ints(table[0])
    wide = torch.cat([ints(table), ints(table)], dim=1)
    for one in (row[:, None].contiguous().t(), wide[:, :len(table[0])]):
        assert one.is_contiguous() and one.stride(0) != one.shape[1]
        out = torch.full_like(q, 7.0)
        K.decode_attention_e4m3(q, out, k, v, ke, ve, ints([p for _, p in rows]), ints([0] * 3), one, P, heads, kv, hd, 0, 0.1, n)
        agree(out, want, size)
        for form in (0, 1):
            out = torch.full_like(q, 7.0)
            with pytest.MonkeyPatch.context() as m:
                m.setattr(K, "e4m3_portions", lambda *a: form)
                K.prefill_attention_e4m3(q, out, k, v, ke, ve, ints([0, 3]), ints([n - 3]), one, P, heads, kv, hd, 0, 0.1)
            agree(out, want, size)
        kk, ee = torch.zeros_like(k), torch.zeros_like(ke)
        K.rope_kv_write_e4m3(x, 0, heads * hd, (heads + kv) * hd, torch.empty_like(q), kk, torch.zeros_like(v), ee, torch.zeros_like(ve),
                             ints([p for _, p in rows]), ints([0] * 3), one, P, heads, kv, hd, 0, None, True)
        for r, p in rows:
            page, i = at(table, r, p, P)
            assert (ee[page, :, i] > 0).all()
