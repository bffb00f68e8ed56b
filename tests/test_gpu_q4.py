"""Products with 4-bit weights against the formula in 64 bits, and the quantiser."""
import pytest
import torch

from cajeta_llm_b200.csrc import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F64 = torch.float64
HALF = 2.0 ** -8           # a rounding to bfloat16, half a step


def weight(shape, group, seed):
    """Codes of every value, scales of five significant bits over ten octaves."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    codes = torch.randint(-8, 8, shape, generator=g, device=DEV).to(torch.int8)
    m = torch.randint(16, 32, tuple(shape[:-1]) + (-(-shape[-1] // group),), generator=g, device=DEV)
    scales = torch.ldexp(m.to(torch.float32), torch.randint(-14, -4, m.shape, generator=g, device=DEV))
    full = codes.to(F64) * scales.to(F64).repeat_interleave(group, dim=-1)[..., :shape[-1]]
    return K.Q4Weight.from_codes(codes, scales, group), full


def sums(K_, x):
    """What float32 sums of K products may be off by, as a share of the sum of their sizes: 64 by the tensor core and one for each 64."""
    return (64 + K_ / 64 + 8) * 2.0 ** -23 * x


def check(got, want, slack):
    rounding = HALF * want.abs() if got.dtype == torch.bfloat16 else 2.0 ** -24 * want.abs()
    worst = ((got.to(F64) - want).abs() - rounding - slack).max()
    assert float(worst) <= 1e-30, float(worst)


SHAPES = [(1, 128, 64, 64), (1, 6144 // 4, 2048, 64), (7, 200, 136, 32), (8, 1, 8, 64), (9, 17, 2056, 128), (16, 130, 512, 64), (17, 384, 1408, 32),
          (33, 257, 320, 64), (64, 640, 1024, 64), (100, 96, 72, 128), (129, 1000, 704, 32), (300, 512, 2048, 64), (513, 300, 192, 64)]


@pytest.mark.parametrize("rows,features,k,group", SHAPES)
@pytest.mark.parametrize("form", ["plain", "bias", "accumulate", "half", "gated"])
def test_dense(rows, features, k, group, form):
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + k)
    w, full = weight((features, k), group, seed=features)
    wide = torch.randn((rows, k + 8), generator=g, device=DEV).to(torch.bfloat16)
    x = wide[:, 4:4 + k]                                                        # rows of a wider matrix, eight bytes off its start
    xd = x.to(F64)
    want, size = xd @ full.T, xd.abs() @ full.abs().T
    if form == "gated":
        up, full_up = weight((features, k), group, seed=features + 1)
        out = torch.empty((rows, features), dtype=torch.bfloat16, device=DEV)
        K.gemm_q4(x, w, out, w_up=up)
        u, usize = xd @ full_up.T, xd.abs() @ full_up.abs().T
        gate = want * torch.sigmoid(want)
        # the sums' errors through silu (slope at most 1.1) and the product, and a fast exponential and division: 2^-20 of the result's
        # size times the exponential's argument
        slack = 1.1 * sums(k, size) * u.abs() + sums(k, usize) * gate.abs() + 2.0 ** -20 * (1 + want.abs()) * (gate * u).abs()
        check(out, gate * u, slack)
        return
    bias = torch.randn(features, generator=g, device=DEV) if form == "bias" else None
    before = torch.randn((rows, features), generator=g, device=DEV)
    out = before.to(torch.bfloat16) if form == "half" else before.clone()
    K.gemm_q4(x, w, out, bias=bias, accumulate=form == "accumulate")
    if bias is not None:
        want = want + bias.to(F64)
    if form == "accumulate":
        want = want + before.to(F64)
    check(out, want, sums(k, size) + 2.0 ** -23 * (before.abs() if form == "accumulate" else 0.0) + (2.0 ** -23 * bias.abs() if bias is not None else 0.0))


@pytest.mark.parametrize("tokens,top,experts,features,k,group", [
    (1, 2, 8, 192, 384, 64), (3, 4, 60, 130, 256, 32), (40, 2, 4, 96, 512, 64), (300, 4, 16, 256, 136, 64), (1000, 2, 3, 384, 256, 32), (5, 1, 5, 70, 64, 64)])
@pytest.mark.parametrize("form", ["plain", "half", "gated", "rows"])
def test_experts(tokens, top, experts, features, k, group, form):
    """Groups of uneven sizes, some empty; rows gathered by index, one of them outside; rows before and behind the groups stay."""
    g = torch.Generator(device=DEV)
    g.manual_seed(tokens)
    w, full = weight((experts, features, k), group, seed=experts)
    up, full_up = weight((experts, features, k), group, seed=experts + 1)
    lean = torch.randn(experts, generator=g, device=DEV) * 2
    picks = (lean + torch.randn((tokens, experts), generator=g, device=DEV)).topk(top, dim=1).indices.reshape(-1)
    order = torch.argsort(picks, stable=True)
    n, lead, tail = picks.numel(), 2, 3
    counts = torch.bincount(picks, minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32) + lead
    index = torch.cat([torch.zeros(lead, device=DEV), order // top, torch.zeros(tail, device=DEV)]).to(torch.int32)
    x = torch.randn((tokens, k), generator=g, device=DEV).to(torch.bfloat16)
    if form == "rows":
        x, index = x[index.long()].contiguous(), None
        rows = x.to(F64)
    else:
        index[lead] = tokens + 5 if tokens > 1 else -1
        rows = x[index.clamp(0, tokens - 1).long()].to(F64)
        rows[lead] = 0
    out = torch.full((lead + n + tail, features), 7.0, dtype=torch.bfloat16 if form in ("half", "gated") else torch.float32, device=DEV)
    K.gemm_q4(x, w, out, w_up=up if form == "gated" else None, group_offsets=offsets, a_row_index=index)
    assert (out[:lead] == 7.0).all() and (out[lead + n:] == 7.0).all()
    at = offsets.tolist()
    for e in range(experts):
        r = slice(at[e], at[e + 1])
        y, size = rows[r] @ full[e].T, rows[r].abs() @ full[e].abs().T
        if not y.numel():
            continue
        if form == "gated":
            u, usize = rows[r] @ full_up[e].T, rows[r].abs() @ full_up[e].abs().T
            gate = y * torch.sigmoid(y)
            slack = 1.1 * sums(k, size) * u.abs() + sums(k, usize) * gate.abs() + 2.0 ** -20 * (1 + y.abs()) * (gate * u).abs()
            check(out[r], gate * u, slack)
        else:
            check(out[r], y, sums(k, size))
    assert not K.wait_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,group", [((5, 200), 64), ((3, 7, 136), 32), ((130, 64), 128)])
def test_quantiser(shape, group, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(shape[-1])
    w = (torch.randn(shape, generator=g, device=DEV) * 0.02).to(dtype)
    w.view(-1, shape[-1])[1, :group] = 0                                         # a group of zeros
    w.view(-1, shape[-1])[2, 3] = 1e-41                                          # and of nothing that float32 holds as a normal number
    w.view(-1, shape[-1])[2, 4:group] = 0
    w.view(-1, shape[-1])[2, :3] = 0
    codes, scales = K.Q4Weight.codes_of(w, group)
    n = -(-shape[-1] // group)
    for i in range(n):
        piece = w[..., i * group:(i + 1) * group].to(F64)
        s, q = scales[..., i].to(F64), codes[..., i * group:(i + 1) * group].to(F64)
        least = piece.abs().amax(-1) / 7
        tiny = least < 2.0 ** -126
        assert (s[~tiny] >= least[~tiny] * (1 - 2.0 ** -23)).all() and (s[~tiny] <= least[~tiny] * (1 + 2.0 ** -4)).all() and (s[tiny] == 0).all()
        assert ((q * s[..., None] - piece).abs() <= 0.5 * s[..., None] * (1 + 1e-6) + tiny[..., None] * 1e-38).all()
        assert (q.abs() <= 7).all()
    assert (scales.view(torch.int32) & 0x7ffff == 0).all()
    held = K.Q4Weight.quantise(w, group)
    again = K.Q4Weight.from_codes(codes, scales, group)
    assert torch.equal(held.data, again.data) and held.shape == tuple(shape)


def test_part_of_a_weight_and_strided_results():
    w, full = weight((300, 128), 64, seed=1)
    x = torch.randn((5, 128), device=DEV).to(torch.bfloat16)
    want, size = x.to(F64) @ full.T, x.to(F64).abs() @ full.abs().T
    wide = torch.full((5, 400), 7.0, device=DEV)
    K.gemm_q4(x, w.first(100), wide[:, 50:150])
    check(wide[:, 50:150], want[:, :100], sums(128, size[:, :100]))
    assert (wide[:, :50] == 7.0).all() and (wide[:, 150:] == 7.0).all()
    w, full = weight((6, 64, 128), 64, seed=2)
    out = torch.empty((5, 64), device=DEV)
    K.gemm_q4(x, w.first(2), out, group_offsets=torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV))
    check(out[2:], x[2:].to(F64) @ full[1].T, sums(128, x[2:].to(F64).abs() @ full[1].abs().T))


def test_infinite_and_missing_entries_stay_in_their_rows():
    w, full = weight((140, 256), 64, seed=4)
    for rows in (4, 40, 200):
        x = torch.randn((rows, 256), device=DEV).to(torch.bfloat16)
        out = torch.empty((rows, 140), device=DEV)
        K.gemm_q4(x, w, out)
        x[1, 7], x[2, 9] = float("nan"), float("inf")
        bad = torch.empty_like(out)
        K.gemm_q4(x, w, bad)
        rest = [r for r in range(rows) if r not in (1, 2)]
        assert torch.equal(bad[rest], out[rest]) and torch.isnan(bad[1]).all() and not torch.isfinite(bad[2]).any()


def test_captured_and_replayed():
    w, full = weight((256, 512), 64, seed=4)
    for rows in (3, 200):
        x = torch.randn((rows, 512), device=DEV).to(torch.bfloat16)
        out = torch.empty((rows, 256), device=DEV)
        K.gemm_q4(x, w, out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.gemm_q4(x, w, out)
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        K.gemm_q4(x, w, out)
        assert torch.equal(got, out)


@pytest.mark.parametrize("rows,features,k,group,form", [
    (2048, 640, 2048, 64, "plain"), (700, 1920, 4032, 64, "accumulate"), (1000, 3584, 3584, 32, "plain"), (130, 5000, 64, 64, "bias"), (24, 6144, 200, 64, "half"),
    (300, 20000, 136, 32, "gated"), (520, 704, 2752, 64, "gated32"), (65, 9000, 1032, 64, "accumulate"), (257, 4096, 8, 64, "plain"), (300, 1000, 1984, 32, "half")])
def test_dense_of_many_rows(rows, features, k, group, form):
    """Several tiles a block, an odd number of blocks of 64 along K, K in parts, rows and features that end inside a tile; twice over."""
    assert K.q4_on_tcgen05(rows, features, 0)
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + k)
    w, full = weight((features, k), group, seed=features)
    x = torch.randn((rows, k + 8), generator=g, device=DEV).to(torch.bfloat16)[:, :k]
    xd = x.to(F64)
    want, size = xd @ full.T, xd.abs() @ full.abs().T
    for _ in range(2):
        if form.startswith("gated"):
            up, full_up = weight((features, k), group, seed=features + 1)
            out = torch.empty((rows, features), dtype=torch.float32 if form == "gated32" else torch.bfloat16, device=DEV)
            K.gemm_q4(x, w, out, w_up=up)
            u, usize = xd @ full_up.T, xd.abs() @ full_up.abs().T
            gate = want * torch.sigmoid(want)
            check(out, gate * u, 1.1 * sums(k, size) * u.abs() + sums(k, usize) * gate.abs() + 2.0 ** -20 * (1 + want.abs()) * (gate * u).abs())
            continue
        bias = torch.randn(features, generator=g, device=DEV) if form == "bias" else None
        before = torch.randn((rows, features), generator=g, device=DEV)
        out = before.to(torch.bfloat16) if form == "half" else before.clone()
        K.gemm_q4(x, w, out, bias=bias, accumulate=form == "accumulate")
        exact = want + (bias.to(F64) if bias is not None else before.to(F64) if form == "accumulate" else 0.0)
        # (a part's sum joins the others and what was there by one float32 addition each)
        check(out, exact, sums(k, size) + 2.0 ** -22 * (before.abs() if form == "accumulate" else bias.abs() if bias is not None else 0.0))


def test_scales_and_entries_out_of_range_are_refused():
    codes = torch.zeros((16, 64), dtype=torch.int8, device=DEV)
    for s in (2.0 ** 123, float("inf"), float("nan"), -(2.0 ** 123)):
        with pytest.raises(K.KernelError, match="below 2\\^123"):
            K.Q4Weight.from_codes(codes, torch.full((16, 1), s, device=DEV))
    for bad in (float("inf"), float("nan"), 3.0e38):
        w = torch.ones((16, 128), device=DEV)
        w[3, 70] = bad
        with pytest.raises(K.KernelError, match="finite"):
            K.Q4Weight.quantise(w)


def test_the_largest_and_smallest_scales():
    """Products of few rows and of many read the same numbers at both ends of the scales' range."""
    codes = (torch.arange(256 * 64, device=DEV) % 16 - 8).to(torch.int8).view(256, 64)
    for s in (31.0 * 2.0 ** 118, 2.0 ** -126):
        w = K.Q4Weight.from_codes(codes, torch.full((256, 1), s, device=DEV))
        x = torch.zeros((1024, 64), dtype=torch.bfloat16, device=DEV)
        x[torch.arange(1024), torch.arange(1024) % 64] = 1.0
        for rows in (1, 8, 1024):
            out = torch.empty((rows, 256), device=DEV)
            K.gemm_q4(x[:rows], w, out)
            assert torch.equal(out.to(F64), codes.to(F64).T[torch.arange(rows, device=DEV) % 64] * s)


def test_more_groups_than_the_tensor_core_form_has_places_for():
    groups, k = 1500, 64
    w, full = weight((groups, 16, k), 64, seed=5)
    rows = 4 * groups
    x = torch.randn((rows, k), device=DEV).to(torch.bfloat16)
    offsets = torch.arange(0, rows + 1, 4, dtype=torch.int32, device=DEV)
    out = torch.empty((rows, 16), device=DEV)
    K.gemm_q4(x, w, out, group_offsets=offsets)
    of = full.repeat_interleave(4, dim=0)
    want = torch.einsum("sk,sfk->sf", x.to(F64), of)
    check(out, want, sums(k, torch.einsum("sk,sfk->sf", x.to(F64).abs(), of.abs())))


def test_rows_of_a_shared_in_memory():
    """One row expanded to many, and rows that overlap."""
    w, full = weight((6144, 128), 64, seed=9)
    x = torch.randn(128 + 8 * 63, device=DEV).to(torch.bfloat16)
    for a in (x[:128].view(1, 128).expand(64, 128), x.as_strided((64, 128), (8, 1))):
        out = torch.empty((64, 6144), device=DEV)
        K.gemm_q4(a, w, out)
        check(out, a.to(F64) @ full.T, sums(128, a.to(F64).abs() @ full.abs().T))
