"""Block quantisation and block-scaled 8-bit contraction on the GPU against their definitions in 64 bits."""
import itertools

import pytest
import torch

import hiptensor_b200 as ht
import training_helpers as ref

pytestmark = pytest.mark.gpu
E4, E5, BF, F16, F32 = ht.R_8F_E4M3, ht.R_8F_E5M2, ht.R_16BF, ht.R_16F, ht.R_32F
KIND = {v[0]: k for k, v in ref.FP8.items()} | {v: k for k, v in ref.TYPES.items()}


@pytest.fixture(scope="module")
def h():
    return ht.Handle()


def desc(h, x):
    return h.tensor_descriptor(x.shape, x.stride(), KIND[x.dtype])


def padded(rows, cols, kind, pad, fill=0x55):
    """rows x cols of a buffer with `pad` more elements in each row, all bytes set to `fill`."""
    size = torch.tensor([], dtype=kind).element_size()
    raw = torch.full((rows, (cols + pad) * size), fill, device="cuda", dtype=torch.uint8)
    return raw.view(kind)[:, :cols], raw


def values(rows, cols, kind, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(2 * torch.randn(rows, 1, generator=g, device="cuda"))
    if rows > 2 and cols > 130:
        x[1] = 0  # blocks of zeros
        x[2, :128] *= 2.0 ** -20
    return x.to(kind)


def quantize(h, x, block, to, transposed=False, padA=0, padQ=0, stream=None):
    kind = ref.FP8[to][0]
    r, c = x.shape
    q, raw = padded(c, r, kind, padQ) if transposed else padded(r, c, kind, padQ)
    s = torch.full([-(-n // b) for n, b in zip(x.shape, block)], -1.0, device="cuda")
    h.block_quantize(x, desc(h, x), (0, 1), block, q, desc(h, q), (1, 0) if transposed else (0, 1), s, desc(h, s), stream)
    used = (c, r) if transposed else (r, c)
    assert bool((raw[:, used[1]:] == 0x55).all()), "padding was written"
    return (q.T if transposed else q), s


def same(q, s, x, block, to):
    want, scale = ref.quantize(x, block, to)
    got = q.double()
    assert torch.equal(s.isnan(), scale.isnan())
    assert torch.equal(s[~s.isnan()], scale[~scale.isnan()])
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~got.isnan()], want[~want.isnan()])


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("kind,to", [(torch.bfloat16, E4), (torch.float16, E5), (torch.float32, E4)])
@pytest.mark.parametrize("rows,cols,padA,padQ", [(1, 1, 0, 0), (1, 4096, 0, 0), (130, 257, 0, 0), (33, 520, 8, 8), (300, 1000, 3, 5),
                                                 (257, 384, 0, 16), (4096, 7, 1, 0)])
def test_quantize_is_the_definition(h, rows, cols, padA, padQ, kind, to, block, transposed):
    x = values(rows, cols + padA, kind, 7)[:, :cols]
    q, s = quantize(h, x, block, to, transposed, padQ=padQ)
    same(q, s, x, block, to)


@pytest.mark.parametrize("to", [E4, E5])
def test_quantize_next_to_borders(h, to):
    # every bf16 mantissa against block maxima whose factor is rounded: products on, just beside and between the borders
    m = torch.arange(128, 256, device="cuda").float()
    rows = []
    for a in list(range(129, 256, 7)) + [192, 224, 255]:
        r = torch.cat([m, m / 2, m / 64, m / 4096])
        r = r[r <= a]
        r = torch.cat([r, torch.zeros(-len(r) % 128, device="cuda")]).view(-1, 128)
        r[:, 127] = a
        rows.append(r)
    x = torch.cat(rows).to(torch.bfloat16)
    q, s = quantize(h, x, (1, 128), to)
    same(q, s, x, (1, 128), to)


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)])
def test_quantize_infinities_nan_and_tiny_blocks(h, block):
    x = torch.randn(256, 300, device="cuda")
    x[0, 0], x[3, 200], x[130, 131], x[131, 290] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[200:, :] = 1e-38
    x[201, 5] = -3e-40
    q, s = quantize(h, x, block, E4)
    same(q, s, x, block, E4)


def test_quantize_batch_of_matrices_and_strided_input(h):
    # two blocked modes under a batch mode; A contiguous along its first mode
    base = torch.randn(3, 200, 260, device="cuda").to(torch.bfloat16)
    x = base.transpose(1, 2)  # (3, 260, 200), stride 1 in the middle
    q = torch.empty(3, 260, 200, device="cuda", dtype=torch.float8_e4m3fn)
    s = torch.empty(3, 3, 2, device="cuda")
    h.block_quantize(x, desc(h, x), (4, 0, 1), (1, 128, 128), q, desc(h, q), (4, 0, 1), s, desc(h, s))
    for i in range(3):
        same(q[i], s[i], x[i], (128, 128), E4)
    # no contiguous mode at all, scales in another order than A
    y = torch.randn(70, 2, 300, 2, device="cuda")[:, 0, :, 0]
    q = torch.empty(70, 300, device="cuda", dtype=torch.float8_e5m2)
    s = torch.empty(3, 70, device="cuda").T
    h.block_quantize(y, desc(h, y), (0, 1), (1, 128), q, desc(h, q), (0, 1), s, desc(h, s))
    same(q, s, y, (1, 128), E5)


def test_quantize_empty(h):
    x = torch.empty(0, 128, device="cuda")
    q, s = quantize(h, x, (1, 128), E4)
    assert q.numel() == 0 and s.numel() == 0


def operand(rows, k, kind, seed, layout="k"):
    """8-bit values of all sizes; layout: "k" contiguous along k in rows of 16-byte words, "odd" rows of odd length, "m" contiguous along the rows."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    largest = ref.FP8[KIND[kind]][1]
    v = (torch.randn(rows, k, generator=g, device="cuda") * largest / 6).clamp(-largest, largest).to(kind)
    if layout == "m":
        return v.T.contiguous().T
    buf, _ = padded(rows, k, kind, (-k % 16) if layout == "k" else 1 - k % 2, fill=0x7F)  # NaN between the rows
    buf.copy_(v)
    return buf


def run_scaled(h, m, n, k, a="e4", b="e4", rowB=False, rowA=True, out=torch.bfloat16, alpha=1.0, beta=None, layoutA="k", layoutB="k",
               colD=False, stream=None):
    kinds = {"e4": torch.float8_e4m3fn, "e5": torch.float8_e5m2}
    A, B = operand(m, k, kinds[a], 1, layoutA), operand(n, k, kinds[b], 2, layoutB)
    g = torch.Generator(device="cuda").manual_seed(3)
    kb = -(-k // 128)
    bA, bB = (1 if rowA else 128, 128), (1 if rowB else 128, 128)
    sA = torch.exp(torch.randn(-(-m // bA[0]), kb, generator=g, device="cuda")) / ref.FP8[KIND[A.dtype]][1]
    sB = torch.exp(torch.randn(-(-n // bB[0]), kb, generator=g, device="cuda")) / ref.FP8[KIND[B.dtype]][1]
    C = None if beta is None else torch.randn((n, m) if colD else (m, n), generator=g, device="cuda").to(out)
    D = torch.full((n, m) if colD else (m, n), float("nan"), device="cuda", dtype=out)
    if colD:
        D, C = D.T, (None if C is None else C.T)
    dD = desc(h, D)
    plan = h.scaled_contraction_plan(desc(h, A), (0, 2), desc(h, sA), bA, desc(h, B), (1, 2), desc(h, sB), bB,
                                     None if C is None else dD, dD, (0, 1))
    h.scaled_contraction(plan, alpha, A, sA, B, sB, beta or 0.0, C, D, stream)
    want, bound = ref.scaled(A, sA, bA, B, sB, bB, alpha, beta, C)
    bound = bound + (ref.half_step(out) * 1.01 if out != torch.float32 else 2.0 ** -23) * want.abs() + 2.0 ** -25 * (out == torch.float16)
    off = (D.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    return D


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 4096, 512), (3, 130, 129), (17, 1000, 1000), (64, 64, 128), (127, 129, 640),
                                   (128, 256, 256), (257, 513, 384), (300, 72, 2064), (1030, 520, 1296), (2100, 2056, 400)])
@pytest.mark.parametrize("rowB", [False, True])
def test_scaled_sizes(h, m, n, k, rowB):
    run_scaled(h, m, n, k, rowB=rowB)


@pytest.mark.parametrize("a,b", list(itertools.product(("e4", "e5"), repeat=2)))
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(5, 200, 300), (600, 640, 512)])
def test_scaled_types(h, m, n, k, a, b, out):
    run_scaled(h, m, n, k, a=a, b=b, out=out)


@pytest.mark.parametrize("rowA,rowB", list(itertools.product((False, True), repeat=2)))
@pytest.mark.parametrize("colD", [False, True])
@pytest.mark.parametrize("m,n,k", [(9, 300, 260), (300, 9, 260), (700, 900, 260)])
def test_scaled_blocks_and_orders_of_the_result(h, m, n, k, rowA, rowB, colD):
    run_scaled(h, m, n, k, rowA=rowA, rowB=rowB, colD=colD, out=torch.float32)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(7, 260, 520), (520, 777, 300), (40, 50, 0), (700, 768, 130), (100, 200, 2048), (2100, 2056, 400)])
@pytest.mark.parametrize("rowB", [False, True])
def test_scaled_alpha_beta(h, m, n, k, out, rowB):
    run_scaled(h, m, n, k, out=out, alpha=-0.75, beta=1.5, rowB=rowB)


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("start,pad", [(0, 0), (1, 2), (3, 1), (0, 3), (0, 7), (8, 11)])
@pytest.mark.parametrize("out", [torch.float32, torch.float16])
@pytest.mark.parametrize("m,n,k,rowB", [(1, 4097, 1100, False), (3, 133, 2100, False), (130, 301, 1000, True), (2307, 2049, 256, False)])
def test_scaled_results_at_any_start_and_row_stride(h, m, n, k, rowB, out, start, pad, add):
    """The result and C are columns start .. start + n of a wider matrix; what lies beside them stays."""
    A, B = operand(m, k, torch.float8_e4m3fn, 1), operand(n, k, torch.float8_e4m3fn, 2)
    bA, bB = (1, 128), (1 if rowB else 128, 128)
    sA = torch.rand(m, -(-k // 128), device="cuda") / 448
    sB = torch.rand(-(-n // bB[0]), -(-k // 128), device="cuda") / 448
    wide = torch.randn(m, start + n + pad, device="cuda").to(out)
    before, D = wide.clone(), wide[:, start : start + n]
    C = before[:, start : start + n]
    dD, C = desc(h, D), C if add else None
    plan = h.scaled_contraction_plan(desc(h, A), (0, 2), desc(h, sA), bA, desc(h, B), (1, 2), desc(h, sB), bB, dD if add else None, dD, (0, 1))
    h.scaled_contraction(plan, 0.5, A, sA, B, sB, 2.0 if add else 0.0, C, D)
    want, bound = ref.scaled(A, sA, bA, B, sB, bB, 0.5, 2.0 if add else None, C)
    bound = bound + (ref.half_step(out) * 1.01 if out != torch.float32 else 2.0 ** -23) * want.abs() + 2.0 ** -25 * (out == torch.float16)
    assert bool(((D.double() - want).abs() <= bound).all())
    assert torch.equal(wide[:, :start], before[:, :start]) and torch.equal(wide[:, start + n :], before[:, start + n :])


@pytest.mark.parametrize("layoutA,layoutB", [("odd", "k"), ("k", "odd"), ("m", "k"), ("k", "m"), ("m", "m"), ("odd", "odd")])
@pytest.mark.parametrize("m,n,k", [(2, 70, 131), (200, 300, 500)])
def test_scaled_layouts(h, m, n, k, layoutA, layoutB):
    run_scaled(h, m, n, k, layoutA=layoutA, layoutB=layoutB, rowB=True, out=torch.float32)


@pytest.mark.parametrize("m,n", [(300, 400), (2304, 2300)])
def test_scaled_in_place_accumulation_and_repeat(h, m, n):
    A, B = operand(m, 1024, torch.float8_e5m2, 1), operand(n, 1024, torch.float8_e4m3fn, 2)
    sA, sB = torch.rand(m, 8, device="cuda"), torch.rand(n, 8, device="cuda")
    D = torch.randn(m, n, device="cuda")
    C, dD = D.clone(), desc(h, D)
    plan = h.scaled_contraction_plan(desc(h, A), (0, 2), desc(h, sA), (1, 128), desc(h, B), (1, 2), desc(h, sB), (1, 128), dD, dD, (0, 1))
    h.scaled_contraction(plan, 0.5, A, sA, B, sB, 1.0, D, D)  # C is D
    E = torch.empty_like(D)
    h.scaled_contraction(plan, 0.5, A, sA, B, sB, 1.0, C, E)
    assert torch.equal(D, E)
    want, bound = ref.scaled(A, sA, (1, 128), B, sB, (1, 128), 0.5, 1.0, C)
    assert bool(((D.double() - want).abs() <= bound + 2.0 ** -23 * want.abs()).all())


def test_scaled_nan_stays_in_its_row_and_column(h):
    A, B = operand(200, 256, torch.float8_e4m3fn, 1), operand(300, 256, torch.float8_e4m3fn, 2)
    A[7, 200] = float("nan")
    sA, sB = torch.rand(200, 2, device="cuda"), torch.rand(3, 2, device="cuda")
    sA[9, 1], sB[2, 0] = float("inf"), float("nan")
    D = torch.zeros(200, 300, device="cuda")
    plan = h.scaled_contraction_plan(desc(h, A), (0, 2), desc(h, sA), (1, 128), desc(h, B), (1, 2), desc(h, sB), (128, 128), None,
                                     desc(h, D), (0, 1))
    h.scaled_contraction(plan, 1.0, A, sA, B, sB, 0.0, None, D)
    bad = ~D.isfinite()
    want = torch.zeros_like(bad)
    want[7], want[9], want[:, 256:] = True, True, True
    assert torch.equal(bad, want)


def test_scaled_rows_past_the_result_are_left(h):
    D = torch.full((40, 96), 7.0, device="cuda")
    A, B = operand(30, 300, torch.float8_e4m3fn, 1), operand(90, 300, torch.float8_e4m3fn, 2)
    sA, sB = torch.rand(30, 3, device="cuda"), torch.rand(1, 3, device="cuda")
    d = D[:30, :90]
    plan = h.scaled_contraction_plan(desc(h, A), (0, 2), desc(h, sA), (1, 128), desc(h, B), (1, 2), desc(h, sB), (128, 128), None,
                                     desc(h, d), (0, 1))
    h.scaled_contraction(plan, 1.0, A, sA, B, sB, 0.0, None, d)
    assert bool((D[30:] == 7).all()) and bool((D[:, 90:] == 7).all()) and bool((d != 7).all())


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (400, 520, 512), (1100, 1200, 256)])
def test_captured_together_on_another_stream(h, m, n, k):
    """x -> quantise -> product with quantised weights, captured on a side stream and replayed on new inputs."""
    x, w = torch.randn(m, k, device="cuda", dtype=torch.bfloat16), torch.randn(n, k, device="cuda") * 0.05
    wq, ws = quantize(h, w, (128, 128), E4)
    xq, xs = torch.empty(m, k, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(m, -(-k // 128), device="cuda")
    y = torch.empty(m, n, device="cuda", dtype=torch.bfloat16)
    dx, dq, ds = desc(h, x), desc(h, xq), desc(h, xs)
    plan = h.scaled_contraction_plan(dq, (0, 2), ds, (1, 128), desc(h, wq), (1, 2), desc(h, ws), (128, 128), None, desc(h, y), (0, 1))

    def step(stream):
        h.block_quantize(x, dx, (0, 1), (1, 128), xq, dq, (0, 1), xs, ds, stream)
        h.scaled_contraction(plan, 1.0, xq, xs, wq, ws, 0.0, None, y, stream)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream())
    for seed in (1, 2):
        x.copy_(torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        same(xq, xs, x, (1, 128), E4)
        want, bound = ref.scaled(xq, xs, (1, 128), wq, ws, (128, 128), 1.0, 0.0, None)
        assert bool(((y.double() - want).abs() <= bound + 1.01 * 2.0 ** -8 * want.abs()).all())


def test_a_wrong_pointer_is_refused(h):
    A, B = operand(16, 128, torch.float8_e4m3fn, 1), operand(16, 128, torch.float8_e4m3fn, 2)
    s, D = torch.ones(16, 1, device="cuda"), torch.zeros(16, 16, device="cuda")
    plan = h.scaled_contraction_plan(desc(h, A), (0, 2), desc(h, s), (1, 128), desc(h, B), (1, 2), desc(h, s), (1, 128), desc(h, D),
                                     desc(h, D), (0, 1))
    for args in [(None, s, B, s, 1.0, D, D), (A, None, B, s, 1.0, D, D), (A, s, B, s, 1.0, None, D), (A, s, B, s, 1.0, D, None),
                 (A, s, B, s, 1.0, D, D.data_ptr() + 2), (A, s.data_ptr() + 1, B, s, 1.0, D, D)]:
        with pytest.raises(ht.HiptensorError) as e:
            h.scaled_contraction(plan, 1.0, *args)
        assert e.value.status == ht.STATUS_INVALID_VALUE
    with pytest.raises(ht.HiptensorError) as e:
        h.scaled_contraction(plan, 1.0, A.cpu(), s, B, s, 1.0, D, D)
    assert e.value.status == ht.STATUS_ARCH_MISMATCH
