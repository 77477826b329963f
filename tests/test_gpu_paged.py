"""The paged-cache operators on the B200 (qtb_paged.py) against plain 64-bit
forms: block tables and slot maps, the append, attention over pages and over
packed prompts -- at the sizes, masks and layouts where they can go wrong.

Bounds of the attention tests.  With u the unit roundoff of the tensors' type
(half its spacing at 1: 2^-8 bf16, 2^-11 f16), o the exact output and
A = sum p |v| / sum p: the output's rounding gives u |o|, the probabilities'
rounding at most u A (f16 below 2^-14: 2^-25 absolute each, at most
L max|v| 2^-25), and a score error e changes o by at most 2 e A, where
e <= 2 d 2^-24 S for f32 sums of d products with S >= scale |q| |k| (sequential
sums and the multiplication by scale), plus 2^-21 for exp2 and the sums over
keys.  The log-sum-exp moves by e, by the sums' 2^-21 and by a few f32
roundings of itself."""
import ctypes as C
import math

import numpy as np
import pytest

import qtts_b200 as Q

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def torch(have_gpu_module):
    import torch as t
    return t


@pytest.fixture(scope="module")
def have_gpu_module():
    from conftest import gpu_available
    if not gpu_available():
        pytest.fail("GPU test selected but no CUDA device / engine library is available")


@pytest.fixture(scope="module")
def P(torch):
    import qtb_paged
    return qtb_paged


def kind(torch, name):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def exact_attention(torch, q, k, v, scale, causal, window):
    """q [n, H, D]: the last n tokens of k, v [L, KV, D] (n may pass L: the first ones then see nothing).
    Returns o, lse and A in 64 bits."""
    n, h, _ = q.shape
    l, kv = k.shape[:2]
    pos = torch.arange(l - n, l, device=q.device)[:, None]
    key = torch.arange(l, device=q.device)
    seen = torch.ones(n, l, dtype=torch.bool, device=q.device)
    if causal:
        seen &= key <= pos
    if window:
        seen &= key > pos - window
    o, lse, a = [], [], []
    for i in range(h):
        j = i * kv // h
        s = (q[:, i].double() @ k[:, j].double().T * scale).masked_fill(~seen, -math.inf)
        top = s.amax(1, keepdim=True).clamp(min=-1e300) if l else torch.zeros(n, 1, device=q.device, dtype=torch.double)
        p = torch.exp(s - top)
        z = p.sum(1, keepdim=True)
        some = z > 0
        w = torch.where(some, p / z.clamp(min=1e-300), 0.0)
        o.append(w @ v[:, j].double())
        a.append(w @ v[:, j].double().abs())
        lse.append(torch.where(some, top + z.clamp(min=1e-300).log(), -math.inf)[:, 0])
    return torch.stack(o, 1), torch.stack(lse, 1), torch.stack(a, 1)


def check(torch, out, lse, q, k, v, scale, causal, window, name):
    """One request's output against the exact one, element by element."""
    o, z, a = exact_attention(torch, q, k, v, scale, causal, window)
    if not q.shape[0]:
        return
    d, l = q.shape[2], max(k.shape[0], 1)
    big = float(k.double().norm(dim=-1).max()) if k.numel() else 0.0
    e = 2 * d * 2.0 ** -24 * abs(scale) * float(q.double().norm(dim=-1).max()) * big + 2.0 ** -21
    vmax = float(v.double().abs().max()) if v.numel() else 0.0
    tol = U[name] * (o.abs() + 1.001 * a) + 2 * e * a + (l * vmax * 2.0 ** -25 + 2.0 ** -24 if name == "f16" else 1e-30)
    err = (out.double() - o).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))
    none = torch.isinf(z)
    assert torch.equal(torch.isinf(lse) & (lse < 0), none)
    assert bool((out[none] == 0).all())
    if not bool(none.all()):
        zt = e + 2.0 ** -21 + 2.0 ** -21 * z[~none].abs()
        assert bool(((lse.double() - z)[~none].abs() <= zt).all()), float((lse.double() - z)[~none].abs().max())


def make_cache(torch, gen, lens, kv, d, page, name, spare=3, garbage=True, token_major=False):
    """Pools with every request's keys in pages of its own, in mixed order; the places that hold no key are NaN, and
    the table's unused entries are not pages.  Returns pools, table and the requests' K and V."""
    pages = sum(-(-n // page) for n in lens) + spare
    shape = (pages, page, kv, d) if token_major else (pages, kv, page, d)
    fill = math.nan if garbage else 0.0
    pools = [torch.full(shape, fill, dtype=kind(torch, name), device="cuda") for _ in range(2)]
    views = [p.transpose(1, 2) if token_major else p for p in pools]
    order = torch.randperm(pages, generator=gen).tolist()
    cols = max([-(-n // page) for n in lens] + [1]) + 2
    table = torch.full((len(lens), cols), -7, dtype=torch.int32)
    ks = []
    for r, n in enumerate(lens):
        both = [torch.randn(n, kv, d, generator=gen).to(kind(torch, name)).cuda() for _ in range(2)]
        ks.append(both)
        for j in range(-(-n // page)):
            pg = order.pop()
            table[r, j] = pg
            part = slice(j * page, min(n, (j + 1) * page))
            for view, x in zip(views, both):
                view[pg, :, :part.stop - part.start] = x[part].transpose(0, 1)
    return views[0], views[1], table.cuda(), ks


def offsets(torch, new):
    return torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")


def run_paged(torch, P, kv_len, new, heads, kv, d, page, name, window=0, causal=True, scale=None, seed=0, hints=True,
              token_major=False, mul=1.0):
    gen = torch.Generator().manual_seed(seed)
    kp, vp, table, ks = make_cache(torch, gen, kv_len, kv, d, page, name, token_major=token_major)
    t = sum(new)
    q = (torch.randn(t, heads, d, generator=gen) * mul).to(kind(torch, name)).cuda()
    cu = offsets(torch, new)
    lens = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    m = (max(new), max(kv_len)) if hints else (0, 0)
    out, lse = P.paged_attention(q, kp, vp, table, cu, lens, *m, scale=scale, causal=causal, window=window, status=status)
    P.check_status(status)
    at = 0
    for r, n in enumerate(new):
        check(torch, out[at:at + n], lse[at:at + n], q[at:at + n], *ks[r], 1 / math.sqrt(d) if scale is None else scale,
              causal, window, name)
        at += n


# ------------------------------------------------------- attention: pages --
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (16, 8), (28, 4), (10, 2), (8, 1), (40, 1)])
def test_single_tokens_over_pages(torch, P, name, d, heads, kv):
    kv_len = [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 500, 1031]
    run_paged(torch, P, kv_len, [1] * len(kv_len), heads, kv, d, 16, name, seed=heads + d)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 256])
@pytest.mark.parametrize("token_major", [False, True])
def test_page_sizes_and_pool_orders(torch, P, page, token_major):
    run_paged(torch, P, [1, 257, 300, 48, 200], [1, 3, 130, 48, 64], 8, 4, 128, page, "bf16", seed=page,
              token_major=token_major)
    run_paged(torch, P, [129, 700], [1, 1], 8, 4, 64, page, "f16", seed=page + 1, token_major=token_major)


@pytest.mark.parametrize("heads,kv,d,name", [(16, 8, 128, "bf16"), (14, 2, 64, "f16"), (5, 1, 128, "f16"), (8, 8, 64, "bf16"),
                                             (128, 1, 128, "bf16"), (65, 1, 64, "bf16")])
@pytest.mark.parametrize("new,kv_len", [([1, 64, 5, 2, 17], [900, 64, 6, 1025, 500]),
                                        ([128, 129, 127, 1], [128, 1000, 127, 3]),
                                        ([300], [2000]), ([33, 1], [4097, 4096])])
def test_chunks_over_pages(torch, P, heads, kv, d, name, new, kv_len):
    run_paged(torch, P, kv_len, new, heads, kv, d, 16, name, seed=heads + len(new))


# One tile of rows over 1 to 5 key tiles, and cut between blocks at odd places; the pages' other positions hold garbage.
@pytest.mark.parametrize("heads,kv,d,name", [(32, 2, 128, "bf16"), (40, 2, 64, "f16")])
@pytest.mark.parametrize("kv_len", [[127, 128, 129, 255, 256, 257, 384, 385, 512], [513, 640, 641], [3000, 130, 4001, 7, 1919],
                                    [2305] * 40])
@pytest.mark.parametrize("window", [0, 1, 140, 300])
def test_one_tile_of_rows_over_many_keys(torch, P, heads, kv, d, name, kv_len, window):
    run_paged(torch, P, kv_len, [3] * len(kv_len), heads, kv, d, 16, name, window=window, seed=len(kv_len) + window)


@pytest.mark.parametrize("new,kv_len", [([0, 1, 0, 3, 0], [5, 5, 0, 3, 100]), ([4, 2], [0, 1]), ([200, 1], [150, 0]),
                                        ([40], [0]), ([0, 0, 70], [0, 64, 70])])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths_of_zero_and_rows_that_see_nothing(torch, P, new, kv_len, causal):
    run_paged(torch, P, kv_len, new, 8, 4, 128, 16, "bf16", causal=causal, seed=3)


@pytest.mark.parametrize("window", [1, 2, 17, 64, 100, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("new,kv_len", [([1, 1, 1], [1, 70, 700]), ([150, 3, 1], [150, 400, 900]), ([260], [1300])])
def test_windows(torch, P, window, new, kv_len):
    run_paged(torch, P, kv_len, new, 8, 4, 128, 16, "bf16", window=window, seed=window % 97)
    run_paged(torch, P, kv_len, new, 6, 2, 64, 32, "f16", window=window, causal=False, seed=window % 89)


def test_evicted_pages_before_the_window_are_not_read(torch, P):
    gen = torch.Generator().manual_seed(5)
    kv_len, new, window = [500, 700], [1, 140], 100
    kp, vp, table, ks = make_cache(torch, gen, kv_len, 4, 128, 16, "bf16")
    table[0, :(500 - 100) // 16] = 10 ** 6      # not pages any more
    table[1, :(560 - 99) // 16] = -1
    q = torch.randn(141, 8, 128, generator=gen).bfloat16().cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = P.paged_attention(q, kp, vp, table, offsets(torch, new), torch.tensor(kv_len, dtype=torch.int32, device="cuda"),
                                 140, 700, window=window, status=status)
    P.check_status(status)
    for r, (a, b) in enumerate([(0, 1), (1, 141)]):
        check(torch, out[a:b], lse[a:b], q[a:b], *ks[r], 128 ** -0.5, True, window, "bf16")


@pytest.mark.parametrize("scale,mul", [(1.0, 1.0), (-0.3, 1.0), (0.0, 1.0), (128 ** -0.5, 40.0), (1e-6, 1.0)])
def test_scales_and_sharp_distributions(torch, P, scale, mul):
    run_paged(torch, P, [1000, 333, 1500], [1, 100, 260], 8, 4, 128, 16, "bf16", scale=scale, mul=mul, seed=8)
    run_paged(torch, P, [1000, 333], [1, 100], 8, 4, 64, 16, "f16", scale=scale, mul=min(mul, 8.0), seed=9)


def test_growing_maximum(torch, P):
    """Keys whose scores rise along the sequence, by little and by much: every tile renews the running maximum."""
    gen = torch.Generator().manual_seed(4)
    for step in (0.02, 0.5):
        n, d = 900, 128
        k = torch.zeros(n, 1, d)
        k[:, 0, 0] = torch.arange(n) * step
        k += 0.1 * torch.randn(n, 1, d, generator=gen)
        k, v = k.bfloat16().cuda(), torch.randn(n, 1, d, generator=gen).bfloat16().cuda()
        q = torch.randn(n, 2, d, generator=gen)
        q[:, :, 0] = 8.0
        q = q.bfloat16().cuda()
        out, lse = P.prompt_attention(q, k, v, offsets(torch, [n]), n)
        check(torch, out, lse, q, k, v, d ** -0.5, True, 0, "bf16")


@pytest.mark.parametrize("requests", [1, 33, 300])
def test_many_requests_without_hints(torch, P, requests):
    rng = np.random.default_rng(requests)
    new = [int(x) for x in rng.choice([0, 1, 1, 1, 2, 9, 40], requests)]
    new[0] = max(new[0], 1)
    kv_len = [n + int(x) for n, x in zip(new, rng.integers(0, 200, requests))]
    run_paged(torch, P, kv_len, new, 4, 2, 64, 16, "bf16", seed=1, hints=False)
    run_paged(torch, P, kv_len, new, 4, 2, 128, 16, "f16", seed=2)


def test_wrong_hints_change_nothing(torch, P):
    gen = torch.Generator().manual_seed(6)
    kv_len, new = [600, 64, 90], [1, 50, 20]
    kp, vp, table, ks = make_cache(torch, gen, kv_len, 2, 128, 16, "bf16")
    q = torch.randn(71, 4, 128, generator=gen).bfloat16().cuda()
    for m in [(1, 16), (10 ** 6, 10 ** 6), (0, 0), (50, 1)]:
        out, lse = P.paged_attention(q, kp, vp, table, offsets(torch, new), torch.tensor(kv_len, dtype=torch.int32, device="cuda"), *m)
        at = 0
        for r, n in enumerate(new):
            check(torch, out[at:at + n], lse[at:at + n], q[at:at + n], *ks[r], 128 ** -0.5, True, 0, "bf16")
            at += n


def test_results_repeat_bit_for_bit(torch, P):
    gen = torch.Generator().manual_seed(7)
    kv_len, new = [2000, 900, 130, 3000], [1, 200, 64, 1]
    kp, vp, table, _ = make_cache(torch, gen, kv_len, 4, 128, 16, "bf16")
    q = torch.randn(sum(new), 16, 128, generator=gen).bfloat16().cuda()
    args = (q, kp, vp, table, offsets(torch, new), torch.tensor(kv_len, dtype=torch.int32, device="cuda"), 200, 3000)
    a, la = P.paged_attention(*args)
    for _ in range(5):
        b, lb = P.paged_attention(*args)
        assert torch.equal(a, b) and torch.equal(la, lb)


@pytest.mark.parametrize("new", [1, 70])
def test_pages_outside_the_pool_are_reported(torch, P, new):
    gen = torch.Generator().manual_seed(8)
    kp, vp, table, _ = make_cache(torch, gen, [200], 2, 128, 16, "bf16")
    q = torch.randn(new, 4, 128, generator=gen).bfloat16().cuda()
    lens, cu = torch.tensor([200], dtype=torch.int32, device="cuda"), offsets(torch, [new])
    for wrong in (-1, kp.shape[0], 2 ** 31 - 1):
        t2 = table.clone()
        t2[0, 3] = wrong
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out, _ = P.paged_attention(q, kp, vp, t2, cu, lens, new, 200, status=status)
        assert int(status) == P.PAGE
        assert bool(torch.isfinite(out).all())
        with pytest.raises(RuntimeError, match="outside the pool"):
            P.check_status(status)


def test_lengths_beyond_the_tensors_are_clipped(torch, P):
    """Offsets and lengths that no plan makes (past the packed tokens, past the table, negative, falling): nothing out of
    range is touched, the tokens that exist get a value."""
    gen = torch.Generator().manual_seed(9)
    kp, vp, table, ks = make_cache(torch, gen, [64, 64], 2, 128, 16, "bf16", garbage=False)
    table.clamp_(min=0)
    q = torch.randn(10, 4, 128, generator=gen).bfloat16().cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    for cu, lens in [([0, 5, 10 ** 9], [64, 64]), ([-5, 5, 10], [64, 64]), ([0, 7, 3], [64, 64]), ([0, 5, 10], [-3, 2 ** 31 - 1])]:
        out = torch.full_like(q, 7.0)
        P.paged_attention(q, kp, vp, table, torch.tensor(cu, **i32), torch.tensor(lens, **i32), 10, 64, out=out)
        P.prompt_attention(q, q[:, :2], q[:, :2], torch.tensor(cu, **i32), 10, out=out)
    torch.cuda.synchronize()


def test_offsets_past_32_bits(torch, P):
    """A pool of more than 2^31 values whose used pages lie at its end."""
    kv, d, page = 8, 128, 64
    pages = 2 ** 31 // (kv * d * page) + 64
    gen = torch.Generator().manual_seed(10)
    kp = torch.empty(pages, kv, page, d, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    lens, new = [600, 700], [1, 200]
    table = torch.arange(pages - 24, pages, dtype=torch.int32, device="cuda").reshape(2, 12)
    ks = [[torch.randn(n, kv, d, generator=gen).bfloat16().cuda() for _ in range(2)] for n in lens]
    for r, n in enumerate(lens):
        slot = torch.arange(n, device="cuda") + int(table[r, 0]) * page
        P.append(*ks[r], kp, vp, slot)
        assert int(slot[0]) * kv * d > 2 ** 31
    q = torch.randn(201, 16, d, generator=gen).bfloat16().cuda()
    out, lse = P.paged_attention(q, kp, vp, table, offsets(torch, new), torch.tensor(lens, dtype=torch.int32, device="cuda"), 200, 700)
    check(torch, out[:1], lse[:1], q[:1], *ks[0], d ** -0.5, True, 0, "bf16")
    check(torch, out[1:], lse[1:], q[1:], *ks[1], d ** -0.5, True, 0, "bf16")


# ----------------------------------------------------- attention: prompts --
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,d", [(16, 8, 128), (4, 4, 64), (7, 1, 128), (24, 8, 64), (2, 1, 64)])
@pytest.mark.parametrize("new", [[1], [64], [130, 1, 0, 300, 17], [1, 2, 3], [511], [1, 1, 1, 128, 256, 129]])
def test_prompts(torch, P, name, heads, kv, d, new):
    gen = torch.Generator().manual_seed(sum(new))
    t = sum(new)
    # parts of one fused projection: neither contiguous nor of the same strides as the output
    qkv = torch.randn(t, heads + 2 * kv, d, generator=gen).to(kind(torch, name)).cuda()
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    for window, causal in ((0, True), (33, True), (0, False)):
        out, lse = P.prompt_attention(q, k, v, offsets(torch, new), max(new), window=window, causal=causal)
        at = 0
        for n in new:
            s = slice(at, at + n)
            check(torch, out[s], lse[s], q[s], k[s], v[s], d ** -0.5, causal, window, name)
            at += n


# Prompts whose items are dealt out by what they cost, and some too many or too unlike for that.
@pytest.mark.parametrize("heads,kv,d,name", [(4, 2, 128, "bf16"), (8, 8, 64, "f16"), (8, 1, 128, "f16")])
@pytest.mark.parametrize("new", [[700, 30, 1500, 5, 900, 64, 0, 333], [520] * 30, [1, 2000, 3], [600, 1, 513, 7] * 20])
@pytest.mark.parametrize("window", [0, 200])
def test_prompts_of_unlike_lengths(torch, P, heads, kv, d, name, new, window):
    gen = torch.Generator().manual_seed(sum(new) + heads)
    t = sum(new)
    q, k, v = (torch.randn(t, h, d, generator=gen).to(kind(torch, name)).cuda() for h in (heads, kv, kv))
    out, lse = P.prompt_attention(q, k, v, offsets(torch, new), max(new), window=window)
    at = 0
    for n in new:
        check(torch, out[at:at + n], lse[at:at + n], q[at:at + n], k[at:at + n], v[at:at + n], d ** -0.5, True, window, name)
        at += n


def test_long_prompt(torch, P):
    gen = torch.Generator().manual_seed(1)
    n = 4097
    q, k, v = (torch.randn(n, h, 128, generator=gen).bfloat16().cuda() for h in (4, 2, 2))
    out, lse = P.prompt_attention(q, k, v, offsets(torch, [n]), n)
    check(torch, out, lse, q, k, v, 128 ** -0.5, True, 0, "bf16")


def test_infinities_and_nan_of_another_prompt_stay_there(torch, P):
    gen = torch.Generator().manual_seed(2)
    new = [70, 50, 90]
    q, k, v = (torch.randn(210, h, 128, generator=gen).bfloat16().cuda() for h in (4, 2, 2))
    k[70:120], v[70:120] = math.inf, math.nan
    out, lse = P.prompt_attention(q, k, v, offsets(torch, new), 90)
    for a, b in ((0, 70), (120, 210)):
        check(torch, out[a:b], lse[a:b], q[a:b], k[a:b], v[a:b], 128 ** -0.5, True, 0, "bf16")
    assert bool(torch.isnan(out[70:120]).all())


def test_strided_heads_and_outputs(torch, P):
    gen = torch.Generator().manual_seed(3)
    q = torch.randn(8, 90, 128, generator=gen).bfloat16().cuda().transpose(0, 1)     # head-major
    k = torch.randn(90, 2, 2, 128, generator=gen).bfloat16().cuda()[:, :, 0]
    v = torch.randn(90, 4, 192, generator=gen).bfloat16().cuda()[:, ::2, 64:]
    out = torch.full((90, 8, 256), 9.0, dtype=torch.bfloat16, device="cuda")
    _, lse = P.prompt_attention(q, k, v, offsets(torch, [90]), 90, out=out[:, :, 64:192])
    check(torch, out[:, :, 64:192], lse, q, k, v, 128 ** -0.5, True, 0, "bf16")
    assert bool((out[:, :, :64] == 9).all()) and bool((out[:, :, 192:] == 9).all())


def test_side_stream_and_graph(torch, P):
    gen = torch.Generator().manual_seed(4)
    new, kv_len = [1, 80], [400, 300]
    kp, vp, table, ks = make_cache(torch, gen, kv_len, 4, 128, 16, "bf16")
    q = torch.randn(81, 8, 128, generator=gen).bfloat16().cuda()
    cu, lens = offsets(torch, new), torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(81, 8, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        P.paged_attention(q, kp, vp, table, cu, lens, 80, 400, out=out, lse=lse)
    side.synchronize()
    want = out.clone()
    check(torch, out[1:], lse[1:], q[1:], *ks[1], 128 ** -0.5, True, 0, "bf16")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        P.paged_attention(q, kp, vp, table, cu, lens, 80, 400, out=out, lse=lse)
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ------------------------------------------------------------- append, plan --
@pytest.mark.parametrize("src,name", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("t,kv,d,page", [(1, 1, 64, 16), (7, 8, 128, 16), (1000, 4, 128, 48), (333, 3, 8, 5)])
def test_append(torch, P, src, name, t, kv, d, page):
    gen = torch.Generator().manual_seed(t)
    pages = -(-t // page) + 2
    both = torch.randn(t, 2 * kv, d, generator=gen)
    both[0, 0, 0], both[-1, -1, -1] = math.inf, 1e-30      # the ends of the range round as they should
    both = both.to(kind(torch, src)).cuda()
    k, v = both[:, :kv], both[:, kv:]
    slot = torch.randperm(pages * page, generator=gen)[:t].cuda()
    if t > 1:
        slot[::3] = -1
    for token_major in (False, True):
        shape = (pages, page, kv, d) if token_major else (pages, kv, page, d)
        pools = [torch.randn(shape, generator=gen).to(kind(torch, name)).cuda() for _ in range(2)]
        want = [p.clone() for p in pools]
        view = (lambda p: p.transpose(1, 2)) if token_major else (lambda p: p)
        for w, x in zip(want, (k, v)):
            for i, s in enumerate(slot.tolist()):
                if s >= 0:
                    view(w)[s // page, :, s % page] = x[i].to(w.dtype)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        P.append(k, v, view(pools[0]), view(pools[1]), slot, status=status)
        assert torch.equal(pools[0], want[0]) and torch.equal(pools[1], want[1])
        assert int(status) == 0
    bad = slot.clone()
    bad[-1] = pages * page
    P.append(k, v, view(pools[0]), view(pools[1]), bad, status=status)
    assert int(status) == P.PAGE


def plain_plan(past, new, table, free, head, page, room):
    table, slot, pos, req, cu = table.copy(), [], [], [], [0]
    for r, (a, n) in enumerate(zip(past, new)):
        for j in range(-(-a // page), -(-(a + n) // page)):
            table[r, j] = free[head]
            head += 1
        for p in range(a, a + n):
            slot.append(int(table[r, p // page]) * page + p % page)
            pos.append(p)
            req.append(r)
        cu.append(len(slot))
    pad = [-1] * (room - len(slot))
    return table, slot + pad, pos + pad, req + pad, cu, head


@pytest.mark.parametrize("requests,page,longest,new_hi", [(1, 16, 0, 1), (1, 16, 40, 70), (3, 1, 9, 5), (64, 16, 2048, 1),
                                                          (1000, 16, 300, 40), (1025, 64, 500, 3), (5000, 128, 100, 2),
                                                          (2, 16, 10, 20000)])
def test_plan(torch, P, requests, page, longest, new_hi):
    rng = np.random.default_rng(requests + page)
    past = rng.integers(0, longest + 1, requests)
    new = rng.integers(0, new_hi + 1, requests)
    cols = -(-(longest + new_hi) // page) + 1
    used = int(sum(-(-int(a) // page) for a in past))
    need = int(sum(-(-int(a + n) // page) - -(-int(a) // page) for a, n in zip(past, new)))
    numbers = rng.permutation(used + need + 9).astype(np.int32)
    table = np.full((requests, cols + 3), -1, np.int32)
    at = 0
    for r, a in enumerate(past):
        n = -(-int(a) // page)
        table[r, :n] = numbers[at:at + n]
        at += n
    free = numbers[used:]
    for head, room in ((0, int(new.sum())), (4, int(new.sum()) + 77)):
        want = plain_plan(past, new, table, free, head, page, room)
        dt = torch.from_numpy(table).cuda()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        i32 = dict(dtype=torch.int32, device="cuda")
        got = P.plan(torch.tensor(past, **i32), torch.tensor(new, **i32), dt[:, :cols], torch.from_numpy(free).cuda(), page,
                     room, free_head=torch.tensor([head], **i32), status=status)
        P.check_status(status)
        assert np.array_equal(dt.cpu().numpy(), want[0])
        for x, y in zip((got.slot, got.pos, got.req, got.cu_new, got.free_head), (*want[1:5], [want[5]])):
            assert x.tolist() == list(y)
        assert np.array_equal(got.kv_len.cpu().numpy(), past + new)


def test_plan_of_no_requests(torch, P):
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    got = P.plan(e, e, e.reshape(0, 4), e, 16, 5)
    assert got.cu_new.tolist() == [0] and got.slot.tolist() == [-1] * 5 and got.free_head.tolist() == [0]


@pytest.mark.parametrize("what,bit", [("pages", 1), ("row", 2), ("room", 4), ("negative", 8), ("old page", 16)])
def test_plan_reports_what_does_not_fit(torch, P, what, bit):
    i32 = dict(dtype=torch.int32, device="cuda")
    past, new = torch.tensor([20, 0], **i32), torch.tensor([30, 40], **i32)
    table = torch.tensor([[5, 6, -1, -1], [-1] * 4], **i32)
    free, room = torch.arange(10, 20, **i32), 70
    if what == "pages":
        free = free[:3]
    if what == "row":
        new[1] = 65
        room = 95
    if what == "room":
        room = 50
    if what == "negative":
        past[0] = -4
    if what == "old page":
        table[0, 1] = -1
    status = torch.zeros(1, **i32)
    got = P.plan(past, new, table, free, 16, room, status=status)
    assert int(status) == bit
    slot = got.slot.tolist()
    assert len(slot) == room
    if what == "pages":      # 2 pages for the first request, 1 of 3 for the second
        assert table.tolist() == [[5, 6, 10, 11], [12, -1, -1, -1]] and slot[46:] == [-1] * 24 and got.free_head.tolist() == [3]
    if what == "row":        # 64 positions fit
        assert slot[94] == -1 and min(slot[:94]) >= 0 and table[1].tolist() == [12, 13, 14, 15]
    if what == "room":
        assert got.cu_new.tolist() == [0, 30, 50] and got.kv_len.tolist() == [50, 20]
    if what == "negative":
        assert got.kv_len.tolist() == [30, 40]
    if what == "old page":   # positions 20 .. 31 lay on it
        assert slot[:12] == [-1] * 12 and min(slot[12:]) >= 0


# ---------------------------------------------------------------- refusals --
def test_tensors_are_checked(torch, P):
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device="cuda")
    cu = torch.tensor([0, 4], **i32)
    P.prompt_attention(q, k, k, cu, 4)
    for a, kw in [((q.cpu(), k, k, cu), {}), ((q.float(), k.float(), k.float(), cu), {}), ((q, k.half(), k, cu), {}),
                  ((q, k, k[:, :, :64], cu), {}), ((q, k[:3], k, cu), {}), ((q, k, k, cu.long()), {}),
                  ((q[:, :7], k, k, cu), {}), ((q[:, :, ::2], k[:, :, ::2], k[:, :, ::2], cu), {}),
                  ((q[:, :, :32], k[:, :, :32], k[:, :, :32], cu), {}), ((q, k, k, cu), {"out": q.half()}),
                  ((q, k, k, cu), {"lse": torch.zeros(4, 4, device="cuda")}), ((q, k, k, cu), {"window": -1}),
                  ((q, k, k, cu), {"scale": math.nan}), ((q, k, k, cu), {"status": torch.zeros(2, **i32)})]:
        with pytest.raises((ValueError, RuntimeError)):
            P.prompt_attention(*a, 4, **kw)
    odd = torch.zeros(4 * 8 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].reshape(4, 8, 128)
    with pytest.raises(RuntimeError, match="16 bytes"):
        P.prompt_attention(odd, k, k, cu, 4)
    pool = torch.zeros(3, 2, 24, 128, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="multiple of 16"):
        P.paged_attention(q, pool, pool, torch.zeros(1, 2, **i32), cu, torch.tensor([4], **i32), 4, 4)
    slot = torch.zeros(4, dtype=torch.int64, device="cuda")
    for a in [(k, k, pool.half(), pool.half(), slot), (k, k, pool, pool, slot.int()), (k, k, pool, pool[:2], slot),
              (k, k[:, :1], pool, pool, slot), (k, k, pool.float(), pool.float(), slot)]:
        with pytest.raises((ValueError, RuntimeError)):
            P.append(*a)
    with pytest.raises(ValueError):
        P.plan(cu, cu[:1], torch.zeros(2, 2, **i32), cu, 16, 4)
    with pytest.raises(ValueError):
        P.plan(cu, cu, torch.zeros(2, 4, **i32)[:, ::2], cu, 16, 4)


# -------------------------------------------------------------- all together --
@pytest.mark.parametrize("rows,chunk,page,name", [(4, 256, 16, "bf16"), (2, 37, 48, "f16")])
def test_requests_served_in_chunks_equal_whole_prompts(torch, P, rows, chunk, page, name):
    """Plan, append and paged attention together, pages recycled between requests, against the prompt form.  Both round
    p and the output, each by at most u of the largest value: twice 2 u between them."""
    import qtb_paged_step
    lengths, prompts = [300, 64, 1, 333, 600, 90, 17], [250, 64, 1, 300, 590, 30, 1]
    worst = qtb_paged_step.serve(lengths, prompts, rows, chunk, page=page, dtype=kind(torch, name))
    for w in worst:
        for x in w:
            assert float(x) <= 4 * U[name], float(x)


# ------------------------------------------- lengths that the tensors do not hold --
def bounded_cache(torch, gen, room, kv, d, page, name):
    """Three requests' pages, `room` positions each, full of keys; returns pools, table, K and V."""
    kp, vp, table, ks = make_cache(torch, gen, [room] * 3, kv, d, page, name)
    return kp, vp, table[:, :room // page].contiguous(), ks


def check_at(torch, out, lse, q, k, v, first, causal, window, name):
    """Tokens at positions first, first + 1, ..., which may lie past the last key."""
    d, room = q.shape[2], k.shape[0]
    for i in range(q.shape[0]):
        p, s = first + i, slice(i, i + 1)
        if p < room:
            n = p + 1 if causal else room
            low = max(p - window + 1, 0) if window else 0
        else:
            n, low = room, min(max(p - window + 1, 0), room) if window else 0
        # the keys that it sees, all of them
        check(torch, out[s], lse[s], q[s], k[low:n], v[low:n], d ** -0.5, False, 0, name)


# hints: one token at most (the kernel of few rows), or none known
@pytest.mark.parametrize("hints", [(1, 1), (0, 0)])
@pytest.mark.parametrize("d,name", [(128, "bf16"), (64, "f16")])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 7), (True, 40), (False, 0), (False, 20)])
def test_tokens_keep_their_positions_past_the_table(torch, P, hints, d, name, causal, window):
    """A request that outgrew its row: the tokens that fit have the positions that they were appended at."""
    gen = torch.Generator().manual_seed(21)
    room, new, kv_len = 64, [10, 3, 5], [70, 50, 200]
    kp, vp, table, ks = bounded_cache(torch, gen, room, 2, d, 16, name)
    q = torch.randn(sum(new), 4, d, generator=gen).to(kind(torch, name)).cuda()
    out, lse = P.paged_attention(q, kp, vp, table, offsets(torch, new), torch.tensor(kv_len, dtype=torch.int32, device="cuda"),
                                 *hints, causal=causal, window=window)
    at = 0
    for n, end, (k, v) in zip(new, kv_len, ks):
        k, v = k[:end], v[:end]
        check_at(torch, out[at:at + n], lse[at:at + n], q[at:at + n], k, v, end - n, causal, window, name)
        at += n


@pytest.mark.parametrize("hints", [(1, 1), (0, 0)])
def test_tokens_keep_their_positions_where_offsets_leave_the_tokens(torch, P, hints):
    """Tokens that do not exist, before the first or past the last, take none of the others' positions."""
    gen = torch.Generator().manual_seed(22)
    kp, vp, table, ks = bounded_cache(torch, gen, 64, 2, 128, 16, "bf16")
    q = torch.randn(10, 4, 128, generator=gen).bfloat16().cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    for cu, spans in [([0, 5, 15, 15], [(0, 5, 59), (5, 10, 54)]), ([-3, 5, 10, 10], [(0, 5, 59), (5, 10, 59)]),
                      ([-2, 30, 30, 30], [(0, 10, 34)])]:
        out, lse = P.paged_attention(q, kp, vp, table, torch.tensor(cu, **i32), torch.tensor([64] * 3, **i32), *hints)
        for (a, b, first), (k, v) in zip(spans, ks):
            check_at(torch, out[a:b], lse[a:b], q[a:b], k, v, first, True, 0, "bf16")


def clipped(new, room):
    got, left = [], room
    for n in new:
        got.append(min(int(n), left))
        left -= got[-1]
    return got


@pytest.mark.parametrize("requests,page,longest,new_hi,share", [(2, 16, 40, 70, 0.6), (64, 16, 100, 40, 0.0), (64, 16, 100, 40, 0.5),
                                                                (1024, 16, 90, 33, 0.97), (2500, 32, 200, 3, 0.3),
                                                                (2500, 32, 200, 3, 0.9)])
def test_plan_takes_no_pages_for_dropped_tokens(torch, P, requests, page, longest, new_hi, share):
    rng = np.random.default_rng(requests + page)
    past, new = rng.integers(0, longest + 1, requests), rng.integers(1, new_hi + 1, requests)
    cols = -(-(longest + new_hi) // page)
    used = sum(-(-int(a) // page) for a in past)
    numbers = rng.permutation(used + int(new.sum()) // page + requests).astype(np.int32)
    table, at = np.full((requests, cols), -1, np.int32), 0
    for r, a in enumerate(past):
        n = -(-int(a) // page)
        table[r, :n] = numbers[at:at + n]
        at += n
    free, room = numbers[used:], int(share * new.sum())
    want = plain_plan(past, clipped(new, room), table, free, 2, page, room)
    i32 = dict(dtype=torch.int32, device="cuda")
    dt, status = torch.from_numpy(table).cuda(), torch.zeros(1, **i32)
    got = P.plan(torch.tensor(past, **i32), torch.tensor(new, **i32), dt, torch.from_numpy(free).cuda(), page, room,
                 free_head=torch.tensor([2], **i32), status=status)
    assert int(status) == P.ROOM
    assert np.array_equal(dt.cpu().numpy(), want[0])
    for x, y in zip((got.slot, got.pos, got.req, got.cu_new, got.free_head), (*want[1:5], [want[5]])):
        assert x.tolist() == list(y)
    assert np.array_equal(got.kv_len.cpu().numpy(), past + np.array(clipped(new, room)))


@pytest.mark.parametrize("what,head,rows", [("room", 4, [[5, 6, 10, 11], [12, 13, -1, -1]]), ("row", 6, [[5, 6, 10, 11], [12, 13, 14, 15]]),
                                            ("negative", 5, [[10, 11, -1, -1], [12, 13, 14, -1]])])
def test_plan_counts_the_pages_it_took(torch, P, what, head, rows):
    i32 = dict(dtype=torch.int32, device="cuda")
    past, new, room = torch.tensor([20, 0], **i32), torch.tensor([30, 40], **i32), 70
    table = torch.tensor([[5, 6, -1, -1], [-1] * 4], **i32)
    if what == "room":
        room = 50
    if what == "row":
        new[1] = 65
        room = 95
    if what == "negative":
        past[0] = -4
        table[0] = -1
    got = P.plan(past, new, table, torch.arange(10, 20, **i32), 16, room)
    assert got.free_head.tolist() == [head] and table.tolist() == rows


def test_workspace_reused_by_calls_in_a_row(torch, P):
    """Calls that cut their work, one behind the other in the same workspace: each joins its own parts."""
    gen = torch.Generator().manual_seed(23)
    kv_len = [3000, 1500]
    kp, vp, table, _ = make_cache(torch, gen, kv_len, 2, 128, 16, "bf16")
    lens = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    calls = []
    for i, new in enumerate([[1, 1], [30, 4], [2, 1], [64, 64]] * 4):
        q = torch.randn(sum(new), 16, 128, generator=gen).bfloat16().cuda()
        calls.append((q, kp, vp, table, offsets(torch, new), lens, max(new), 3000))
    alone = []
    for a in calls:
        alone.append(P.paged_attention(*a))
        torch.cuda.synchronize()
    for _ in range(5):
        for (o, z), (a, b) in zip([P.paged_attention(*a) for a in calls], alone):
            assert torch.equal(o, a) and torch.equal(z, b)


# ------------------------------------------------------ what the device reports --
@pytest.mark.parametrize("hints", [(1, 1), (0, 0)])
@pytest.mark.parametrize("requests", [2, 70])
@pytest.mark.parametrize("cu,lens,bits", [([0, 5, 10], [64, 65], 2), ([0, 5, 10], [2 ** 31 - 1, 64], 2), ([0, 5, 10], [64, -3], 8),
                                          ([0, 5, 10 ** 9], [64, 64], 8), ([-5, 5, 10], [64, 64], 8), ([0, 7, 3], [64, 64], 8),
                                          ([0, 5, 10], [64, 64], 0), ([0, 12, 12], [-1, 70], 10)])
def test_attention_reports_lengths_out_of_range(torch, P, hints, requests, cu, lens, bits):
    gen = torch.Generator().manual_seed(24)
    kp, vp, table, _ = bounded_cache(torch, gen, 64, 2, 128, 16, "bf16")
    q = torch.randn(10, 4, 128, generator=gen).bfloat16().cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    more = requests - 2              # requests of no token behind them
    cu, lens = cu + [cu[-1]] * more, lens + [64] * more
    rows = table[:2].repeat(requests // 2, 1)
    status = torch.zeros(1, **i32)
    P.paged_attention(q, kp, vp, rows, torch.tensor(cu, **i32), torch.tensor(lens, **i32), *hints, status=status)
    assert int(status) == bits
    wrong = P.LENGTH if min(cu) < 0 or max(cu) > 10 or sorted(cu) != cu else 0     # without lengths of keys
    for scale in (1.0, -1.0):
        status.zero_()
        P.prompt_attention(q, q[:, :2], q[:, :2], torch.tensor(cu, **i32), scale=scale, status=status)
        assert int(status) == wrong


@pytest.mark.parametrize("requests", [12, 100])
def test_requests_that_share_tokens_without_end(torch, P, requests):
    """Offsets that fall let requests have the same tokens; work that could no longer be counted is not begun."""
    gen = torch.Generator().manual_seed(25)
    n, d = 10240, 64
    q, k, v = (torch.randn(n, 1, d, generator=gen).bfloat16().cuda() for _ in range(3))
    i32 = dict(dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, n] * 6 + [n] * (requests - 11), **i32)    # six times 40 pairs of tiles, where there are 40
    status, out = torch.zeros(1, **i32), torch.full_like(q, 7.0)
    P.prompt_attention(q, k, v, cu, out=out, status=status)
    assert int(status) == P.LENGTH and bool((out == 7).all())
    pools = [x.reshape(n // 64, 64, 1, d).transpose(1, 2) for x in (k, v)]
    table = torch.arange(n // 64, **i32).expand(requests, -1)
    status.zero_()
    P.paged_attention(q, *pools, table, cu, torch.full((requests,), n, **i32), out=out, status=status)
    assert int(status) == P.LENGTH and bool((out == 7).all())


@pytest.mark.parametrize("hints", [(1, 1), (0, 0)])
def test_offsets_that_fall(torch, P, hints):
    gen = torch.Generator().manual_seed(30)
    kp, vp, table, ks = bounded_cache(torch, gen, 64, 2, 128, 16, "bf16")
    q = torch.randn(10, 4, 128, generator=gen).bfloat16().cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    status, out = torch.zeros(1, **i32), torch.full_like(q, 7.0)
    _, lse = P.paged_attention(q, kp, vp, table, torch.tensor([0, 7, 3, 3], **i32), torch.tensor([64] * 3, **i32), *hints, out=out,
                               status=status)
    assert int(status) == P.LENGTH and bool((out[7:] == 7).all())
    check_at(torch, out[:7], lse[:7], q[:7], *ks[0], 57, True, 0, "bf16")


# ------------------------------------------------------------------------- steps --
def test_a_step_without_tokens(torch, P):
    import qtb_paged_step
    cache = qtb_paged_step.PagedCache(1, 3, 8, 16, 64, 2, 64)
    for new in ([0, 0, 0], [5, 0, 1], [0, 0, 0], [1, 1, 0]):
        step = cache.begin(new)
        t = sum(new)
        assert step.tokens == t and step.max_new == max(new)
        q, k, v = (torch.randn(t, h, 64, device="cuda").bfloat16() for h in (4, 2, 2))
        assert cache.attend(step, 0, q, k, v).shape == (t, 4, 64)
    cache.check()
    assert cache.length == [6, 1, 1] and int(cache.head) == cache.taken == 3


# ------------------------------------------------------------ rows beside others --
@pytest.mark.parametrize("heads,kv", [(4, 4), (5, 1), (8, 2)])
@pytest.mark.parametrize("n", [1, 17, 70, 130])
def test_results_do_not_depend_on_other_requests(torch, P, heads, kv, n):
    """The rows that a tile has beside a request's own are the next request's, or old ones: they must not move its running
    maximum, which would round its results differently."""
    gen = torch.Generator().manual_seed(26)
    d, more = 128, 200
    q = torch.randn(n + more, heads, d, generator=gen).bfloat16().cuda()
    k, v = (torch.randn(n + more, kv, d, generator=gen).bfloat16().cuda() for _ in range(2))
    cu = offsets(torch, [n, more])
    want, lse = P.prompt_attention(q, k, v, cu, more)
    check(torch, want[:n], lse[:n], q[:n], k[:n], v[:n], d ** -0.5, True, 0, "bf16")
    for mul in (0.0, -3.0, 30.0, 300.0):
        q2 = q.clone()
        q2[n:] *= mul
        out, z = P.prompt_attention(q2, k, v, cu, more)
        assert torch.equal(out[:n], want[:n]) and torch.equal(z[:n], lse[:n])


@pytest.mark.parametrize("name", ["bf16", "f16"])
def test_results_over_pages_do_not_depend_on_other_requests(torch, P, name):
    gen = torch.Generator().manual_seed(27)
    kv_len, new = [700, 300, 900], [9, 100, 3]
    kp, vp, table, _ = make_cache(torch, gen, kv_len, 2, 128, 16, name)
    q = torch.randn(sum(new), 10, 128, generator=gen).to(kind(torch, name)).cuda()
    lens = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    want, lse = P.paged_attention(q, kp, vp, table, offsets(torch, new), lens, 100, 900)
    for mul in (0.0, -3.0, 30.0):
        q2 = q.clone()
        q2[9:109] *= mul
        out, z = P.paged_attention(q2, kp, vp, table, offsets(torch, new), lens, 100, 900)
        for s in (slice(0, 9), slice(109, 112)):
            assert torch.equal(out[s], want[s]) and torch.equal(z[s], lse[s])


# --------------------------------------------------------------------- arguments --
def test_bounds_of_any_size_change_nothing(torch, P):
    gen = torch.Generator().manual_seed(28)
    kv_len, new = [600, 64], [1, 3]
    kp, vp, table, ks = make_cache(torch, gen, kv_len, 2, 128, 16, "bf16")
    q = torch.randn(4, 8, 128, generator=gen).bfloat16().cuda()
    for m in [(2 ** 62, 2 ** 62), (2 ** 61 + 1, 600), (2 ** 63 - 1, 2 ** 63 - 1)]:
        out, lse = P.paged_attention(q, kp, vp, table, offsets(torch, new), torch.tensor(kv_len, dtype=torch.int32, device="cuda"), *m)
        at = 0
        for r, n in enumerate(new):
            check(torch, out[at:at + n], lse[at:at + n], q[at:at + n], *ks[r], 128 ** -0.5, True, 0, "bf16")
            at += n


def test_strides_of_single_tokens_and_heads_do_not_matter(torch, P):
    """A tensor's stride along an axis of one is any number: cut from a wider row, or expanded."""
    gen = torch.Generator().manual_seed(29)
    kp, vp, table, ks = make_cache(torch, gen, [300], 1, 128, 16, "bf16")
    lens, cu = torch.tensor([300], dtype=torch.int32, device="cuda"), offsets(torch, [1])
    row = torch.randn(1, 6 * 128 + 3, generator=gen).bfloat16().cuda()
    q, k, v = (row.as_strided((1, n, 128), (row.shape[1], 128 if n > 1 else 3, 1), a * 128) for a, n in ((0, 4), (4, 1), (5, 1)))
    out, lse = P.paged_attention(q, kp, vp, table, cu, lens, 1, 300)
    check(torch, out, lse, q, *ks[0], 128 ** -0.5, True, 0, "bf16")
    out, lse = P.prompt_attention(q, k, v, cu, 1)
    check(torch, out, lse, q, k, v, 128 ** -0.5, True, 0, "bf16")
    slot = torch.tensor([299 + 16 * int(table[0, 18]) - 288], device="cuda")
    odd = [p.as_strided(p.shape, (p.stride(0), 3, p.stride(2), 1)) for p in (kp, vp)]     # one head
    P.append(k, v, *odd, slot)
    out, lse = P.paged_attention(q, *odd, table, cu, lens, 1, 300)
    keys, values = (torch.cat([x[:299], y]) for x, y in zip(ks[0], (k, v)))
    check(torch, out, lse, q, keys, values, 128 ** -0.5, True, 0, "bf16")


def test_results_that_need_a_gradient_say_that_there_is_none(torch, P):
    q = torch.randn(5, 4, 64, device="cuda").half().requires_grad_()
    k, v = (torch.randn(5, 2, 64, device="cuda").half() for _ in range(2))
    cu = offsets(torch, [5])
    want, _ = P.prompt_attention(q.detach(), k, v, cu, 5)
    assert not want.requires_grad
    out, lse = P.prompt_attention(q, k, v, cu, 5)
    assert torch.equal(out, want)
    for x in (out, lse):
        with pytest.raises(RuntimeError, match="no backward"):
            x.float().sum().backward()
    with torch.no_grad():
        assert not P.prompt_attention(q, k, v, cu, 5)[0].requires_grad
    pool = torch.zeros(2, 2, 16, 64, device="cuda").half()
    i32 = dict(dtype=torch.int32, device="cuda")
    out, _ = P.paged_attention(q, pool, pool, torch.zeros(1, 1, **i32), cu, torch.tensor([5], **i32), 5, 5)
    with pytest.raises(RuntimeError, match="no backward"):
        out.float().sum().backward()
    with pytest.raises(RuntimeError, match="gradient"):
        P.prompt_attention(q, k, v, cu, 5, out=torch.empty_like(want))
