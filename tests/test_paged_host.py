"""The paged-cache operators' host side without a GPU: what the C entry points refuse before they touch the device, field
by field of the descriptors as qtb_paged.py packs them (a field in a wrong place would be refused for another reason),
and the Python checks."""
import pytest

import qtts_b200 as Q

torch = pytest.importorskip("torch")
import qtb_paged as P  # noqa: E402

INVALID, UNSUPPORTED = -1, -5
PTR = 1 << 20      # an aligned address that nothing reads: every call here is refused first


def plan_desc(**kw):
    f = dict(past=PTR, new=PTR, table=PTR, free=PTR, head=0, cu=PTR, kv=PTR, slot=PTR, pos=PTR, req=PTR, head_out=0, status=0,
             n_req=2, max_tokens=8, cols=4, stride=4, n_free=9, page=16)
    f.update(kw)
    return P._PLAN(*f.values())


def append_desc(**kw):
    f = dict(k=PTR, v=PTR, kp=PTR, vp=PTR, slot=PTR, status=0, ks0=256, ks1=128, vs0=256, vs1=128, kp0=4096, kp1=2048, kp2=128,
             vp0=4096, vp1=2048, vp2=128, tokens=3, n_kv=2, dim=128, page=16, pages=5, src=1, dst=1)
    f.update(kw)
    return P._APPEND(*f.values())


def attn_desc(**kw):
    f = dict(q=PTR, k=PTR, v=PTR, out=PTR, lse=PTR, cu=PTR, kv_len=PTR, table=PTR, status=0, ws=0, ws_bytes=0, qs0=512, qs1=128,
             os0=512, os1=128, ks0=4096, ks1=2048, ks2=128, vs0=4096, vs1=2048, vs2=128, t_stride=4, cols=4, page=16, pages=5,
             n_req=2, tokens=6, heads=4, n_kv=2, dim=128, max_new=3, max_kv=50, dtype=1, causal=1, window=0, scale=0.1)
    f.update(kw)
    return P._ATTN(*f.values())


def refusal(fn, desc, *more):
    rc = fn(desc, *more)
    return rc, Q.lib().qtb_last_error().decode()


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_req=-1), INVALID, "-1 requests"), (dict(max_tokens=1 << 30), INVALID, "1073741824 tokens"),
    (dict(n_free=-2), INVALID, "-2 free pages"), (dict(page=0), INVALID, "of 0"), (dict(cols=-3), INVALID, "-3 table columns"),
    (dict(cols=1 << 29, page=64), INVALID, "table columns"), (dict(stride=-1), INVALID, "table columns"),
    (dict(past=0), INVALID, "null"), (dict(new=0), INVALID, "null"), (dict(table=0), INVALID, "null"), (dict(free=0), INVALID, "null"),
    (dict(cu=0), INVALID, "null"), (dict(kv=0), INVALID, "null"), (dict(slot=0), INVALID, "null"), (dict(pos=0), INVALID, "null"),
    (dict(req=0), INVALID, "null"), (dict(head=PTR, head_out=PTR), INVALID, "another word")])
def test_plan_refusals(kw, code, text):
    rc, said = refusal(P._lib().qtb_paged_plan, plan_desc(**kw), 0)
    assert rc == code and text in said, said


@pytest.mark.parametrize("kw,code,text", [
    (dict(src=2), UNSUPPORTED, "type 2 into a cache of type 1"), (dict(dst=0), UNSUPPORTED, "cache of type 0"),
    (dict(dst=7, src=7), UNSUPPORTED, "type 7"), (dict(tokens=-1), INVALID, "-1 tokens"), (dict(n_kv=0), INVALID, "0 heads"),
    (dict(dim=12), INVALID, "of 12"), (dict(page=0), INVALID, "5 pages of 0"), (dict(pages=-1), INVALID, "-1 pages"),
    (dict(k=0), INVALID, "null"), (dict(v=0), INVALID, "null"), (dict(kp=0), INVALID, "null"), (dict(vp=0), INVALID, "null"),
    (dict(slot=0), INVALID, "null"), (dict(k=PTR + 2), INVALID, "16 bytes"), (dict(vp=PTR + 8), INVALID, "16 bytes"),
    (dict(ks0=252), INVALID, "16 bytes"), (dict(vs1=4), INVALID, "16 bytes"), (dict(kp2=-8), INVALID, "16 bytes"),
    (dict(vp0=4097), INVALID, "16 bytes")])
def test_append_refusals(kw, code, text):
    rc, said = refusal(P._lib().qtb_paged_append, append_desc(**kw), 0)
    assert rc == code and text in said, said


BOTH = [(dict(dtype=0), UNSUPPORTED, "dtype 0"), (dict(dim=96), UNSUPPORTED, "head_dim 96"),
        (dict(heads=5), INVALID, "5 query heads over 2 key heads"), (dict(n_kv=0), INVALID, "over 0"),
        (dict(heads=258, n_kv=2), UNSUPPORTED, "129 query heads to a key head"), (dict(n_req=-1), INVALID, "-1 requests"),
        (dict(tokens=1 << 30), INVALID, "tokens"), (dict(n_req=(1 << 24) - 1, heads=1024, n_kv=1024), UNSUPPORTED, "over 1024 key heads"),
        (dict(window=-1), INVALID, "window -1"), (dict(max_new=-4), INVALID, "max_new -4"), (dict(scale=float("nan")), INVALID, "finite"),
        (dict(scale=float("inf")), INVALID, "finite"), (dict(q=0), INVALID, "null"), (dict(out=0), INVALID, "null"),
        (dict(cu=0), INVALID, "null"), (dict(k=0), INVALID, "null"), (dict(v=0), INVALID, "null"), (dict(q=PTR + 4), INVALID, "16 bytes"),
        (dict(out=PTR + 8), INVALID, "16 bytes"), (dict(qs0=516), INVALID, "16 bytes"), (dict(os1=-128), INVALID, "16 bytes"),
        (dict(ks1=2044), INVALID, "16 bytes"), (dict(vs0=1), INVALID, "16 bytes"), (dict(qs1=0), INVALID, "expanded"),
        (dict(os0=0), INVALID, "expanded"), (dict(ks0=0), INVALID, "expanded"), (dict(vs1=0), INVALID, "expanded")]
PAGED = [(dict(page=24), INVALID, "page 24"), (dict(page=8), INVALID, "page 8"), (dict(pages=0), INVALID, "0 pages"),
         (dict(cols=-1), INVALID, "-1 table columns"), (dict(cols=1 << 27), INVALID, "table columns"), (dict(t_stride=-4), INVALID, "table"),
         (dict(kv_len=0), INVALID, "null"), (dict(table=0), INVALID, "null"), (dict(ks2=4), INVALID, "16 bytes"),
         (dict(vs2=0), INVALID, "expanded")]


@pytest.mark.parametrize("form,kw,code,text", [("paged", *c) for c in BOTH + PAGED] + [("prompt", *c) for c in BOTH])
def test_attention_refusals(form, kw, code, text):
    L = P._lib()
    for fn, more in ((getattr(L, f"qtb_{form}_attention"), 0), (L.qtb_attn_workspace, int(form == "paged"))):
        rc, said = refusal(fn, attn_desc(**kw), more)
        assert rc == code and text in said, said


def test_null_descriptors_and_nothing_to_do():
    L = P._lib()
    for fn in (L.qtb_paged_plan, L.qtb_paged_append, L.qtb_paged_attention, L.qtb_prompt_attention):
        assert fn(None, 0) == INVALID
    assert L.qtb_attn_workspace(None, 0) == INVALID
    for kw in (dict(tokens=0), dict(n_req=0)):
        assert L.qtb_prompt_attention(attn_desc(**kw), 0) == 0 and L.qtb_attn_workspace(attn_desc(**kw), 1) == 0
    assert L.qtb_paged_append(append_desc(tokens=0), 0) == 0


def test_tensors_off_the_gpu_are_refused():
    i, q, pool = torch.zeros(2, dtype=torch.int32), torch.zeros(4, 2, 64, dtype=torch.float16), torch.zeros(3, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        P.plan(i, i, i.reshape(2, 1), i, 16, 4)
    with pytest.raises(ValueError):
        P.append(q, q, pool, pool, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        P.paged_attention(q, pool, pool, i.reshape(1, 2), i, i[:1])
    with pytest.raises(ValueError):
        P.prompt_attention(q, q, q, i)


def test_status_words():
    P.check_status(torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="free list.*pool"):
        P.check_status(torch.tensor([P.NO_PAGES | P.PAGE], dtype=torch.int32))


# ------------------------------------------------------------------ a step's cache --
def cache_on_cpu(lengths=(20, 0, 3), page=16, max_len=64, pages=10):
    """A cache whose rows have some tokens, as after a step (the operators themselves need a GPU)."""
    import qtb_paged_step
    c = qtb_paged_step.PagedCache(1, len(lengths), pages, page, max_len, 1, 64, device="cpu")
    for r, n in enumerate(lengths):
        k = -(-n // page)
        c.table[r, :k] = c.free[c.taken:c.taken + k]
        c.taken += k
    c.length, c.head = list(lengths), torch.tensor([c.taken], dtype=torch.int32)
    return c


def state(c):
    return list(c.length), c.taken, int(c.head), c.free.tolist(), c.table.tolist()


@pytest.mark.parametrize("new,error", [([1, 1], ValueError), ([1, 1, 1, 1], ValueError), ([1, -1, 0], ValueError), ([], ValueError),
                                       ([45, 0, 0], RuntimeError), ([0, 65, 0], RuntimeError), ([1, 0, 2 ** 40], RuntimeError),
                                       ([44, 64, 61], RuntimeError)])
def test_steps_that_do_not_fit_are_refused(new, error):
    c = cache_on_cpu()
    before = state(c)
    with pytest.raises(error, match="room for 64|of each of 3 rows|pages needed"):
        c.begin(new)
    assert state(c) == before


def test_retired_rows_return_their_pages_once():
    c = cache_on_cpu()                       # pages 0, 1 | none | 2
    before = state(c)
    for rows in ([0, 0], [2, -1], [3], [-1], [0, 1, 0]):
        with pytest.raises(ValueError, match="rows"):
            c.retire(rows)
        assert state(c) == before
    c.retire([2, 1])
    assert c.free.tolist() == [3, 4, 5, 6, 7, 8, 9, 2] and c.length == [20, 0, 0] and c.taken == int(c.head) == 0
    c.retire([0])
    c.retire([])
    assert sorted(c.free.tolist()) == list(range(10)) and c.length == [0, 0, 0]


@pytest.mark.parametrize("kw", [dict(tokens=1, qs0=515, os0=3), dict(heads=1, n_kv=1, qs1=1, os1=0, ks1=5, vs1=-7), dict(pages=1, ks0=0, vs0=9)])
def test_strides_of_an_axis_of_one_are_not_refused(kw):
    """Such calls go on to the device (where there is one, they are given no token here)."""
    L = P._lib()
    rc, said = refusal(L.qtb_paged_attention, attn_desc(**kw, n_req=0), 0)
    assert rc == 0, said


def test_strides_of_other_axes_stay_refused():
    L = P._lib()
    for kw in (dict(tokens=1, qs1=12), dict(heads=1, n_kv=1, ks0=4), dict(pages=1, ks2=4)):
        rc, said = refusal(L.qtb_paged_attention, attn_desc(**kw, n_req=0), 0)
        assert rc == INVALID and "16 bytes" in said, said
