"""Drafted tokens over a K/V cache in pages (manual_whisper_amd.paged): refusals on the CPU, then every operator on the GPU
against its plain 64-bit restatement (oracle/paged_ref.py)."""
import ctypes as C
import itertools

import numpy as np
import pytest

from manual_whisper_amd import _lib             # before torch: it sets the number of hardware queues
import torch
from oracle import paged_ref as ref

BAD = 0x1000            # an address that nothing may follow: refusals come before anything is read


# ------------------------------------------------------------------------------------------------ refusals, no GPU

def _cache(**kw):
    c = _lib.PagedCache(BAD, BAD, None, None, 64 * 20 * 64, 64 * 64, 64, 8, 64, 20, 64, 1)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _refused(rc, who):
    text = _lib.load().mw_last_error(None).decode()
    assert rc == -1 and text.startswith(who + ": "), (rc, text)
    return text


CACHE_FAULTS = [dict(k=None), dict(v=None), dict(dtype=0), dict(dtype=4), dict(head_dim=32), dict(head_dim=96), dict(n_heads=0), dict(page_size=8),
                dict(page_size=48), dict(page_size=8192), dict(n_pages=0), dict(n_pages=1 << 26), dict(dtype=3), dict(k_scale=BAD), dict(v_scale=BAD),
                dict(page_stride=4), dict(token_stride=60), dict(head_stride=100), dict(k=BAD + 8), dict(token_stride=8), dict(page_stride=-64)]


@pytest.mark.parametrize("fault", CACHE_FAULTS, ids=str)
def test_cache_descriptions_are_checked(fault):
    lib = _lib.load()
    c = _cache(**fault)
    _refused(lib.mw_paged_write(C.byref(c), BAD, BAD, 1, 1280, 64, 1280, 64, BAD, 4, 0, None), "mw_paged_write")
    _refused(lib.mw_paged_compact(C.byref(c), 1, 0, BAD, 8, 8, BAD, BAD, 4, BAD, 2, 0, None), "mw_paged_compact")
    a = _tree_args(cache=c)
    _refused(lib.mw_tree_attention(C.byref(a), 0, None), "mw_tree_attention")
    assert lib.mw_tree_attention_workspace(C.byref(a)) == -1


def _plan_args(**kw):
    a = _lib.PlanArgs(2, 8, 64, 16, 8, BAD, BAD, None, BAD, 8, BAD, BAD + 16, BAD, BAD, BAD + 32, BAD, BAD, BAD, BAD, None, 0, BAD, BAD, 4, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fault", [dict(batch=0), dict(batch=2049), dict(rows=-1), dict(page_size=24), dict(page_size=0), dict(max_pages=0),
                                   dict(max_pages=1 << 26), dict(table_stride=7), dict(n_pages=0), dict(kept=None), dict(fresh=None),
                                   dict(table=None), dict(pages_in=None), dict(pages_out=BAD), dict(n_free_out=BAD), dict(free_list=None),
                                   dict(row_start=None), dict(admitted=None), dict(slots=None), dict(positions=None), dict(parents=BAD),
                                   dict(parents=BAD, mask=BAD, mask_words=9), dict(parents=BAD, mask=BAD, mask_words=0), dict(units=None),
                                   dict(unit_start=None), dict(chunk_units=-1), dict(chunk_units=70000), dict(chunk_min=0), dict(units=BAD + 4)], ids=str)
def test_plan_arguments_are_checked(fault):
    _refused(_lib.load().mw_paged_plan(C.byref(_plan_args(**fault)), 0, None), "mw_paged_plan")


@pytest.mark.parametrize("change", [dict(dtype=0), dict(dtype=2), dict(rows=-1), dict(k=None), dict(v=None), dict(slots=None), dict(k=BAD + 8),
                                    dict(k_row=1281), dict(v_head=60)], ids=str)
def test_write_arguments_are_checked(change):
    a = dict(k=BAD, v=BAD, dtype=1, k_row=1280, k_head=64, v_row=1280, v_head=64, slots=BAD, rows=4)
    a.update(change)
    _refused(_lib.load().mw_paged_write(C.byref(_cache()), a["k"], a["v"], a["dtype"], a["k_row"], a["k_head"], a["v_row"], a["v_head"], a["slots"],
                                        a["rows"], 0, None), "mw_paged_write")


def _tree_args(**kw):
    a = _lib.TreeArgs(_cache(), BAD, 1280, 64, BAD, 1280, 64, 1, 20, 8, 2, 4, BAD, 8, 8, BAD, BAD, BAD, BAD, 2, None, 0, 0.125, None, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fault", [dict(dtype=0), dict(dtype=2), dict(n_heads=0), dict(n_heads=30), dict(batch=0), dict(rows=-1), dict(max_nodes=-1),
                                   dict(n_units=-1), dict(max_pages=0), dict(table_stride=7), dict(mask=BAD, mask_words=0), dict(scale=0.0),
                                   dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(out=None), dict(table=None), dict(kept=None),
                                   dict(row_start=None), dict(units=None), dict(unit_start=None), dict(q=BAD + 2), dict(q_row_stride=1284),
                                   dict(out_head_stride=62), dict(out=BAD + 4), dict(units=BAD + 8), dict(n_units=3),
                                   dict(n_units=3, workspace=BAD, workspace_bytes=100), dict(mask=BAD, mask_words=1, max_nodes=40)], ids=str)
def test_attention_arguments_are_checked(fault):
    _refused(_lib.load().mw_tree_attention(C.byref(_tree_args(**fault)), 0, None), "mw_tree_attention")


def test_attention_workspace_is_none_without_cuts():
    lib = _lib.load()
    assert lib.mw_tree_attention_workspace(C.byref(_tree_args())) == 0
    assert lib.mw_tree_attention_workspace(C.byref(_tree_args(n_units=5))) == 5 * 20 * 4 * 66 * 4


@pytest.mark.parametrize("fault", [dict(dtype=3), dict(rows=-1), dict(vocab=0), dict(batch=0), dict(depth=0), dict(depth=1025), dict(logits=None),
                                   dict(tokens=None), dict(parents=None), dict(row_start=None), dict(best=None), dict(path=None), dict(count=None),
                                   dict(out_tokens=None), dict(workspace=None), dict(logits_stride=99), dict(logits=BAD + 2), dict(workspace_bytes=8)], ids=str)
def test_accept_arguments_are_checked(fault):
    a = _lib.AcceptArgs(BAD, 100, 0, 8, 100, 2, 4, None, BAD, BAD, BAD, BAD, BAD, BAD, BAD, BAD, 8 * 8)
    for k, v in fault.items():
        setattr(a, k, v)
    _refused(_lib.load().mw_tree_accept(C.byref(a), 0, None), "mw_tree_accept")


@pytest.mark.parametrize("change", [dict(layers=0), dict(layers=2, stride=60), dict(layers=2, stride=1284), dict(batch=0), dict(columns=-1),
                                    dict(max_pages=0), dict(table_stride=3), dict(table=None), dict(kept=None), dict(path=None), dict(count=None)], ids=str)
def test_compact_arguments_are_checked(change):
    a = dict(layers=1, stride=0, table=BAD, table_stride=8, max_pages=8, kept=BAD, path=BAD, columns=4, count=BAD, batch=2)
    a.update(change)
    _refused(_lib.load().mw_paged_compact(C.byref(_cache()), a["layers"], a["stride"], a["table"], a["table_stride"], a["max_pages"], a["kept"],
                                          a["path"], a["columns"], a["count"], a["batch"], 0, None), "mw_paged_compact")


def test_tensors_are_checked_before_the_library_sees_them():
    from manual_whisper_amd import paged
    from manual_whisper_amd.engine import EngineError
    k = torch.zeros(4, 2, 64, 64, dtype=torch.float16)
    for fault in (lambda: paged.PagedCache(k, k), lambda: paged.PagedCache(k, k[:2]), lambda: paged.PagedCache(k, k.transpose(1, 2)),
                  lambda: paged.PagePool(torch.zeros(2, 4, dtype=torch.int32), None, None, None, 64),
                  lambda: paged.accept(torch.zeros(4, 10), None, None, torch.zeros(2, dtype=torch.int32), 4)):
        with pytest.raises(EngineError):
            fault()


def test_calls_beyond_one_launch_are_refused():
    """A launch has fewer than 2^32 threads along a dimension: what would need more is refused, at the first size that does."""
    lib = _lib.load()
    rows = 2 ** 32 // (20 * 8)                                # 8 threads per (row, head) of 64 values
    assert "too many rows" in _refused(lib.mw_paged_write(C.byref(_cache()), BAD, BAD, 1, 1280, 64, 1280, 64, BAD, rows, 0, None), "mw_paged_write")
    for fault in (dict(n_units=838861), dict(batch=1 << 13, n_units=(1 << 13) + 1, max_nodes=1 << 11)):          # attention; join of the pieces
        args = _tree_args(workspace=BAD, workspace_bytes=1 << 62, **fault)
        assert "too many units or rows" in _refused(lib.mw_tree_attention(C.byref(args), 0, None), "mw_tree_attention")
    a = _lib.AcceptArgs(BAD, 100, 0, 1 << 24, 100, 2, 4, None, BAD, BAD, BAD, BAD, BAD, BAD, BAD, BAD, 1 << 40)
    assert "rows" in _refused(lib.mw_tree_accept(C.byref(a), 0, None), "mw_tree_accept")


def test_units_of_the_restatement_cover_every_key_once():
    """The oracle's own work units: pieces of a request follow each other and reach its end, whatever the lengths."""
    rng = np.random.default_rng(5)
    for _ in range(200):
        B = int(rng.integers(1, 9))
        kept, fresh = rng.integers(0, 3000, B).tolist(), rng.integers(0, 40, B).tolist()
        target, least = int(rng.integers(0, 40)), int(rng.choice([1, 64, 100, 512]))
        n = [-(-(a + b) // 16) for a, b in zip(kept, fresh)]
        got = ref.plan(kept, fresh, 16, 300, sum(fresh), [0] * B, [[-1] * 300 for _ in range(B)], list(range(sum(n))), sum(n), target=target, least=least)
        assert len(got["units"]) == B + target and got["admitted"] == [1] * B
        for b in range(B):
            mine = [u for u in got["units"] if u[0] == b]
            assert (fresh[b] > 0) == bool(mine) and all(u[3] == len(mine) and u[1] % 64 == 0 or u[1] == u[2] for u in mine)
            assert not mine or (mine[0][1] == 0 and mine[-1][2] == kept[b] + fresh[b] and all(x[2] == y[1] for x, y in zip(mine, mine[1:])))


# ------------------------------------------------------------------------------------------------ GPU

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def _dev(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _forest(rng, sizes, faults=False):
    """Parents of trees: any earlier node; with `faults` also what is no earlier node of the tree."""
    out = []
    for n in sizes:
        for i in range(n):
            u = int(rng.integers(0, 10))
            if faults and u == 0:
                out.append(int(rng.choice([-7, i, i + 1, 1 << 30])))
            elif i == 0 or (faults and u == 1):
                out.append(-1)
            else:
                out.append(int(rng.integers(max(0, i - 4), i)))
    return out


def _signed(words):
    return np.array(words, dtype=np.uint32).astype(np.int64).reshape(len(words), -1) if len(words) else np.zeros((0, 1), np.int64)


PLANS = [  # kept, fresh, page, max_pages, spare pages, pages held beyond the kept tokens', tree words, row capacity beyond the sum, target, least
    ([0], [1], 16, 1, 0, [0], 0, 0, 0, 64),
    ([0, 0], [0, 0], 16, 4, 3, [0, 2], 0, 2, 4, 64),
    ([5, 0, 31, 16], [3, 8, 1, 0], 16, 6, 0, [0, 0, 0, 0], 1, 3, 0, 64),
    ([100, 1, 63, 64, 65], [5, 33, 1, 64, 7], 64, 4, 1, [1, 0, 2, 0, 0], 2, 0, 8, 64),
    ([100, 1, 63, 64, 65], [5, 33, 1, 64, 7], 64, 4, -2, [1, 0, 2, 0, 0], 2, 0, 8, 64),
    ([40, -3, 20, 7], [4, 4, -1, 9], 16, 4, 2, [0, 0, 0, 0], 1, 0, 3, 1),
    ([10, 20, 30], [10, 40, 10], 16, 8, 6, [0, 0, 0], 1, 0, 2, 64),                     # the second tree is larger than its mask
    ([10, 20, 30], [10, 40, 10], 16, 3, 6, [0, 0, 0], 0, 0, 2, 64),                     # the second request is larger than its table
    ([10, 20, 30], [10, 12, 10], 16, 8, 6, [0, 0, 0], 0, -5, 2, 64),                    # the last request's rows do not fit
    ([1000, 3, 70000, 512], [300, 1, 20, 2049], 128, 600, 5, [0, 3, 1, 0], 0, 7, 40, 500),
    ([0] * 7, [256, 255, 1, 2, 129, 64, 65], 32, 9, 4, [0] * 7, 8, 1, 3, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(PLANS)))
def test_plan(case):
    from manual_whisper_amd import paged
    kept, fresh, page, max_pages, spare, extra, words, over, target, least = PLANS[case]
    rng = np.random.default_rng(case)
    B = len(kept)
    held = [min(max_pages, max(0, -(-max(0, k) // page)) + e) for k, e in zip(kept, extra)]
    wanted = sum(max(0, -(-(max(0, k) + max(0, f)) // page) - h) for k, f, h in zip(kept, fresh, held))
    n_free = max(0, wanted + spare)
    ids = rng.permutation(sum(held) + n_free + 1).tolist()
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (max_pages - h))
        at += h
    free = ids[at:at + n_free] + [-1] * (len(ids) - n_free)
    total = sum(max(0, f) for f in fresh)
    rows = max(0, total + over)
    parents = _forest(rng, [max(0, f) for f in fresh], faults=True) + [-1] * max(0, over) if words else None
    want = ref.plan(kept, fresh, page, max_pages, rows, held, table, free, n_free, parents[:rows] if words else None, words, target, least)
    pool = paged.PagePool(_dev(table), _dev(held), _dev(free), _dev([n_free]), page)
    for again in range(2):              # planned again from the same counts it is the same plan
        got = pool.plan(_dev(kept), _dev(fresh), rows, None if parents is None else _dev(parents[:rows]), words or None, target, least)
        for name in ("row_start", "admitted", "pages", "slots", "positions", "units", "unit_start"):
            assert getattr(got, name).cpu().tolist() == want[name], (name, again)
        assert got.n_free.item() == want["n_free"]
        if words:
            assert (got.mask.cpu().numpy().astype(np.int64) & 0xFFFFFFFF).tolist() == [[int(w) for w in r] for r in want["mask"]]
        now = pool.table.cpu().tolist()
        for b in range(B):
            n = want["pages"][b]
            assert now[b][:n] == want["table"][b][:n]
    pool.commit(got)
    # every page is held once or lies on the stack once
    seen = list(itertools.chain(*[pool.table.cpu().tolist()[b][:n] for b, n in enumerate(pool.pages.cpu().tolist())]))
    seen += pool.free.cpu().tolist()[:pool.n_free.item()]
    assert sorted(seen) == sorted(ids[:at] + ids[at:at + n_free])


@pytest.mark.gpu
def test_plan_of_many_requests_grows_shrinks_and_ends_empty():
    """2048 requests through ten steps of random growth and release; the plan matches the restatement at each and all pages come back."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(11)
    B, page, cols = 2048, 16, 12
    pool = paged.PagePool.create(9000, page, B, cols)
    kept = np.zeros(B, int)
    for step in range(10):
        fresh = rng.integers(0, 40, B) if step < 9 else np.zeros(B, int)
        kept = np.minimum(kept, cols * page - 40) if step < 9 else np.zeros(B, int)
        state = (pool.pages.cpu().tolist(), pool.table.cpu().tolist(), pool.free.cpu().tolist(), pool.n_free.item())
        rows = int(fresh.sum())
        want = ref.plan(kept.tolist(), fresh.tolist(), page, cols, rows, state[0], state[1], state[2], state[3], target=100, least=64)
        got = pool.plan(_dev(kept.tolist()), _dev(fresh.tolist()), rows, units=100, chunk=64)
        for name in ("row_start", "admitted", "pages", "slots", "positions", "units", "unit_start"):
            assert getattr(got, name).cpu().tolist() == want[name], (name, step)
        assert got.n_free.item() == want["n_free"]
        pool.commit(got)
        kept = np.where(np.array(want["admitted"]) == 1, kept + rng.integers(0, 2, B) * fresh, kept)
    assert pool.n_free.item() == 9000 and sorted(pool.free.cpu().tolist()) == list(range(9000))


@pytest.mark.gpu
@pytest.mark.parametrize("n_free", [0, 3, 4])
def test_plan_takes_no_more_pages_back_than_there_are(n_free):
    """Counts that claim 16 pages of a pool of 4: the stack ends at 4, and what grows is served from those."""
    from manual_whisper_amd import paged
    table = [[0] * 8, [1] * 8, [-1] * 8]
    pool = paged.PagePool(_dev(table), _dev([8, 8, 0]), _dev([3, 2, 2, 2]), _dev([n_free]), 16)
    got = pool.plan(_dev([0, 0, 40]), _dev([0, 0, 8]), 8, units=2, chunk=64)
    assert got.admitted.cpu().tolist() == [1, 1, 1] and got.pages.cpu().tolist() == [0, 0, 3] and got.n_free.item() == 1
    stack = ([3, 2, 2, 2][:n_free] + [0] * 8)[:4]
    assert pool.free.cpu().tolist() == stack and pool.table.cpu().tolist()[2][:3] == stack[:0:-1]
    assert got.slots.cpu().tolist() == [16 * stack[1] + 8 + i for i in range(8)]
    none = pool.plan(_dev([0, 0, 60]), _dev([0, 0, 8]), 8)
    assert none.admitted.cpu().tolist() == [1, 1, 0] and none.pages.cpu().tolist() == [0, 0, 0] and none.n_free.item() == 4


def _new_cache(rng, kind, shape, layout="head"):
    """(PagedCache, values of k, of v as float64): random contents in one of two memory orders."""
    from manual_whisper_amd import paged
    pages, heads, page, dim = shape[-4:]
    order = shape if layout == "head" else shape[:-4] + (pages, page, heads, dim)

    def put(x):
        t = torch.tensor(x, device="cuda")
        return t if layout == "head" else t.transpose(-3, -2)

    if kind == "e4m3":
        ts, values = [], []
        for _ in range(2):
            code = rng.integers(0, 256, order).astype(np.uint8)
            code[(code & 0x7F) == 0x7F] = 0x3C
            t = put(code)
            s = torch.tensor(rng.uniform(0.2, 3, shape[:-1]).astype(np.float32) / 448, device="cuda")
            ts += [t, s]
            values.append((t.view(torch.float8_e4m3fn).float().double() * s.double()[..., None]).cpu().numpy())
        return paged.PagedCache(ts[0], ts[2], ts[1], ts[3]), values[0], values[1]
    ts = [put(rng.standard_normal(order).astype(np.float32)).to(DT[kind]) for _ in range(2)]
    return paged.PagedCache(*ts), ts[0].double().cpu().numpy(), ts[1].double().cpu().numpy()


def _values(cache, name):
    x, s = getattr(cache, name), getattr(cache, name + "_scale")
    x = x.view(torch.float8_e4m3fn).float() if x.dtype == torch.uint8 else x
    return (x.double() if s is None else x.double() * s.double()[..., None]).cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rows_type", [("f16", "f16"), ("bf16", "bf16"), ("e4m3", "f16"), ("e4m3", "bf16")])
@pytest.mark.parametrize("heads,dim,page,rows,layout", [(1, 64, 16, 1, "head"), (20, 64, 64, 37, "head"), (8, 128, 32, 130, "token"), (3, 128, 16, 5, "head")])
def test_write(kind, rows_type, heads, dim, page, rows, layout):
    from manual_whisper_amd import paged
    rng = np.random.default_rng(rows)
    n_pages = rows // page + 3
    cache, k0, v0 = _new_cache(rng, kind, (n_pages, heads, page, dim), layout)
    slots = rng.permutation(n_pages * page)[:rows]
    qkv = torch.tensor(rng.standard_normal((rows, heads * 3, dim)).astype(np.float32), device="cuda").to(DT[rows_type])
    k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
    k[0, 0] = 0                                               # a row of zeros: scale 0, codes 0
    if rows > 4:
        slots[2] = -1
        slots[3] = n_pages * page + 5                         # beyond the cache: dropped
        v[1] *= 300                                           # rows of very different size
        k[4] *= 2.0 ** -12
    paged.write(cache, k, v, _dev(slots.tolist(), torch.int64))
    for name, before, x in (("k", k0, k), ("v", v0, v)):
        got, want = _values(cache, name), before.copy()
        x = x.double().cpu().numpy()
        off = np.zeros_like(want)
        for r, t in enumerate(slots):
            if 0 <= t < n_pages * page:
                want[t // page, :, t % page] = x[r]
                if kind == "e4m3":
                    scale, err = ref.e4m3_rows(x[r])
                    off[t // page, :, t % page] = err
                    have = getattr(cache, name + "_scale")[t // page, :, t % page].double().cpu().numpy()
                    assert np.abs(have - scale[:, 0]).max() <= 2.0 ** -23 * scale.max()
        assert (np.abs(got - want) <= off).all()              # 16-bit values and every other row: exactly


@pytest.mark.gpu
def test_write_of_rows_without_a_scale():
    """An infinity or a NaN: the whole e4m3 row reads back as NaN, its neighbours are untouched; a 16-bit cache keeps the bits."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(3)
    cache, k0, v0 = _new_cache(rng, "e4m3", (2, 2, 16, 64))
    k = torch.randn(3, 2, 64, device="cuda", dtype=torch.float16)
    v = torch.randn(3, 2, 64, device="cuda", dtype=torch.float16)
    k[0, 1, 5], v[1, 0, 63] = float("inf"), float("nan")
    paged.write(cache, k, v, _dev([3, 20, 31], torch.int64))
    gk, gv = _values(cache, "k"), _values(cache, "v")
    assert np.isnan(gk[0, 1, 3]).all() and np.isfinite(gk[0, 0, 3]).all() and np.isnan(gv[1, 0, 4]).all() and np.isfinite(gv[1, 1, 4]).all()
    assert np.isfinite(np.delete(gk[0, 1], 3, 0)).all() and (gk[1, :, :4] == k0[1, :, :4]).all()
    plain, _, _ = _new_cache(rng, "f16", (2, 2, 16, 64))
    paged.write(plain, k, v, _dev([3, 20, 31], torch.int64))
    assert torch.equal(plain.k[0, :, 3].view(torch.int16), k[0].view(torch.int16)) and torch.equal(plain.v[1, :, 4].view(torch.int16), v[1].view(torch.int16))


def _tree_case(rng, kept, fresh, page, spare=2):
    """Tables over shuffled pages, and ancestors' masks of random trees as truth values and words."""
    need = [-(-(k + f) // page) for k, f in zip(kept, fresh)]
    ids = rng.permutation(sum(need) + spare)
    cols, at, table = max(1, max(need)), 0, []
    for n in need:
        table.append(ids[at:at + n].tolist() + [-1] * (cols - n))
        at += n
    start = np.concatenate([[0], np.cumsum(fresh)]).tolist()
    parents = _forest(rng, fresh)
    words = max(1, -(-max(fresh + [1]) // 32))
    see = np.zeros((start[-1], words * 32), bool)
    for b in range(len(kept)):
        for i in range(fresh[b]):
            j = i
            see[start[b] + i, i] = True
            while 0 <= parents[start[b] + j] < j:
                j = parents[start[b] + j]
                see[start[b] + i, j] = True
    return table, sum(need) + spare, start, see, words


def _pack(see):
    w = (see.reshape(see.shape[0], -1, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32)
    return torch.tensor(w.view(np.int32), device="cuda")


def _units(kept, fresh, target, least):
    B = len(kept)
    p = ref.plan(kept, fresh, 16, 1 << 20, sum(fresh), [0] * B, [[]] * B, [], 0, target=0, least=64)       # row starts only
    assert p["row_start"][-1] == sum(fresh)
    up64 = lambda n: -(-n // 64) * 64      # noqa: E731
    lens = [k + f if f else 0 for k, f in zip(kept, fresh)]
    most = max(up64(-(-sum(lens) // target) if target else sum(lens)), up64(least))
    units, first = [], [0]
    for b in range(B):
        n = max(1, -(-lens[b] // most)) if fresh[b] else 0
        each = up64(-(-lens[b] // n)) if n else 0
        units += [[b, min(u * each, lens[b]), min((u + 1) * each, lens[b]), n] for u in range(n)]
        first.append(first[-1] + n)
    units += [[-1] * 4] * (B + target - len(units))
    return _dev(units), _dev(first)


def _close(got, want, size, big, vmax, kind, dim, keys, e4m3):
    """|got - want| against what the roundings allow.  u: half a step of the type.  The weights are rounded once (u each, relative to
    sum p |v|), the result once (u); scores carry dim + 8 roundings of 2^-24 relative to sum |q k| scale, twice (numerator and
    denominator), sums of up to `keys` weights and products another keys * 2^-24; fp16 weights below 2^-14 are off by up to 2^-25 of
    the largest (e4m3: of the largest times the row scales' range of 32, codes up to 448)."""
    u = torch.finfo(DT[kind]).eps / 2
    tol = (2.01 * u + 2 * (dim + 8) * 2.0 ** -24 * (1 + big) + 2 * (keys + 64) * 2.0 ** -24) * size + u * np.abs(want) * 1e-2
    if kind == "f16":
        tol = tol + keys * 2.0 ** -25 * vmax * (32 if e4m3 else 1) + 2.0 ** -25
    bad = np.abs(got - want) > tol
    assert not bad.any(), (int(bad.sum()), float((np.abs(got - want) / np.maximum(tol, 1e-30)).max()))


ATTEND = [  # kept, fresh, heads, kv heads, dim, page, target, least
    ([0], [1], 1, 1, 64, 16, 0, 64),
    ([1], [1], 4, 2, 128, 16, 0, 64),
    ([0, 5, 0], [3, 0, 1], 2, 2, 64, 16, 0, 64),
    ([63, 64, 65, 127], [1, 1, 1, 1], 3, 1, 64, 64, 0, 64),
    ([37, 120, 400, 3], [8, 8, 8, 8], 20, 20, 64, 64, 0, 64),
    ([200, 17, 0], [17, 5, 30], 8, 2, 128, 32, 0, 64),
    ([300, 70], [33, 64], 4, 4, 64, 16, 3, 64),
    ([513, 40], [64, 9], 6, 6, 128, 128, 6, 64),
    ([100, 1000], [61, 20], 8, 2, 128, 16, 9, 128),
    ([40], [130], 2, 1, 64, 32, 4, 64),
    ([2000, 5, 700, 0], [1, 1, 1, 1], 16, 2, 128, 64, 12, 64),
    ([900, 1500], [16, 3], 40, 5, 64, 256, 20, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cache_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3")])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention(case, tree, kind, cache_kind):
    from manual_whisper_amd import paged
    kept, fresh, heads, kv, dim, page, target, least = ATTEND[case]
    rng = np.random.default_rng(100 + case)
    table, n_pages, start, see, words = _tree_case(rng, kept, fresh, page)
    cache, k, v = _new_cache(rng, cache_kind, (n_pages, kv, page, dim), "token" if case % 3 == 2 else "head")
    qkv = torch.tensor(rng.standard_normal((start[-1], heads + 2, dim)).astype(np.float32), device="cuda").to(DT[kind])
    q = qkv[:, 1:1 + heads]                                   # rows of a fused buffer
    units, first = _units(kept, fresh, target, least)
    out = torch.full((start[-1] + 2, heads, dim), 7.0, dtype=DT[kind], device="cuda")
    got = paged.tree_attention(q, cache, _dev(table), _dev(kept), _dev(start), units, first, max(fresh), mask=_pack(see) if tree else None,
                               out=out[:start[-1]])
    want, size, big, vmax = ref.attention(q.double().cpu().numpy(), k, v, table, page, kept, start, see if tree else None)
    _close(got.double().cpu().numpy(), want, size, big, vmax, kind, dim, max(a + b for a, b in zip(kept, fresh)), cache_kind == "e4m3")
    assert (out[start[-1]:] == 7).all()                       # rows behind the last request
    again = paged.tree_attention(q, cache, _dev(table), _dev(kept), _dev(start), units, first, max(fresh), mask=_pack(see) if tree else None)
    assert torch.equal(again, got)                            # the same bits each time


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cache_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("fresh", [4, 21, 70])
def test_attention_of_empty_rows_and_arbitrary_masks(kind, cache_kind, fresh):
    """Masks of any bits (later nodes too); a row without any key is zero, with no kept tokens and with bits of absent nodes."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(fresh)
    kept, n, page, heads, kv, dim = [0, 70, 0], [fresh, fresh, 3], 16, 4, 2, 64
    table, n_pages, start, see, words = _tree_case(rng, kept, n, page)
    see = rng.random(see.shape) < 0.4
    see[0] = see[2] = False
    see[start[2] + 1] = False
    see[start[2] + 1, 5:] = True                              # nodes that the request does not have
    cache, k, v = _new_cache(rng, cache_kind, (n_pages, kv, page, dim))
    q = torch.randn(start[-1], heads, dim, device="cuda").to(DT[kind])
    units, first = _units(kept, n, 0, 64)
    got = paged.tree_attention(q, cache, _dev(table), _dev(kept), _dev(start), units, first, max(n), mask=_pack(see)).double().cpu().numpy()
    want, size, big, vmax = ref.attention(q.double().cpu().numpy(), k, v, table, page, kept, start, see)
    assert (got[0] == 0).all() and (got[2] == 0).all() and (got[start[2] + 1] == 0).all()
    _close(got, want, size, big, vmax, kind, dim, 70 + fresh, cache_kind == "e4m3")


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cache_kind", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("nodes,heads", [(6, 2), (20, 4), (40, 8)])
def test_attention_keeps_what_a_row_does_not_see_away(kind, cache_kind, nodes, heads):
    """Infinities and NaN in K and V of one branch, behind the last node and in pages of nobody: rows that do not see them are as
    without them, rows that do are not finite."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(nodes)
    kept, n, page, kv, dim = [21, 64], [nodes, nodes], 16, 2, 64
    table, n_pages, start, _, words = _tree_case(rng, kept, n, page)
    see = np.zeros((start[-1], words * 32), bool)
    for b in range(2):                                        # two branches under the root: odd nodes and even nodes
        for i in range(nodes):
            see[start[b] + i, 0] = True
            see[start[b] + i, 2 - i % 2:i + 1:2] = True
            see[start[b] + i, i] = True
    cache, k, v = _new_cache(rng, cache_kind, (n_pages, kv, page, dim))
    q = torch.randn(start[-1], heads, dim, device="cuda").to(DT[kind])
    units, first = _units(kept, n, 0, 64)
    args = (_dev(table), _dev(kept), _dev(start), units, first, nodes)
    clean = paged.tree_attention(q, cache, *args, mask=_pack(see))
    used = {(table[b][p // page], p % page) for b in range(2) for p in range(kept[b] + nodes)}
    bad = float("nan")
    for pg in range(n_pages):
        for o in range(page):
            if (pg, o) not in used:
                if cache_kind == "e4m3":
                    cache.k[pg, :, o], cache.v[pg, :, o] = 0x7F, 0xFF
                    cache.k_scale[pg, :, o] = cache.v_scale[pg, :, o] = bad
                else:
                    cache.k[pg, :, o], cache.v[pg, :, o] = bad, float("inf")
    same = paged.tree_attention(q, cache, *args, mask=_pack(see))
    assert torch.equal(same, clean)
    for b in range(2):                                        # node 3 (the odd branch): V infinite, K a NaN in one head
        at = kept[b] + 3
        pg, o = table[b][at // page], at % page
        if cache_kind == "e4m3":
            cache.v[pg, 0, o, 5], cache.v_scale[pg, 1, o], cache.k_scale[pg, 1, o] = 0x7F, bad, bad
        else:
            cache.v[pg, 0, o, 5], cache.v[pg, 1, o, 9], cache.k[pg, 1, o, 0] = float("inf"), bad, bad
    got = paged.tree_attention(q, cache, *args, mask=_pack(see)).double().cpu().numpy()
    clean = clean.double().cpu().numpy()
    for b in range(2):
        for i in range(nodes):
            r = start[b] + i
            if see[r, 3]:
                assert not np.isfinite(got[r, :heads // 2, 5]).any() and not np.isfinite(got[r, heads // 2:, 9]).any()
            else:
                assert np.isfinite(got[r]).all()
                # nothing of node 3: the clean result up to the roundings of the weights (two ways to form the product)
                assert np.abs(got[r] - clean[r]).max() <= 4 * torch.finfo(DT[kind]).eps * np.abs(v).max()


@pytest.mark.gpu
def test_attention_of_missing_pages_and_refused_requests():
    """Ids outside the cache count as not seen; a refused request (a unit without keys) is zero; so is one whose table is too short."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(8)
    kept, n, page = [100, 33, 50], [5, 4, 3], 16
    table, n_pages, start, see, words = _tree_case(rng, kept, n, page)
    cache, k, v = _new_cache(rng, "f16", (n_pages, 2, page, 64))
    q = torch.randn(start[-1], 4, 64, device="cuda", dtype=torch.float16)
    units, first = _units(kept, n, 0, 64)
    table[0][1], table[0][3] = -5, n_pages + 1000
    units[1, 1:3] = 0
    got = paged.tree_attention(q, cache, _dev(table), _dev(kept), _dev(start), units, first, 5, mask=_pack(see)).double().cpu().numpy()
    want, size, big, vmax = ref.attention(q.double().cpu().numpy(), k, v, table, page, kept, start, see)
    keep = [r for r in range(start[-1]) if not start[1] <= r < start[2]]
    _close(got[keep], want[keep], size[keep], big, vmax[keep], "f16", 64, 110, False)
    assert (got[start[1]:start[2]] == 0).all()
    short = _dev([r[:2] for r in table])                      # 32 positions only
    got = paged.tree_attention(q, cache, short, _dev(kept), _dev(start), units, first, 5, mask=_pack(see)).double().cpu().numpy()
    want, size, big, vmax = ref.attention(q.double().cpu().numpy(), k, v, [r[:2] for r in table], page, kept, start, see)
    _close(got[keep], want[keep], size[keep], big, vmax[keep], "f16", 64, 110, False)


@pytest.mark.gpu
def test_attention_with_large_scores_and_a_scale():
    """Scores in the thousands, one key far above the rest, a scale of the caller's, and equal keys."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(9)
    kept, n, page = [150, 150], [6, 6], 32
    table, n_pages, start, see, words = _tree_case(rng, kept, n, page)
    cache, k, v = _new_cache(rng, "bf16", (n_pages, 1, page, 64))
    q = (30 * torch.randn(start[-1], 2, 64, device="cuda")).to(torch.bfloat16)
    units, first = _units(kept, n, 0, 64)
    for scale in (None, 3.0, 1e-6):
        got = paged.tree_attention(q, cache, _dev(table), _dev(kept), _dev(start), units, first, 6, mask=_pack(see), scale=scale).double().cpu().numpy()
        want, size, big, vmax = ref.attention(q.double().cpu().numpy(), k, v, table, page, kept, start, see, scale)
        _close(got, want, size, big, vmax, "bf16", 64, 160, False)


@pytest.mark.gpu
def test_attention_beyond_32_bits_of_offset():
    """A cache of more than 2^32 elements: rows in its last pages are found."""
    from manual_whisper_amd import paged
    n_pages, heads, page, dim = 36000, 2, 512, 128            # 4.7e9 elements, 9.4 GB each of k and v
    k = torch.zeros(n_pages, heads, page, dim, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    cache = paged.PagedCache(k, v)
    table = _dev([[n_pages - 1, 3], [n_pages - 2, 33333]])
    kept, start = [600, 90], [0, 2, 3]
    rows_k = torch.randn(693, heads, dim, device="cuda", dtype=torch.float16)
    rows_v = torch.randn(693, heads, dim, device="cuda", dtype=torch.float16)
    at = [(0, p) for p in range(602)] + [(1, p) for p in range(91)]
    slots = torch.tensor([int(table[b, p // page]) * page + p % page for b, p in at], device="cuda")
    paged.write(cache, rows_k, rows_v, slots)
    q = torch.randn(3, 4, dim, device="cuda", dtype=torch.float16)
    units, first = _units(kept, [2, 1], 3, 64)
    got = paged.tree_attention(q, cache, table, _dev(kept), _dev(start), units, first, 2).double().cpu().numpy()
    small = {int(p): i for i, p in enumerate(table.flatten().tolist())}
    kk, vv = (x[table.flatten().long()].double().cpu().numpy() for x in (k, v))
    want, size, big, vmax = ref.attention(q.double().cpu().numpy(), kk, vv, [[small[int(p)] for p in r] for r in table.tolist()], page, kept, start)
    _close(got, want, size, big, vmax, "f16", dim, 602, False)
    paged.compact(cache, table, _dev([600, 89]), _dev([[1], [1]]), _dev([1, 1]))
    assert torch.equal(k[3, :, 600 - 512], rows_k[601]) and torch.equal(k[n_pages - 2, :, 89], rows_k[692])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("nodes,vocab,stride", [([1], 1, 1), ([1, 0, 3], 7, 9), ([8] * 5, 1000, 1001), ([33, 2, 70], 51866, 51866), ([5, 9], 128001, 128001)])
def test_accept(dtype, nodes, vocab, stride):
    from manual_whisper_amd import paged
    rng = np.random.default_rng(vocab)
    start = np.concatenate([[0], np.cumsum(nodes)]).tolist()
    rows, B = start[-1], len(nodes)
    store = torch.tensor(np.round(rng.standard_normal((rows, stride)) * 8).astype(np.float32) / 8, device="cuda").to(dtype)      # many ties
    logits = store[:, :vocab]
    suppress = (rng.random(vocab) < 0.3).astype(np.uint8)
    suppress[0] = 1
    parents = _forest(rng, nodes, faults=True)
    depth = max(nodes)
    host = logits.float().cpu().numpy()
    for sup in (None, suppress):
        best = ref.accept(host, [0] * rows, parents, start, depth, sup)[0]
        tokens = [int(best[start[b] + parents[r]]) if 0 <= parents[r] < r - start[b] and rng.random() < 0.8 else int(rng.integers(0, vocab))
                  for b in range(B) for r in range(start[b], start[b + 1])]
        for d in {depth, max(1, depth // 2), depth + 3}:
            want = ref.accept(host, tokens, parents, start, d, sup)
            got = paged.accept(logits, _dev(tokens), _dev(parents), _dev(start), d, None if sup is None else _dev(sup.tolist(), torch.uint8))
            for g, w in zip(got, want):
                assert g.cpu().tolist() == w.tolist()


@pytest.mark.gpu
def test_accept_of_rows_without_a_choice():
    """NaN, infinities, a row of lowest values, a row all of whose ids are suppressed; rows behind the last request stay."""
    from manual_whisper_amd import paged
    x = torch.zeros(6, 20000, device="cuda")
    x[0, 7], x[0, 3] = float("nan"), 1.0
    x[1] = float("nan")
    x[2] = float("-inf")
    x[2, 9000] = torch.finfo(torch.float32).min
    x[3, 15000] = x[3, 16000] = float("inf")
    x[4] = float("-inf")
    got = paged.accept(x, _dev([0] * 6), _dev([-1, 0, 0, 0, 0, 0]), _dev([0, 5]), 8)
    assert got[0][:5].tolist() == [3, 0, 9000, 15000, 0] and got[1].tolist() == [[0] + [-1] * 7] and got[2].tolist() == [1]
    assert paged.accept(x, _dev([0] * 6), _dev([-1] * 6), _dev([0, 5]), 8, torch.ones(20000, dtype=torch.uint8, device="cuda"))[0][:5].tolist() == [0] * 5


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("layers,heads,dim,page,layout", [(1, 1, 64, 16, "head"), (3, 5, 64, 32, "token"), (2, 8, 128, 16, "head"), (None, 2, 128, 64, "head")])
def test_compact(kind, layers, heads, dim, page, layout):
    from manual_whisper_amd import paged
    rng = np.random.default_rng(dim + page)
    kept, nodes = [0, 17, 40, 3, 9], [1, 30, 300, 8, 5]
    table, n_pages, start, _, _ = _tree_case(rng, kept, nodes, page)
    depth = max(nodes)
    path = [sorted([0] + rng.choice(np.arange(1, n), size=max(0, n // 2), replace=False).tolist()) if n > 1 else [0] for n in nodes]
    count = [len(p) for p in path]
    path[3], count[3] = [0, 0, 5, 2, 7], 5                    # an entry below its index is skipped, as are the ones behind `count`
    path[4], count[4] = [0, 1, 2, 4], 3
    path = [p + [-1] * (depth - len(p)) for p in path]
    shape = (n_pages, heads, page, dim) if layers is None else (layers, n_pages, heads, page, dim)
    cache, k, v = _new_cache(rng, kind, shape, layout)
    paged.compact(cache, _dev(table), _dev(kept), _dev(path), _dev(count))
    for name, x in (("k", k), ("v", v)):
        want = ref.compact(x[None] if layers is None else x, table, page, kept, path, count)
        assert (_values(cache, name) == (want[0] if layers is None else want)).all()
    table[1][1] = -1                                          # a page that does not exist: its rows stay
    before = _values(cache, "k")
    paged.compact(cache, _dev(table), _dev(kept), _dev(path), _dev(count))
    want = ref.compact(before[None] if layers is None else before, table, page, kept, path, count)
    assert (_values(cache, "k") == (want[0] if layers is None else want)).all()


@pytest.mark.gpu
def test_strides_of_dimensions_of_one_and_of_shared_rows():
    """The stride of a dimension of one says nothing and may be anything; a table whose rows share memory is refused."""
    from manual_whisper_amd import paged
    from manual_whisper_amd.engine import EngineError
    mem = [torch.zeros(3 * 64 * 64, device="cuda", dtype=torch.float16) for _ in range(4)]
    plain = paged.PagedCache(mem[0].view(3, 1, 64, 64), mem[1].view(3, 1, 64, 64))
    odd = paged.PagedCache(mem[2].as_strided((3, 1, 64, 64), (4096, 3, 64, 1)), mem[3].as_strided((3, 1, 64, 64), (4096, 0, 64, 1)))
    rows = torch.randn(1, 64, device="cuda", dtype=torch.float16)
    slots = torch.tensor([70], device="cuda")
    paged.write(plain, rows.view(1, 1, 64), rows.view(1, 1, 64), slots)
    paged.write(odd, rows.as_strided((1, 1, 64), (7, 5, 1)), rows.as_strided((1, 1, 64), (1, 3, 1)), slots)
    assert mem[0].any() and torch.equal(mem[0], mem[2]) and torch.equal(mem[1], mem[3])
    table, kept, path = _dev([[1, 0, 2]]), _dev([2]), _dev([[0, 4]])
    for cache in (plain, odd):
        paged.compact(cache, table.as_strided((1, 3), (1, 1)), kept, path, _dev([2]))
    assert mem[0].view(3, 64, 64)[1, 3].any() and torch.equal(mem[0], mem[2])
    out = [paged.tree_attention(q, cache, table, kept, _dev([0, 1]), _dev([[0, 0, 3, 1]]), _dev([0, 1]), 1)
           for q, cache in ((rows.view(1, 1, 64), plain), (rows.as_strided((1, 1, 64), (9, 9, 1)), odd))]
    assert torch.equal(*out)
    for fault in (lambda: paged.compact(plain, table.expand(2, 3), _dev([2, 2]), _dev([[0, 4]] * 2), _dev([2, 2])),
                  lambda: paged.PagePool(table.expand(2, 3), _dev([1, 1]), _dev([0]), _dev([0]), 64)):
        with pytest.raises(EngineError):
            fault()


def _dense_step(q, k, v, ctx, see):
    """One request's rows in 64 bits over plain arrays."""
    kk, vv = np.concatenate([ctx[0], k]), np.concatenate([ctx[1], v])
    out = np.zeros(q.shape)
    for i in range(q.shape[0]):
        sees = np.concatenate([np.ones(len(ctx[0]), bool), see[i][:len(k)]])
        for h in range(q.shape[1]):
            s = kk[sees][:, h // (q.shape[1] // kk.shape[1])] @ q[i, h] / np.sqrt(q.shape[2])
            p = np.exp(s - s.max())
            out[i, h] = p / p.sum() @ vv[sees][:, h // (q.shape[1] // kk.shape[1])]
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_steps_together(kind):
    """Five steps of three requests over two layers, as a program runs them: plan, write, attend, accept, compact, commit.  Every
    step's attention is that of dense caches kept beside it, from which rejected branches are dropped."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(21)
    B, L, H, KV, D, page, vocab = 3, 2, 4, 2, 64, 16, 500
    pool = paged.PagePool.create(40, page, B, 12)
    cache = paged.PagedCache.empty(L, 40, KV, page, D, DT[kind])
    kept = [0] * B
    dense = [[(np.zeros((0, KV, D)), np.zeros((0, KV, D))) for _ in range(B)] for _ in range(L)]
    dropped = 0
    for step in range(5):
        nodes = [int(n) for n in rng.integers(1, 40 if step else 60, B)]
        parents = _forest(rng, nodes)
        rows = sum(nodes) + 2
        up = _dev(parents + [-1, -1])
        plan = pool.plan(_dev(kept), _dev(nodes), rows, up, 2, units=4, chunk=64)
        assert plan.admitted.tolist() == [1] * B
        start = plan.row_start.tolist()
        see = ((plan.mask.cpu().numpy()[:, :, None] >> np.arange(32)) & 1).reshape(rows, -1).astype(bool)
        fresh_kv = []
        for layer in range(L):
            qkv = torch.tensor(rng.standard_normal((rows, H + 2 * KV, D)).astype(np.float32), device="cuda").to(DT[kind])
            one = cache.layer(layer)
            paged.write(one, qkv[:, H:H + KV], qkv[:, H + KV:], plan.slots)
            got = paged.tree_attention(qkv[:, :H], one, pool.table, _dev(kept), plan.row_start, plan.units, plan.unit_start, max(nodes), mask=plan.mask)
            x = qkv.double().cpu().numpy()
            for b in range(B):
                part = x[start[b]:start[b + 1]]
                want = _dense_step(part[:, :H], part[:, H:H + KV], part[:, H + KV:], dense[layer][b], see[start[b]:start[b + 1]])
                # 2 u of values up to 5, and the scores' part
                assert np.abs(got[start[b]:start[b + 1]].double().cpu().numpy() - want).max() <= (2.01 * torch.finfo(DT[kind]).eps / 2 + 1e-4) * 5
            fresh_kv.append(x)
        logits = torch.tensor(rng.standard_normal((rows, vocab)).astype(np.float32), device="cuda")
        best = logits.argmax(1).tolist()
        tokens = [best[start[b] + parents[r]] if parents[r] >= 0 and rng.random() < 0.7 else 0 for b in range(B) for r in range(start[b], start[b + 1])]
        _, path, count, ids = paged.accept(logits, _dev(tokens + [0, 0]), up, plan.row_start, max(nodes))
        want = ref.accept(logits.cpu().numpy(), tokens, parents, start, max(nodes))
        assert path.tolist() == want[1].tolist() and count.tolist() == want[2].tolist() and ids.tolist() == want[3].tolist()
        paged.compact(cache, pool.table, _dev(kept), path, count)
        pool.commit(plan)
        for b in range(B):
            taken = [start[b] + i for i in path[b].tolist() if i >= 0]
            dropped += nodes[b] - len(taken)
            for layer in range(L):
                k, v = dense[layer][b]
                dense[layer][b] = (np.concatenate([k, fresh_kv[layer][taken, H:H + KV]]), np.concatenate([v, fresh_kv[layer][taken, H + KV:]]))
            kept[b] += len(taken)
    assert dropped > 20
    end = pool.plan(_dev([0] * B), _dev([0] * B), 0)
    pool.commit(end)
    assert pool.n_free.item() == 40


@pytest.mark.gpu
def test_calls_on_other_streams_and_in_graphs():
    """Two captured steps on streams of their own, replayed between eager calls: every replay equals the eager result."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(31)
    kept, fresh, page = [700, 90, 333], [9, 4, 12], 16
    table, n_pages, start, see, words = _tree_case(rng, kept, fresh, page)
    cache, _, _ = _new_cache(rng, "bf16", (n_pages, 2, page, 128))
    units, first = _units(kept, fresh, 16, 64)
    fixed = (_dev(table), _dev(kept), _dev(start), units, first, 12)
    mask = _pack(see)
    pool = paged.PagePool(_dev(table), _dev([-(-k // page) for k in kept]), _dev([-1] * n_pages), _dev([0]), page)
    pool.pages.copy_(_dev([-(-(k + f) // page) for k, f in zip(kept, fresh)]))
    parents = _dev(_forest(rng, fresh))
    qs = [torch.randn(25, 8, 128, device="cuda").to(torch.bfloat16) for _ in range(3)]
    logits = torch.randn(25, 5000, device="cuda")

    def step(q):
        plan = pool.plan(fixed[1], _dev_fresh, 25, parents, 1, units=16, chunk=64)
        out = paged.tree_attention(q, cache, pool.table, fixed[1], plan.row_start, plan.units, plan.unit_start, 12, mask=plan.mask)
        more = paged.tree_attention(q, cache, *fixed, mask=mask)
        return (out, more) + paged.accept(logits, tokens, parents, plan.row_start, 12)

    _dev_fresh = _dev(fresh)
    tokens = logits.argmax(1).to(torch.int32).roll(1)
    eager = [[t.clone() for t in step(q)] for q in qs]
    graphs, outs, ins = [], [], []
    for k in range(2):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        q = qs[k].clone()
        with torch.cuda.stream(s):
            step(q)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                o = step(q)
        graphs.append(g), outs.append(o), ins.append(q)
    torch.cuda.synchronize()
    for turn in range(3):
        for k in range(2):
            ins[k].copy_(qs[(turn + k) % 3])
        both = [torch.cuda.Stream(), torch.cuda.Stream()]
        for k in range(2):                                    # two replays that may overlap
            both[k].wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(both[k]):
                graphs[k].replay()
        now = step(qs[turn])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(now, eager[turn]))
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], eager[(turn + k) % 3])), (turn, k)


KEPT_POISON = [  # kept, nodes, heads, kv heads, page, target of the cut, table columns (None: all), poisoned kept positions of request 0
    (70, 4, 4, 2, 16, 0, None, (3, 64, 66, 69)),              # a tile that kept tokens share with the nodes, and the tile before it
    (70, 1, 4, 2, 64, 0, None, (65,)),
    (63, 9, 4, 2, 32, 0, None, (0, 62)),
    (200, 20, 8, 2, 16, 0, None, (192, 199)),
    (130, 40, 4, 2, 16, 0, None, (5, 128, 129)),
    (700, 7, 4, 2, 16, 6, None, (130, 640, 699)),             # cut into pieces
    (90, 3, 4, 2, 16, 0, 5, (64, 70, 79)),                    # the table ends before the kept tokens do
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cache_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("case", range(len(KEPT_POISON)))
def test_infinities_and_nan_of_kept_tokens_reach_every_row(case, tree, kind, cache_kind):
    """All rows see every kept token: a value of V there that is no finite number leaves none of the request's results at its head and
    dimension finite, wherever the token lies in a tile; every other result keeps its bits."""
    from manual_whisper_amd import paged
    kept0, nodes, heads, kv, page, target, columns, places = KEPT_POISON[case]
    rng = np.random.default_rng(case)
    kept, n, dim = [kept0, 17], [nodes, min(nodes, 3)], 64
    table, n_pages, start, see, words = _tree_case(rng, kept, n, page)
    cache, _, _ = _new_cache(rng, cache_kind, (n_pages, kv, page, dim))
    q = torch.randn(start[-1], heads, dim, device="cuda").to(DT[kind])
    units, first = _units(kept, n, target, 64)
    dev_table = _dev([r[:columns] for r in table] if columns else table)

    def attend():
        return paged.tree_attention(q, cache, dev_table, _dev(kept), _dev(start), units, first, nodes, mask=_pack(see) if tree else None)

    clean = attend()
    for i, place in enumerate(places):
        pg, o = table[0][place // page], place % page
        bads = [0x7F, 0xFF] if cache_kind == "e4m3" else [float("inf"), float("nan"), float("-inf")]
        for bad in bads:
            d, g = (7 * i + 3) % dim, i % kv
            before = cache.v[pg, g, o, d].clone()
            cache.v[pg, g, o, d] = bad
            got = attend()
            cache.v[pg, g, o, d] = before
            hit = torch.zeros_like(got, dtype=torch.bool)
            hit[:start[1], g * (heads // kv):(g + 1) * (heads // kv), d] = True
            assert not torch.isfinite(got[hit]).any(), (place, bad)
            assert torch.equal(got[~hit], clean[~hit]), (place, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("nodes,heads", [(6, 2), (20, 4), (40, 8)])
@pytest.mark.parametrize("target", [0, 4])
def test_row_scales_of_nodes_that_a_row_does_not_see_stay_away(nodes, heads, target, kind):
    """e4m3: a node of one branch whose V has a row scale far above the others' (or an infinite one) leaves the bits of the rows that
    do not see it; those that see a finite one are right."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(nodes)
    kept, n, page, kv, dim = [21, 164], [nodes, nodes], 16, 2, 64
    table, n_pages, start, _, words = _tree_case(rng, kept, n, page)
    see = np.zeros((start[-1], words * 32), bool)
    for b in range(2):                                        # two branches under the root: odd nodes and even nodes
        for i in range(nodes):
            see[start[b] + i, 0] = True
            see[start[b] + i, 2 - i % 2:i + 1:2] = True
            see[start[b] + i, i] = True
    cache, _, _ = _new_cache(rng, "e4m3", (n_pages, kv, page, dim))
    q = torch.randn(start[-1], heads, dim, device="cuda").to(DT[kind])
    units, first = _units(kept, n, target, 64)
    args = (_dev(table), _dev(kept), _dev(start), units, first, nodes)
    clean = paged.tree_attention(q, cache, *args, mask=_pack(see))
    sees = torch.tensor(see[:, 3], device="cuda")
    ordinary = float(cache.v_scale.max())
    for factor in (2.0 ** 7, 2.0 ** 14, 2.0 ** 25, 2.0 ** 100, float("inf")):
        for b in range(2):
            at = kept[b] + 3
            cache.v_scale[table[b][at // page], :, at % page] = ordinary * factor
        got = paged.tree_attention(q, cache, *args, mask=_pack(see))
        assert torch.equal(got[~sees], clean[~sees]), factor
        if factor <= 2.0 ** 14 and kind == "bf16":            # (fp16 results may be infinite)
            want, size, big, _ = ref.attention(q.double().cpu().numpy(), _values(cache, "k"), _values(cache, "v"), table, page, kept, start, see)
            # weights and results rounded once each (u); scores and sums as in _close
            u, keys = torch.finfo(DT[kind]).eps / 2, max(kept) + nodes
            tol = (2.01 * u + 2 * (dim + 8) * 2.0 ** -24 * (1 + big) + 2 * (keys + 64) * 2.0 ** -24) * size + u * np.abs(want) * 1e-2
            assert (np.abs(got.double().cpu().numpy() - want) <= tol).all(), factor


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cache_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("nats", [12, 16, 18])
@pytest.mark.parametrize("nodes,heads", [(2, 2), (20, 2), (45, 2)])
def test_small_weights_beside_a_dominant_key(nodes, heads, nats, kind, cache_kind):
    """A long cache whose first token draws nearly all of the attention and has a V of zeros, every other token the same small weight:
    the result is what the small weights add up to."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(nats)
    kept, page, dim = 20000, 64, 64
    n_pages = -(-(kept + nodes) // page)
    k = np.zeros((n_pages, 1, page, dim), np.float32)
    v = rng.uniform(0.5, 1.5, k.shape).astype(np.float32)
    k[0, 0, 0] = 1.0
    v[0, 0, 0] = 0
    q = torch.full((nodes, heads, dim), 0.25, dtype=DT[kind], device="cuda")
    scale = nats / (dim * 0.25)                               # scores: `nats` of the first token, zero of the others
    if cache_kind == "e4m3":
        one = torch.ones(k.shape[:-1], dtype=torch.float32, device="cuda")
        cache = paged.PagedCache(*(torch.tensor(x, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8) for x in (k, v)), one, one.clone())
    else:
        cache = paged.PagedCache(*(torch.tensor(x, device="cuda").to(DT[kind]) for x in (k, v)))
    table, start = [rng.permutation(n_pages).tolist()], [0, nodes]
    table[0].remove(0)
    table[0].insert(0, 0)                                     # page 0 holds the first token
    units, first = _units([kept], [nodes], 0, 64)
    got = paged.tree_attention(q, cache, _dev(table), _dev([kept]), _dev(start), units, first, nodes, scale=scale).double().cpu().numpy()
    kk, vv = _values(cache, "k")[table[0], 0].reshape(-1, dim), _values(cache, "v")[table[0], 0].reshape(-1, dim)
    s = kk @ np.full(dim, 0.25) * scale
    u, tiles = torch.finfo(DT[kind]).eps / 2, -(-(kept + nodes) // 64)
    for i in range(nodes):
        p = np.exp(s[:kept + i + 1] - s.max())
        want = p @ vv[:kept + i + 1] / p.sum()
        # the weights are rounded once, the result once (u each); the score of the first token, 18 log2 e = 26, carries 2 roundings of
        # 2^-24 and so does the exponent; up to 65 roundings a tile on the way of a value into its sum; fp16 weights below 2^-14 are off
        # by 2^-25 where the largest is 2^10 at least (e4m3: times V's scale relative to a power of two, at most 2 above it)
        tol = (2.01 * u + 4 * 26 * 2.0 ** -24 + 2 * 65 * tiles * 2.0 ** -24) * want
        if kind == "f16":
            tol = tol + (kept + nodes) * 2.0 ** -35 * (2 if cache_kind == "e4m3" else 1) * 1.5 + 2.0 ** -25
        assert (np.abs(got[i] - want) <= tol).all(), (i, float((np.abs(got[i] - want) / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("fresh", [3, 20])
def test_cut_requests_among_idle_ones_without_a_workspace(fresh):
    """No more units than requests, and still one request in several pieces (the others are idle): it is attended to as a whole, and a
    workspace that the call does not ask for is not written."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(fresh)
    kept, n, page, heads, kv, dim = [10, 700, 0, 90], [0, fresh, 0, 0], 16, 4, 2, 64
    table, n_pages, start, see, words = _tree_case(rng, kept, n, page)
    cache, k, v = _new_cache(rng, "f16", (n_pages, kv, page, dim))
    q = torch.randn(fresh, heads, dim, device="cuda", dtype=torch.float16)
    want, size, big, vmax = ref.attention(q.double().cpu().numpy(), k, v, table, page, kept, start, see)
    dev = [_dev(table), _dev(kept), _dev(start)]
    mask, c = _pack(see), cache
    for pieces in (2, 3, 4):
        units, first = _units(kept, n, pieces, 64)
        assert first.tolist() == [0, 0, pieces, pieces, pieces]
        units = units[:pieces].contiguous()
        got = paged.tree_attention(q, cache, *dev, units, first, fresh, mask=mask)
        _close(got.double().cpu().numpy(), want, size, big, vmax, "f16", dim, 700 + fresh, False)
        guard, out = torch.full((1 << 20,), 7.0, device="cuda"), torch.zeros_like(q)
        one = _lib.PagedCache(c.k.data_ptr(), c.v.data_ptr(), None, None, *c.k.stride()[:3], n_pages, page, kv, dim, 1)
        a = _lib.TreeArgs(one, q.data_ptr(), heads * dim, dim, out.data_ptr(), heads * dim, dim, 1, heads, fresh, 4, fresh, dev[0].data_ptr(),
                          dev[0].shape[1], dev[0].shape[1], dev[1].data_ptr(), dev[2].data_ptr(), units.data_ptr(), first.data_ptr(), pieces,
                          mask.data_ptr(), words, dim ** -0.5, guard.data_ptr(), 16)
        assert _lib.load().mw_tree_attention_workspace(C.byref(a)) == 0
        assert _lib.load().mw_tree_attention(C.byref(a), 0, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out, got) and (guard == 7).all()


def _hip():
    """The HIP runtime that the library and torch run on."""
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    return C.CDLL(path)


@pytest.mark.gpu
def test_an_error_that_somebody_else_left_is_not_the_calls():
    """The runtime keeps a failed call's error until somebody asks: a call that follows neither fails for it nor takes it away."""
    from manual_whisper_amd import paged
    hip = _hip()
    rng = np.random.default_rng(4)
    cache, _, _ = _new_cache(rng, "f16", (4, 2, 16, 64))
    rows = torch.randn(3, 2, 64, device="cuda", dtype=torch.float16)
    slots = _dev([5, 17, 40], torch.int64)
    table, kept, start = _dev([[0, 1, 2, 3]]), _dev([41]), _dev([0, 1])
    units, first, one = _dev([[0, 0, 42, 1]]), _dev([0, 1]), _dev([1])
    pool = paged.PagePool.create(4, 16, 1, 4)
    logits, zero = torch.randn(1, 50, device="cuda"), _dev([0])
    calls = [lambda: paged.write(cache, rows, rows, slots), lambda: pool.plan(kept, one, 1),
             lambda: paged.tree_attention(rows[:1], cache, table, kept, start, units, first, 1),
             lambda: paged.accept(logits, zero, zero, start, 1), lambda: paged.compact(cache, table, kept, _dev_path, one)]
    _dev_path = _dev([[0]])
    for call in calls:                                        # (torch's allocator has what the calls need)
        call()
    torch.cuda.synchronize()
    for call in calls:
        hip.hipGetLastError()
        assert hip.hipSetDevice(4096) != 0                    # no such device
        left = hip.hipPeekAtLastError()
        try:
            call()
        finally:
            still = hip.hipGetLastError()
        assert still == left
    torch.cuda.synchronize()
    assert torch.equal(cache.k[1, :, 1], rows[1])


def test_rows_that_require_gradients():
    """Refused where a gradient would be lost, backward or forward, and taken as values under no_grad."""
    from torch.autograd import forward_ad
    from manual_whisper_amd import paged
    from manual_whisper_amd.engine import EngineError
    x = torch.zeros(2, 3, 64)
    leaf = torch.zeros(2, 3, 64, requires_grad=True)
    assert paged._rows3(x, "q", -1)[1:] == (192, 64)
    for t in (leaf, leaf * 2):
        with pytest.raises(EngineError, match="gradient"):
            paged._rows3(t, "q", -1)
        with torch.no_grad():
            assert paged._rows3(t, "q", -1)[1:] == (192, 64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert paged._rows3(x, "q", -1)[1:] == (192, 64)
        for t in (dual, dual * 2):
            with pytest.raises(EngineError, match="tangent"):
                paged._rows3(t, "q", -1)
            with torch.no_grad(), pytest.raises(EngineError, match="tangent"):       # no_grad leaves tangents as they are
                paged._rows3(t, "q", -1)


@pytest.mark.gpu
def test_parameters_are_taken_under_no_grad():
    from manual_whisper_amd import paged
    from manual_whisper_amd.engine import EngineError
    cache = paged.PagedCache.empty(1, 4, 2, 16, 64).layer(0)
    rows = torch.randn(3, 2, 64, device="cuda", dtype=torch.float16)
    leaf, slots = rows.clone().requires_grad_(), _dev([5, 17, 40], torch.int64)
    args = (_dev([[0, 1, 2, 3]]), _dev([38]), _dev([0, 3]), _dev([[0, 0, 41, 1]]), _dev([0, 1]), 3)
    calls = [lambda t: paged.write(cache, t, t, slots), lambda t: paged.tree_attention(t, cache, *args),
             lambda t: paged.accept(t.view(3, 128), _dev([0] * 3), _dev([-1, 0, 1]), _dev([0, 3]), 3)]
    for call in calls:
        with pytest.raises(EngineError):
            call(leaf)
        with torch.no_grad():
            got, want = call(leaf), call(rows)
        assert got is None or all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(cache.k[2, :, 8], rows[2]) and torch.equal(cache.v[0, :, 5], rows[0])


@pytest.mark.parametrize("rows,row,head,shared", [(8, 0, 64, True), (8, 1280, 0, True), (8, 64, 64, True), (8, 1216, 64, True), (8, 60, 8000, True),
                                                  (8, 1280, 32, True), (8, 1280, -64, False), (8, 64, 512, False), (8, 64, 448, True), (1, 0, 64, False)])
def test_rows_of_the_result_that_share_memory_are_refused(rows, row, head, shared):
    """20 heads of 64: rows side by side, heads side by side, or neither (what passes this check meets the next one: units)."""
    text = _refused(_lib.load().mw_tree_attention(C.byref(_tree_args(rows=rows, out_row_stride=row, out_head_stride=head, units=BAD + 8)), 0, None),
                    "mw_tree_attention")
    assert ("overlap" in text) == shared and ("units" in text) != shared


@pytest.mark.gpu
@pytest.mark.parametrize("fresh,target", [(3, 0), (3, 6), (40, 0), (40, 6)])
def test_results_in_place_of_the_queries(fresh, target):
    """`out` may be q itself (whole requests and cut ones), and not a tensor whose rows share memory."""
    from manual_whisper_amd import paged
    from manual_whisper_amd.engine import EngineError
    rng = np.random.default_rng(fresh)
    kept, n, page, heads, kv, dim = [300, 70], [fresh, 2], 16, 8, 2, 64
    table, n_pages, start, see, words = _tree_case(rng, kept, n, page)
    cache, _, _ = _new_cache(rng, "bf16", (n_pages, kv, page, dim))
    q = torch.randn(start[-1], heads, dim, device="cuda").to(torch.bfloat16)
    args = (cache, _dev(table), _dev(kept), _dev(start), *_units(kept, n, target, 64), fresh)
    want = paged.tree_attention(q, *args, mask=_pack(see))
    with pytest.raises(EngineError, match="overlap"):
        paged.tree_attention(q, *args, mask=_pack(see), out=q[:1].clone().expand_as(q))
    assert paged.tree_attention(q, *args, mask=_pack(see), out=q) is q and torch.equal(q, want)


def test_the_stride_between_layers_says_nothing_of_a_single_one():
    """K and V of one layer out of caches of different depth: taken as far as the check of the device."""
    from manual_whisper_amd import paged
    from manual_whisper_amd.engine import EngineError
    k, v = torch.zeros(1, 3, 2, 16, 64, dtype=torch.float16), torch.zeros(3, 2, 16, 64, dtype=torch.float16).as_strided((1, 3, 2, 16, 64), (8, 2048, 1024, 64, 1))
    with pytest.raises(EngineError, match="on a GPU"):
        paged.PagedCache(k, v)
    with pytest.raises(EngineError, match="layout"):
        paged.PagedCache(k, torch.zeros(1, 2, 3, 16, 64, dtype=torch.float16).transpose(1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cache_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3"), ("bf16", "e4m3")])
@pytest.mark.parametrize("nodes,heads,target", [(6, 2, 0), (20, 4, 0), (40, 8, 0), (40, 8, 6)])
def test_what_a_row_does_not_see_leaves_its_bits(nodes, heads, target, kind, cache_kind):
    """K and V of a node of one branch, ordinary, large, infinite or NaN: the rows of the other branch keep their bits."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(nodes)
    kept, n, page, kv, dim = [21, 300], [nodes, nodes], 16, 2, 64
    table, n_pages, start, _, words = _tree_case(rng, kept, n, page)
    see = np.zeros((start[-1], words * 32), bool)
    for b in range(2):                                        # two branches under the root: odd nodes and even nodes
        for i in range(nodes):
            see[start[b] + i, 0] = True
            see[start[b] + i, 2 - i % 2:i + 1:2] = True
            see[start[b] + i, i] = True
    cache, _, _ = _new_cache(rng, cache_kind, (n_pages, kv, page, dim))
    q = torch.randn(start[-1], heads, dim, device="cuda").to(DT[kind])
    args = (_dev(table), _dev(kept), _dev(start), *_units(kept, n, target, 64), nodes)
    clean = paged.tree_attention(q, cache, *args, mask=_pack(see))
    sees = torch.tensor(see[:, 3], device="cuda")
    at = [(table[b][(kept[b] + 3) // page], (kept[b] + 3) % page) for b in range(2)]
    e4m3 = cache_kind == "e4m3"
    for value in (0x7E, 0x08, 0xFF) if e4m3 else (-3.0, 1000.0, 60000.0, float("inf"), float("nan")):
        for scale in (1.0, 1e4, float("inf"), float("nan")) if e4m3 else (None,):
            for pg, o in at:
                cache.k[pg, :, o], cache.v[pg, :, o] = value, value
                cache.k[pg, :, o, 1::2] = 0                   # scores of either sign and size
                if e4m3:
                    cache.k_scale[pg, :, o], cache.v_scale[pg, :, o] = scale, scale
            got = paged.tree_attention(q, cache, *args, mask=_pack(see))
            assert torch.equal(got[~sees], clean[~sees]), (value, scale)
            assert not torch.equal(got[sees], clean[sees])


@pytest.mark.gpu
@pytest.mark.parametrize("kind,cache_kind", [("f16", "f16"), ("bf16", "bf16"), ("f16", "e4m3")])
@pytest.mark.parametrize("kept,fresh,target", [([0], [1100], 0), ([0], [1100], 9), ([0, 900, 40, 3], [700, 1, 9, 0], 0), ([513, 2500, 40, 3], [700, 1, 9, 1], 12)],
                         ids=["prompt", "prompt cut", "mixed", "mixed cut"])
def test_attention_of_prompts_and_of_mixed_batches(kept, fresh, target, kind, cache_kind):
    """Chains of many hundred rows, alone and among single rows and short chains."""
    from manual_whisper_amd import paged
    rng = np.random.default_rng(len(kept) + target)
    page, heads, kv, dim = 32, 4, 2, 64
    table, n_pages, start, _, _ = _tree_case(rng, kept, fresh, page)
    cache, k, v = _new_cache(rng, cache_kind, (n_pages, kv, page, dim))
    q = torch.randn(start[-1], heads, dim, device="cuda").to(DT[kind])
    got = paged.tree_attention(q, cache, _dev(table), _dev(kept), _dev(start), *_units(kept, fresh, target, 64), max(fresh))
    want, size, big, vmax = ref.attention(q.double().cpu().numpy(), k, v, table, page, kept, start)
    _close(got.double().cpu().numpy(), want, size, big, vmax, kind, dim, max(a + b for a, b in zip(kept, fresh)), cache_kind == "e4m3")
