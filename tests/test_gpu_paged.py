"""Paged KV cache operators on the GPU against the float64 oracle: page plans,
row writes, causal attention of new tokens, the accepted path's compaction, and
a run of them together with the tree verify.  Whole numbers and copies are
equal; attention is held element by element to the oracle's derived bound."""
import numpy as np
import pytest
import torch

from oracle import builder as OB
from oracle import paged as OP

pytestmark = pytest.mark.gpu
DEV = "cuda"
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BAD_INDEX, NO_PAGES = 4, 16


@pytest.fixture(scope="module", autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from dforktree_b200 import build
    build.build()


def _K():
    from dforktree_b200 import kernels
    return kernels


def _np(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------- plan --
class Tables:
    """Device tables and the oracle's copies of them."""

    def __init__(self, R, max_pages, n_pages, page, seed):
        rng = np.random.default_rng(seed)
        self.page, self.n_pages = page, n_pages
        self.stack = [int(x) for x in rng.permutation(n_pages)]
        self.table, self.held = np.full((R, max_pages), -1), np.zeros(R, np.int64)
        # a table of wider pitch: its rows are a slice
        self.d_table = torch.full((R, max_pages + 3), -1, dtype=torch.int32, device=DEV)[:, :max_pages]
        self.d_held, self.d_free = _i32([0] * R), _i32(self.stack)
        self.d_n = _i32([n_pages])

    def plan(self, cached, fresh, rows, tokens, keys=None, status=None):
        out = _K().page_plan_outputs(len(cached), tokens, self.n_pages * self.page if keys is None else keys, DEV)
        for t in out.values():
            t.fill_(77)
        r = None if rows is None else _i64(rows)
        return _K().page_plan(_i64(cached), _i64(fresh), self.d_table, self.d_held, self.d_free, self.d_n, self.page,
                              rows=r, out=out, status=status)

    def same(self):
        n = int(self.d_n.item())
        assert n == len(self.stack) and self.d_free[:n].tolist() == self.stack
        assert self.d_held.tolist() == self.held.tolist()
        got = self.d_table.cpu().numpy()
        for r, h in enumerate(self.held):
            assert got[r, :h].tolist() == self.table[r, :h].tolist(), r


def _same_maps(out, want, tokens, keys):
    qo, kv, idx, slots, pos = want
    assert out["qo_indptr"].tolist() == qo and out["kv_indptr"].tolist() == kv
    assert out["kv_indices"].tolist() == idx + [77] * (keys - len(idx))
    assert out["slot_map"].tolist() == slots + [-1] * (tokens - len(slots))
    assert out["positions"].tolist() == pos + [0] * (tokens - len(pos))


@pytest.mark.parametrize("B,R,page,longest", [(1, 1, 1, 40), (3, 5, 16, 200), (64, 64, 4, 90), (33, 40, 64, 700),
                                              (1024, 1030, 16, 60), (2, 2, 1024, 3000)])
def test_plan_grows_and_shrinks_like_the_oracle(B, R, page, longest):
    rng = np.random.default_rng(B * 7 + page)
    width = -(-longest // page)
    n_pages = R * width
    t = Tables(R, width, n_pages, page, B)
    length = np.zeros(R, np.int64)
    for step in range(6):
        rows = rng.permutation(R)[:B]
        cached = np.array([rng.integers(0, length[r] + 1) for r in rows])
        fresh = np.array([rng.integers(0, longest - c + 1) * rng.integers(0, 2) for c in cached])
        if step == 4:
            cached[:], fresh[:] = 0, 0                      # every request finishes
        want = OP.page_plan(cached, fresh, rows, t.table, t.held, t.stack, page)
        tokens, keys = int(fresh.sum()) + step, n_pages * page
        st = _status()
        out = t.plan(cached, fresh, rows, tokens, status=st)
        assert st.item() == 0
        _same_maps(out, want, tokens, keys)
        t.same()
        length[rows] = cached + fresh


def test_plan_without_rows_and_of_no_requests():
    t = Tables(3, 4, 12, 8, 1)
    want = OP.page_plan([0, 0], [9, 1], [0, 1], t.table, t.held, t.stack, 8)
    _same_maps(t.plan([0, 0], [9, 1], None, 10), want, 10, 96)
    t.same()
    out = t.plan([], [], None, 3)
    assert out["qo_indptr"].tolist() == [0] and out["kv_indptr"].tolist() == [0]
    assert out["slot_map"].tolist() == [-1] * 3 and out["positions"].tolist() == [0] * 3
    t.same()


@pytest.mark.parametrize("kw,bit", [
    (dict(fresh=[200, 0, 0], tokens=200, keys=300), NO_PAGES),                    # more than the stack holds
    (dict(cached=[-1, 0, 0]), BAD_INDEX), (dict(fresh=[0, -3, 0]), BAD_INDEX),
    (dict(cached=[30, 9, 1]), BAD_INDEX),                   # beyond the pages held
    (dict(cached=[2 ** 62, 0, 0], fresh=[2 ** 62, 0, 0]), BAD_INDEX),
    (dict(fresh=[2 ** 40, 0, 0]), BAD_INDEX), (dict(fresh=[2000, 0, 0]), BAD_INDEX),   # beyond the table's width
    (dict(rows=[0, 5, 0]), BAD_INDEX), (dict(rows=[0, 1, 99]), BAD_INDEX), (dict(rows=[-1, 1, 2]), BAD_INDEX),
    (dict(tokens=2, fresh=[2, 1, 0]), BAD_INDEX), (dict(keys=8, tokens=9, fresh=[9, 0, 0]), BAD_INDEX),
])
def test_a_plan_that_cannot_be_made_changes_nothing(kw, bit):
    t = Tables(6, 60, 24, 4, 3)
    OP.page_plan([0, 0, 0], [20, 8, 0], [0, 5, 3], t.table, t.held, t.stack, 4)
    t.plan([0, 0, 0], [20, 8, 0], [0, 5, 3], 28)
    t.same()
    a = dict(cached=[0, 0, 0], fresh=[0, 0, 0], rows=[0, 5, 3], tokens=6, keys=96)
    a.update(kw)
    st = _status()
    out = t.plan(a["cached"], a["fresh"], a["rows"], a["tokens"], a["keys"], st)
    assert st.item() == bit
    assert out["qo_indptr"].tolist() == [0] * 4 and out["kv_indptr"].tolist() == [0] * 4
    assert out["slot_map"].tolist() == [-1] * a["tokens"] and out["kv_indices"].tolist() == [77] * a["keys"]
    t.same()


def test_plan_with_corrupt_counts_changes_nothing():
    t = Tables(3, 8, 12, 4, 5)
    t.d_n.fill_(13)
    st = _status()
    t.plan([0, 0], [4, 4], None, 8, status=st)
    assert st.item() == BAD_INDEX and t.d_held.tolist() == [0, 0, 0]
    t.d_n.fill_(12)
    t.d_held[1] = 9
    st = _status()
    t.plan([0, 0], [4, 4], None, 8, status=st)
    assert st.item() == BAD_INDEX and t.d_n.item() == 12


# ----------------------------------------------------------------- append --
@pytest.mark.parametrize("T,Hkv,D,dtype,fused", [(1, 4, 256, torch.bfloat16, True), (7, 2, 128, torch.float16, True),
                                                 (130, 8, 64, torch.bfloat16, False), (5, 3, 30, torch.float16, True),
                                                 (1000, 4, 256, torch.bfloat16, True), (3, 1, 1, torch.bfloat16, False)])
@pytest.mark.parametrize("layout", ["split", "fused", "heads"])
def test_append_writes_the_named_slots_only(T, Hkv, D, dtype, fused, layout):
    g = torch.Generator(device=DEV).manual_seed(T + D)
    if fused:
        x = torch.randn(T, (5 + 2 * Hkv) * D, device=DEV, generator=g).to(dtype)
        k, v = (x[:, (5 + i * Hkv) * D:(5 + (i + 1) * Hkv) * D].view(T, Hkv, D) for i in (0, 1))
    else:
        k, v = (torch.randn(Hkv, T, D, device=DEV, generator=g).to(dtype).transpose(0, 1) for _ in range(2))
    slots = T + 9
    if layout == "split":
        kc, vc = (torch.randn(slots, Hkv, D, device=DEV, generator=g).to(dtype) for _ in range(2))
    elif layout == "fused":
        c = torch.randn(slots, 2, Hkv, D, device=DEV, generator=g).to(dtype)
        kc, vc = c[:, 0], c[:, 1]
    else:
        kc, vc = (torch.randn(Hkv, slots, D, device=DEV, generator=g).to(dtype).transpose(0, 1) for _ in range(2))
    slot = torch.randperm(slots, device=DEV, generator=g)[:T]
    slot[T // 3::5] = -1
    if T > 4:
        slot[4] = -2 ** 40
    wk, wv = kc.clone(), vc.clone()
    live = slot >= 0
    wk[slot[live]], wv[slot[live]] = k[live], v[live]
    st = _status()
    _K().kv_append(k, v, kc, vc, slot, status=st)
    assert st.item() == 0 and torch.equal(kc, wk) and torch.equal(vc, wv)


def test_append_refuses_slots_past_the_cache_and_takes_no_tokens():
    k = torch.ones(4, 2, 64, device=DEV, dtype=torch.bfloat16)
    c = torch.zeros(5, 2, 64, device=DEV, dtype=torch.bfloat16)
    d = c.clone()
    st = _status()
    _K().kv_append(k, k, c, d, _i64([0, 5, 2 ** 40, 3]), status=st)
    assert st.item() == BAD_INDEX
    assert c[:, 0, 0].tolist() == [1, 0, 0, 1, 0] and torch.equal(c, d)
    _K().kv_append(k[:0], k[:0], c, d, _i64([]))
    assert c[:, 0, 0].tolist() == [1, 0, 0, 1, 0]


# ----------------------------------------------------------------- commit --
@pytest.mark.parametrize("B,Ln,N,P,Hkv,D,dtype", [(1, 1, 1, 1, 1, 64, torch.bfloat16), (3, 2, 32, 24, 4, 256, torch.bfloat16),
                                                  (5, 3, 64, 70, 2, 128, torch.float16), (4, 1, 16, 5, 3, 30, torch.float16)])
def test_commit_moves_the_accepted_rows(B, Ln, N, P, Hkv, D, dtype):
    rng = np.random.default_rng(B + N)
    lens = [N + int(rng.integers(0, 50)) for _ in range(B)]
    slots = sum(lens) + 5
    idx = rng.permutation(slots)[:sum(lens)]
    kv = np.concatenate([[0], np.cumsum(lens)])
    path = np.full((B, P), -1)
    alen = rng.integers(0, min(N, P) + 1, B)
    alen[0] = min(N, P)
    for b in range(B):
        path[b, :alen[b]] = np.sort(rng.permutation(N)[:alen[b]])
    if B > 2:
        alen[2] = P + 7                    # longer than the path kept: the path's end counts
    kc, vc = (torch.randn(Ln, slots, Hkv, D, device=DEV).to(dtype) for _ in range(2))
    wk, wv = (OP.kv_commit(_np(c), kv, idx, path, alen, N) for c in (kc, vc))
    st = _status()
    _K().kv_commit(kc, vc, _i32(kv), _i32(idx), _i64(path), _i64(alen), N, status=st)
    assert st.item() == 0 and np.array_equal(_np(kc), wk) and np.array_equal(_np(vc), wv)


@pytest.mark.parametrize("path,alen,kv", [([0, 2, 2, -1], 3, 8), ([1, 0, 3, -1], 3, 8), ([0, 8, -1, -1], 2, 8),
                                          ([0, 1, 2, 3], 4, 7), ([0, 2, 3, 4], 4, 9)])
def test_commit_refuses_what_is_no_path(path, alen, kv):
    kc = torch.randn(20, 2, 64, device=DEV).to(torch.bfloat16)
    vc = torch.randn(20, 2, 64, device=DEV).to(torch.bfloat16)
    k0, v0 = kc.clone(), vc.clone()
    idx = _i32([3, 1, 4, 15, 9, 2, 6, 5])
    st = _status()
    _K().kv_commit(kc, vc, _i32([0, kv]), idx, _i64([path]), _i64([alen]), 8, status=st)
    assert st.item() == BAD_INDEX and torch.equal(kc, k0) and torch.equal(vc, v0)


def test_commit_refuses_slots_outside_the_cache():
    kc = torch.randn(20, 2, 64, device=DEV).to(torch.bfloat16)
    k0 = kc.clone()
    for bad in (20, -1):
        st = _status()
        _K().kv_commit(kc, kc.clone(), _i32([0, 4]), _i32([3, 1, bad, 2]), _i64([[0, 2, 3]]), _i64([3]), 4, status=st)
        assert st.item() == BAD_INDEX and torch.equal(kc, k0)


# ----------------------------------------------------------------- attend --
def _attn_case(fresh, cached, Hq, Hkv, D, dtype, page=1, seed=0, layout="split", scale=None, ramp=None, pad=0,
               lens=None):
    """Packed queries, a cache with every request's pages scattered, and maps.
    lens overrides the key counts (default cached + fresh)."""
    rng = np.random.default_rng(seed + 31 * len(fresh) + sum(fresh) + D)
    g = torch.Generator(device=DEV).manual_seed(int(rng.integers(1 << 30)))
    lens = [c + f for c, f in zip(cached, fresh)] if lens is None else lens
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    perm = rng.permutation(pages)
    idx, at = [], 0
    for n, p in zip(lens, need):
        mine = perm[at:at + p]
        at += p
        idx += [int(mine[j // page]) * page + j % page for j in range(n)]
    slots, T = pages * page, sum(fresh) + pad
    # q is a slice of a fused projection
    q = torch.randn(T, (Hq + 2) * D, device=DEV, generator=g).to(dtype)[:, D:(Hq + 1) * D].view(T, Hq, D)
    k, v = (torch.randn(slots, Hkv, D, device=DEV, generator=g) for _ in range(2))
    if ramp is not None:          # key norms rising along each request's context
        m = torch.ones(slots, device=DEV)
        o = 0
        for n in lens:
            m[torch.tensor(idx[o:o + n], dtype=torch.int64, device=DEV)] = torch.linspace(0.2, ramp, n, device=DEV)
            o += n
        k = k * m[:, None, None]
    k, v = k.to(dtype), v.to(dtype)
    if layout == "fused":
        c = torch.stack([k, v], 1)
        k, v = c[:, 0], c[:, 1]
    elif layout == "heads":
        k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    return dict(q=q, k=k, v=v, qo=np.concatenate([[0], np.cumsum(fresh)]), kv=np.concatenate([[0], np.cumsum(lens)]),
                idx=np.array(idx, np.int64), scale=D ** -0.5 if scale is None else scale)


def _attend(c, status=None, o=None, **kw):
    idx = c["idx"] if len(c["idx"]) else np.zeros(0, np.int32)
    return _K().chunk_attention(c["q"], c["k"], c["v"], _i32(c["qo"]), _i32(c["kv"]), _i32(idx), sm_scale=c["scale"],
                                o=o, status=status, **kw)


def _oracle(c):
    return OP.chunk_attention(_np(c["q"]), _np(c["k"]), _np(c["v"]), c["qo"], c["kv"], c["idx"], c["scale"],
                              UNIT[c["q"].dtype])


def _held(c, got, rows=None):
    want, bound = _oracle(c)
    rows = slice(0, c["qo"][-1]) if rows is None else rows
    got, want, bound = _np(got)[rows], want[rows], bound[rows]
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), (np.abs(got - want).max(), float((np.abs(got - want) / np.maximum(bound, 1e-30)).max()),
                              np.argwhere(off > 0)[:4].tolist())


BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("fresh,cached,Hq,Hkv,D,dtype,page", [
    ([1], [0], 4, 1, 256, BF, 1),                          # one token, one key
    ([1], [1], 16, 4, 256, BF, 16),
    ([1, 1, 1, 1], [62, 63, 64, 65], 16, 4, 256, BF, 16),  # key counts round a tile's edge
    ([1, 1, 1, 1], [126, 127, 128, 129], 8, 8, 128, HF, 4),
    ([1] * 9, [0, 1, 5, 31, 32, 33, 900, 2000, 4095], 16, 4, 256, BF, 16),
    ([1], [5000], 16, 2, 256, BF, 64),                     # few rows, a long axis
    ([1, 1], [3000, 17], 4, 4, 64, BF, 16),                # one q-head per kv-head
    ([1, 1], [700, 1300], 24, 2, 128, HF, 4),              # twelve q-heads per kv-head
    ([40], [0], 16, 4, 256, BF, 1),
    ([33, 32, 31, 1], [0, 5, 64, 100], 16, 4, 256, BF, 16),
    ([70, 3, 130], [10, 250, 0], 6, 2, 128, BF, 16),       # three q-heads per kv-head: 42 tokens a tile
    ([129, 128, 127], [1, 0, 300], 8, 8, 128, BF, 64),
    ([200, 1, 1, 65], [100, 500, 0, 63], 8, 2, 64, HF, 16),
    ([257], [0], 8, 1, 256, HF, 4),                        # eight q-heads, float16, one kv-head
    ([5, 9], [40, 300], 128, 1, 64, BF, 16),               # a whole tile per token
    ([3, 2], [200, 30], 254, 2, 64, BF, 16),               # 127 q-heads per kv-head
    ([0, 5, 0, 1, 0], [10, 3, 0, 200, 64], 16, 4, 256, BF, 16),   # requests that bring nothing
    ([300], [700], 4, 1, 256, BF, 16),
    ([190], [2500], 4, 2, 128, HF, 16),
    # several long units to a CTA, masked tiles far apart
    ([1] * 40, list(range(2000, 4000, 50)), 16, 4, 256, BF, 16),
    ([1] * 70, [1500 + 13 * b for b in range(70)], 32, 8, 128, HF, 16),
    ([1, 250, 1, 1, 1, 40] * 3, [1900] * 18, 16, 2, 128, BF, 16),
    ([700, 650, 1, 900], [0, 300, 1700, 20], 16, 8, 64, BF, 16),
    ([1500], [100], 16, 8, 256, BF, 64),
])
def test_attention_within_the_derived_bound(fresh, cached, Hq, Hkv, D, dtype, page):
    c = _attn_case(fresh, cached, Hq, Hkv, D, dtype, page)
    st = _status()
    o = _attend(c, st)
    assert st.item() == 0
    _held(c, o)


@pytest.mark.parametrize("layout", ["fused", "heads"])
@pytest.mark.parametrize("D,dtype", [(256, BF), (128, HF), (64, BF)])
def test_attention_of_other_cache_layouts(layout, D, dtype):
    c = _attn_case([1, 50, 7], [300, 20, 129], 8, 4, D, dtype, 16, layout=layout)
    _held(c, _attend(c))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_with_rising_scores_and_other_scales(D, dtype):
    # the running maximum rises tile after tile; weights concentrate on few keys
    c = _attn_case([1, 60], [900, 400], 8, 2, D, dtype, 16, seed=3, scale=3.0 * D ** -0.5, ramp=3.0)
    _held(c, _attend(c))
    c["scale"] = 1e-4
    _held(c, _attend(c))


def test_rows_that_see_nothing_and_rows_of_no_request():
    # fewer keys than tokens: the first tokens see nothing and get 0
    c = _attn_case([6, 70, 3, 4], [0] * 4, 16, 4, 256, BF, 1, lens=[2, 40, 0, 4], pad=9)
    o = torch.full(c["q"].shape, 5.0, device=DEV, dtype=BF)
    st = _status()
    _attend(c, st, o=o)
    assert st.item() == 0
    _held(c, o)
    assert (o[:4] == 0).all() and (o[6:36] == 0).all() and (o[76:79] == 0).all()
    assert (o[83:] == 5.0).all()


@pytest.mark.parametrize("D,dtype", [(256, BF), (128, HF), (64, BF)])
def test_unseen_values_do_not_reach_a_row(D, dtype):
    """NaN and infinities at later tokens' keys, in the rest of a page and in
    unused pages; each row is what it is without them, and a row that does see
    one is NaN (its value) in the same dims as the formula's."""
    fresh, cached = [1, 90, 1], [70, 37, 0]
    c = _attn_case(fresh, cached, 8, 2, D, dtype, 64, seed=5)
    clean = _np(_attend(c))
    used = np.zeros(c["k"].shape[0], bool)
    used[c["idx"]] = True
    k, v = c["k"].clone(), c["v"].clone()
    spare = torch.from_numpy(~used).to(DEV)
    k[spare], v[spare] = float("nan"), float("inf")
    late = [int(c["idx"][71 + 37 + 50]), int(c["idx"][71 + 37 + 81])]     # the keys of tokens 50 and 81
    k[late[0]] = float("nan")
    v[late[0], :, 3] = float("nan")
    v[late[0], :, 5] = float("inf")
    v[late[1], 1, 7] = float("-inf")
    got = _np(_attend(dict(c, k=k, v=v)))
    rows = list(range(0, 51)) + [91]                         # requests 0 and 2, and tokens before the first
    assert np.array_equal(got[rows], clean[rows])
    assert np.isnan(got[51:91]).all()                        # their scores are NaN
    # only values: scores stay finite, so only the dims concerned change
    got = _np(_attend(dict(c, v=v)))
    assert np.array_equal(got[rows], clean[rows])
    for i, t in enumerate(range(51, 91)):
        for hq in range(8):
            odd = {3, 5} | ({7} if i >= 31 and hq // 4 == 1 else set())
            fine = [d for d in range(D) if d not in odd]
            assert np.isnan(got[t, hq, 3]) and got[t, hq, 5] == np.inf
            if 7 in odd:
                assert got[t, hq, 7] == -np.inf
            # all but those dims as without them, to the type's own rounding of a sum taken in two parts
            assert np.isfinite(got[t, hq, fine]).all()
            assert np.abs(got[t, hq, fine] - clean[t, hq, fine]).max() <= 2 * UNIT[dtype] * np.abs(clean[t, hq]).max()


def test_a_value_that_every_row_sees_is_not_hidden():
    c = _attn_case([3], [200], 4, 1, 128, BF, 16)
    c["v"][int(c["idx"][20]), 0, 9] = float("inf")
    got = _np(_attend(c))
    assert (got[:, :, 9] == np.inf).all() and np.isfinite(np.delete(got, 9, 2)).all()
    c = _attn_case([3], [200], 4, 1, 128, BF, 16)
    c["q"][1, 2] = float("nan")
    got = _np(_attend(c))
    assert np.isnan(got[1, 2]).all() and np.isfinite(got[[0, 2]]).all() and np.isfinite(got[1, [0, 1, 3]]).all()


def test_offsets_and_slots_out_of_range_are_reported_and_nothing_else_is_touched():
    c = _attn_case([4, 5], [30, 20], 8, 2, 128, BF, 1)
    clean = _np(_attend(c))
    for slot in (c["k"].shape[0], -1, 2 ** 31 - 1):
        idx = c["idx"].copy()
        idx[10] = slot
        st = _status()
        got = _np(_attend(dict(c, idx=idx), st))
        assert st.item() == BAD_INDEX and np.array_equal(got[4:], clean[4:]) and np.isfinite(got).all()
    for qo, kv, kept in (([0, 4, 10], [0, 34, 59], 0), ([0, 4, 3], [0, 34, 59], 0), ([0, 4, 9], [0, 34, 60], 0),
                         ([0, 4, 9], [0, 34, 33], 0), ([-1, 4, 9], [0, 34, 59], 1), ([0, 4, 9], [-2, 34, 59], 1)):
        o = torch.full(c["q"].shape, 5.0, device=DEV, dtype=BF)
        st = _status()
        _attend(dict(c, qo=qo, kv=kv), st, o=o)
        assert st.item() == BAD_INDEX
        got = _np(o)
        good = slice(0, 4) if kept == 0 else slice(4, 9)
        assert np.array_equal(got[good], clean[good])
        rest = np.delete(got, np.r_[good], 0)
        assert (rest == 5.0).all()


def test_no_tokens_and_no_requests():
    c = _attn_case([0, 0], [5, 0], 4, 2, 64, BF)
    assert _attend(c).shape == (0, 4, 64)
    c = _attn_case([4], [5], 4, 2, 64, BF)
    o = torch.full(c["q"].shape, 5.0, device=DEV, dtype=BF)
    _attend(dict(c, qo=[0], kv=[0]), o=o)
    assert (o == 5.0).all()


def test_slots_past_32_bit_offsets():
    """A cache whose last slots lie past 2^31 elements and 2^32 bytes."""
    slots = 2_200_000
    k, v = (torch.empty(slots, 4, 256, device=DEV, dtype=BF) for _ in range(2))
    idx = np.concatenate([np.arange(slots - 90, slots), np.arange(5)])
    q = torch.randn(11, 16, 256, device=DEV).to(BF)
    t = torch.from_numpy(idx).to(DEV)
    new = torch.randn(2, 95, 4, 256, device=DEV).to(BF)
    _K().kv_append(new[0], new[1], k, v, t)
    assert torch.equal(k[t], new[0]) and torch.equal(v[t], new[1])
    st = _status()
    o = _K().chunk_attention(q, k, v, _i32([0, 11]), _i32([0, 95]), _i32(idx), status=st)
    assert st.item() == 0
    c = dict(q=q, k=new[0], v=new[1], qo=[0, 11], kv=[0, 95], idx=np.arange(95), scale=1 / 16)
    _held(c, o)
    path, tree = [0, 3, 4], t[-8:]
    _K().kv_commit(k, v, _i32([0, 95]), _i32(idx), _i64([path]), _i64([3]), 8)
    assert torch.equal(k[tree[:3]], new[0][-8:][path]) and torch.equal(v[tree[:3]], new[1][-8:][path])


def test_many_requests_and_a_long_ragged_batch():
    rng = np.random.default_rng(2)
    fresh = [1] * 1024
    cached = [int(x) for x in rng.integers(0, 40, 1024)]
    c = _attn_case(fresh, cached, 4, 2, 64, BF, 4)
    _held(c, _attend(c))
    fresh = [int(x) for x in rng.integers(0, 60, 40)]
    cached = [int(x) for x in rng.integers(0, 200, 40)]
    c = _attn_case(fresh, cached, 8, 2, 128, BF, 16)
    _held(c, _attend(c))


def test_the_same_call_twice_and_on_another_stream():
    c = _attn_case([1, 300, 2], [3000, 100, 64], 16, 4, 256, BF, 16)
    a = _attend(c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = _attend(c)
    d = _attend(c)                         # at the same time, on the first stream
    s.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, d)


def test_a_workspace_that_is_too_small_is_refused():
    from dforktree_b200 import _lib as L
    c = _attn_case([1], [300], 4, 1, 256, BF)
    with pytest.raises(L.DFTError):
        _attend(c, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))


# -------------------------------------------------------------- together --
def test_prompt_chunks_tokens_and_a_tree_step_together():
    """Two requests: prompts in chunks, single tokens, a tree step with its
    masked verify, commit of the accepted path, then tokens again, with a third
    request finishing and its pages reused; every attention output against the
    oracle over each request's own history of K / V rows."""
    from dforktree_b200 import synth
    from dforktree_b200.paged_kv import PagedKV
    Hq, Hkv, D, N, P, Ln = 16, 4, 256, 32, 24, 2
    g = torch.Generator(device=DEV).manual_seed(8)
    rng = np.random.default_rng(8)
    kv = PagedKV(rows=3, max_len=400, layers=Ln, Hkv=Hkv, D=D, page_size=16, n_pages=40)
    hist = [[np.zeros((0, Hkv, D))] * 2 for _ in range(3 * Ln)]     # (K, V) rows of (request, layer)
    length = np.zeros(3, np.int64)

    def rnd(*s):
        return torch.randn(*s, device=DEV, generator=g).to(BF)

    def step(reqs, fresh, pad=0):
        T = sum(fresh) + pad
        kv.plan(_i64(length[reqs]), _i64(fresh), tokens=T, rows=_i64(reqs))
        for layer in range(Ln):
            q, k, v = rnd(T, Hq, D), rnd(T, Hkv, D), rnd(T, Hkv, D)
            kv.append(layer, k, v)
            o = kv.attend(layer, q)
            at = 0
            for r, n in zip(reqs, fresh):
                h = hist[r * Ln + layer]
                hist[r * Ln + layer] = [np.concatenate([x, _np(y[at:at + n])]) for x, y in zip(h, (k, v))]
                kk, vv = hist[r * Ln + layer]
                want, bound = OP.chunk_attention(_np(q[at:at + n]), kk, vv, [0, n], [0, len(kk)],
                                                 np.arange(len(kk)), D ** -0.5, 2.0 ** -8)
                assert (np.abs(_np(o[at:at + n]) - want) <= bound).all()
                at += n
        for r, n in zip(reqs, fresh):
            length[r] += n

    step([0, 1, 2], [100, 17, 60])
    step([2, 0], [40, 30], pad=5)
    step([0, 1, 2], [1, 1, 1])
    kv.plan(_i64([0]), _i64([0]), tokens=0, rows=_i64([2]))          # request 2 finishes
    assert kv.n_free.item() == 40 - sum(-(-int(n) // 16) for n in length[:2])
    # a tree step of requests 0 and 1
    parents = [synth.random_tree_parents(N, rng) for _ in range(2)]
    anc = np.stack([OB.tree_struct(p, 4)[0] for p in parents])
    kv.plan(_i64(length[:2]), _i64([N, N]), tokens=2 * N, rows=_i64([0, 1]))
    tree = kv.tree(torch.from_numpy(anc).to(DEV), Hq)
    path = np.full((2, P), -1)
    for b in range(2):
        nodes = np.nonzero(anc[b][int(np.argmax(anc[b].sum(1)))] > 0.5)[0][:P]
        path[b, :len(nodes)] = nodes
    alen = (path >= 0).sum(1)
    for layer in range(Ln):
        q, k, v = rnd(2, N, Hq, D), rnd(2, N, Hkv, D), rnd(2, N, Hkv, D)
        kv.append(layer, k.flatten(0, 1), v.flatten(0, 1))
        o = _np(tree.run(q, (kv.k_cache[layer], kv.v_cache[layer])))
        for b in range(2):
            kk, vv = (np.concatenate([x, _np(y[b])]) for x, y in zip(hist[b * Ln + layer], (k, v)))
            for n in (0, 5, 31):
                see = np.concatenate([np.arange(length[b]), length[b] + np.nonzero(anc[b][n] > 0.5)[0]])
                want, bound = OP.chunk_attention(_np(q[b, n:n + 1]), kk, vv, [0, 1], [0, len(see)], see, D ** -0.5,
                                                 2.0 ** -8)
                assert (np.abs(o[b, n] - want[0]) <= bound[0]).all()
            hist[b * Ln + layer] = [np.concatenate([x, _np(y[b])[path[b][:alen[b]]]])
                                    for x, y in zip(hist[b * Ln + layer], (k, v))]
    kv.commit(_i64(path), _i64(alen), N)
    length[:2] += alen
    step([1, 0], [1, 1])
    length[2] = 0
    for layer in range(Ln):
        hist[2 * Ln + layer] = [np.zeros((0, Hkv, D))] * 2
    step([0, 2, 1], [1, 90, 20])                                      # a new request on the freed pages
    assert kv.device_status() == 0


def test_a_captured_step_follows_its_lengths():
    """plan + append + attend captured once, replayed at other lengths, while a
    second graph of the same cache lives."""
    from dforktree_b200.paged_kv import PagedKV
    B, T, Hq, Hkv, D = 3, 24, 8, 2, 128
    kv = PagedKV(rows=B, max_len=300, layers=1, Hkv=Hkv, D=D, page_size=16)
    cached, fresh = _i64([0] * B), _i64([0] * B)
    q = torch.zeros(T, Hq, D, device=DEV, dtype=BF)
    k, v = (torch.zeros(T, Hkv, D, device=DEV, dtype=BF) for _ in range(2))
    o = torch.zeros_like(q)
    maps = [kv.outputs(B, T) for _ in range(2)]

    def body(m):
        kv.plan(cached, fresh, out=m)
        kv.append(0, k, v)
        kv.attend(0, q, o=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body(maps[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for m in maps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            body(m)
    hist = [[np.zeros((0, Hkv, D))] * 2 for _ in range(B)]
    for step, f in enumerate(([8, 1, 0], [1, 1, 1], [10, 0, 14], [1, 20, 3], [0, 0, 0], [24, 0, 0])):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=DEV))
        fresh.copy_(_i64(f))
        o.fill_(5.0)
        graphs[step % 2].replay()
        at = 0
        for b, n in enumerate(f):
            hist[b] = [np.concatenate([x, _np(y[at:at + n])]) for x, y in zip(hist[b], (k, v))]
            want, bound = OP.chunk_attention(_np(q[at:at + n]), *hist[b], [0, n], [0, len(hist[b][0])],
                                             np.arange(len(hist[b][0])), D ** -0.5, 2.0 ** -8)
            assert (np.abs(_np(o[at:at + n]) - want) <= bound).all()
            at += n
        assert (o[at:] == 5.0).all()
        cached += fresh
    assert kv.device_status() == 0


def test_the_cycle_on_paged_caches():
    """DraftTreeCycle with page_size: prompts by extend(), then steps; the tree
    verify's outputs against the oracle over the rows kept, lengths following
    the accepted paths."""
    from dforktree_b200 import synth
    from dforktree_b200.cycle import CycleConfig, DraftTreeCycle
    from dforktree_b200.ngram_gpu import load_npz_arrays
    from dforktree_b200.workload import cycle_inputs, path_target
    V = 2048
    cfg = CycleConfig(B=3, V=V, N=16, layers=3, Hk=2, Hv=4, attn_layers=1, Hq=8, Hkv=2, Da=256, prefix=64, P=8,
                      page_size=16, max_len=256)
    table = _K().Table(load_npz_arrays(synth.make_ngram_table(V, 20000, 60000, seed=1)), beta3=60.0)
    cyc = DraftTreeCycle(cfg, table, DEV)
    g = torch.Generator(device=DEV).manual_seed(4)

    def rnd(*s):
        return torch.randn(*s, device=DEV, generator=g).to(BF)

    fresh = [40, 1, 17]
    q, k, v = rnd(1, 60, 8, 256), rnd(1, 60, 2, 256), rnd(1, 60, 2, 256)
    o = cyc.extend(_i64(fresh), q, k, v)
    hist, at = [], 0
    for n in fresh:
        hist.append([_np(y[0, at:at + n]) for y in (k, v)])
        want, bound = OP.chunk_attention(_np(q[0, at:at + n]), *hist[-1], [0, n], [0, n], np.arange(n), 1 / 16,
                                         2.0 ** -8)
        assert (np.abs(_np(o[0, at:at + n]) - want) <= bound).all()
        at += n
    assert (o[0, 58:] == 0).all() and cyc.kv_len.tolist() == fresh
    for s in range(3):
        inp = cycle_inputs(cfg, DEV, seed=50 + s)
        k, v = rnd(1, 3, 16, 2, 256), rnd(1, 3, 16, 2, 256)
        cyc.step(inp["logits"], inp["root"], inp["pre1"], inp["x"], inp["a"], inp["b"],
                 lambda tree: path_target(tree, inp["acc_len"]), inp["q"], k, v)
        anc, path, alen = _np(cyc.tree["anc"]), cyc.path.cpu().numpy(), cyc.accept_len.clamp(max=8).tolist()
        out = _np(cyc.o_attn)
        for b in range(3):
            n0 = len(hist[b][0])
            kk, vv = (np.concatenate([x, _np(y[0, b])]) for x, y in zip(hist[b], (k, v)))
            for n in (0, 7, 15):
                see = np.concatenate([np.arange(n0), n0 + np.nonzero(anc[b][n] > 0.5)[0]])
                want, bound = OP.chunk_attention(_np(inp["q"][0, b, n:n + 1]), kk, vv, [0, 1], [0, len(see)], see,
                                                 1 / 16, 2.0 ** -8)
                assert (np.abs(out[b, n] - want[0]) <= bound[0]).all()
            hist[b] = [np.concatenate([x, _np(y[0, b])[path[b][:alen[b]]]]) for x, y in zip(hist[b], (k, v))]
        assert cyc.kv_len.tolist() == [len(h[0]) for h in hist]
    assert int(cyc.status.item()) == 0


# ----------------------------------------------------------------- edges --
def test_more_work_than_31_bits_of_keys():
    """One q-head group of 128 (a token a tile): the tiles' keys sum to 2.5e9,
    past what the schedule counts one by one."""
    n, L = 12289, 200003
    g = torch.Generator(device=DEV).manual_seed(5)
    q = torch.randn(n, 128, 64, device=DEV, generator=g).to(BF)
    k, v = (torch.randn(L, 1, 64, device=DEV, generator=g).to(BF) for _ in range(2))
    st = _status()
    o = _K().chunk_attention(q, k, v, _i32([0, n]), _i32([0, L]), torch.arange(L, dtype=torch.int32, device=DEV),
                             status=st)
    assert st.item() == 0
    for i in (0, 1, 4095, 6000, n - 2, n - 1):           # each as the last token of a request of its own
        end = L - n + i + 1
        c = dict(q=q[i:i + 1], k=k[:end], v=v[:end], qo=[0, 1], kv=[0, end], idx=np.arange(end), scale=0.125)
        _held(c, o[i:i + 1])


def test_a_request_of_too_many_keys_is_reported():
    n = (1 << 25) + 1
    idx = torch.zeros(n + 9, dtype=torch.int32, device=DEV)
    q, k = torch.randn(3, 4, 64, device=DEV).to(BF), torch.randn(8, 2, 64, device=DEV).to(BF)
    o, st = torch.full_like(q, 5.0), _status()
    _K().chunk_attention(q, k, k, _i32([0, 1, 3]), _i32([0, n, n + 9]), idx, o=o, status=st)
    assert st.item() == BAD_INDEX and (o[0] == 5.0).all()
    assert torch.equal(o[1:], k[:1].repeat_interleave(2, 1).expand(2, 4, 64))    # nine times the same key


@pytest.mark.parametrize("D,G", [(64, 5), (128, 7), (256, 3), (256, 5), (256, 64), (256, 100), (256, 128)])
def test_head_groups_that_do_not_divide_a_tile(D, G):
    c = _attn_case([90, 1, 33], [150, 600, 0], 2 * G, 2, D, BF, 16)
    st = _status()
    o = _attend(c, st)
    assert st.item() == 0
    _held(c, o)


def test_expanded_queries_and_strided_outputs():
    c = _attn_case([6, 2], [40, 200], 8, 4, 128, BF, 16)
    one = torch.randn(1, 8, 128, device=DEV).to(BF)
    for q in (one.expand(8, 8, 128), one[:, :1].expand(8, 8, 128), one[:, :1].expand(1, 8, 128).expand(8, 8, 128)):
        d = dict(c, q=q)
        wide = torch.full((8, 8, 256), 7.0, device=DEV, dtype=BF)
        heads_first = torch.empty(8, 8, 128, device=DEV, dtype=BF).transpose(0, 1)
        for o in (None, wide[..., 64:192], heads_first):
            _held(d, _attend(d, o=o))
        assert (wide[..., :64] == 7.0).all() and (wide[..., 192:] == 7.0).all()


def test_two_calls_at_once_with_different_inputs():
    """Alternating on two streams, each ordered within itself only."""
    cs = [_attn_case([1] * 30, [900 + 7 * b for b in range(30)], 16, 4, 256, BF, 16),
          _attn_case([300, 40], [200, 1000], 16, 8, 128, HF, 16)]
    alone = [_attend(c) for c in cs]
    args = [(c["q"], c["k"], c["v"], _i32(c["qo"]), _i32(c["kv"]), _i32(c["idx"])) for c in cs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cs], [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_K().chunk_attention(*args[i], sm_scale=cs[i]["scale"]))
    torch.cuda.synchronize()
    for a, os in zip(alone, got):
        assert all(torch.equal(a, o) for o in os)


def test_a_padded_batch_leaves_what_lies_behind():
    """Fixed buffers with room for more tokens than there are: the maps' spare
    entries write no cache row, and o keeps its rows."""
    from dforktree_b200.paged_kv import PagedKV
    kv = PagedKV(3, 50, 1, 2, 64, page_size=8, device=DEV)
    out = kv.outputs(3, 40)
    kv.plan(_i64([0, 0, 0]), _i64([17, 0, 5]), out=out)
    k, v = (torch.randn(40, 2, 64, device=DEV).to(BF) for _ in range(2))
    kv.append(0, k, v)
    q, o = torch.randn(40, 4, 64, device=DEV).to(BF), torch.full((40, 4, 64), 7.0, device=DEV, dtype=BF)
    kv.attend(0, q, o=o)
    assert kv.device_status() == 0 and (o[22:] == 7.0).all()
    slots = out["slot_map"][:22]
    assert torch.equal(kv.k_cache[0][slots], k[:22]) and torch.equal(kv.v_cache[0][slots], v[:22])
    rest = torch.ones(kv.k_cache.shape[1], dtype=torch.bool, device=DEV)
    rest[slots] = False
    assert (kv.k_cache[0][rest] == 0).all() and (kv.v_cache[0][rest] == 0).all()
    c = dict(q=q, k=k, v=v, qo=[0, 17, 17, 22], kv=[0, 17, 17, 22], idx=np.arange(22), scale=0.125)
    _held(c, o)


def test_a_pool_that_runs_out_and_recovers():
    from dforktree_b200.paged_kv import PagedKV
    kv = PagedKV(3, 64, 2, 2, 64, page_size=16, n_pages=5, device=DEV)
    zero = _i64([0, 0, 0])
    kv.plan(zero, _i64([33, 20, 0]), tokens=60)              # three pages and two
    k, v, q = torch.randn(60, 2, 64, device=DEV).to(BF), torch.randn(60, 2, 64, device=DEV).to(BF), torch.randn(
        60, 4, 64, device=DEV).to(BF)
    kv.append(0, k, v)
    before = kv.k_cache.clone(), kv.v_cache.clone(), kv.block_table.clone(), kv.held.clone(), kv.free_pages.clone()
    m = kv.plan(_i64([33, 20, 0]), _i64([16, 0, 1]), tokens=60)   # two more: there are none
    assert kv.device_status() == NO_PAGES and m["qo_indptr"].tolist() == [0] * 4 and (m["slot_map"] == -1).all()
    o = torch.full_like(q, 7.0)
    kv.append(0, v, k)
    kv.attend(0, q, o=o)
    kv.commit(_i64([[0, 1]] * 3), _i64([0, 0, 0]), 1)             # no request holds a tree: reported, nothing moves
    assert (o == 7.0).all() and kv.device_status() == NO_PAGES | BAD_INDEX
    for a, b in zip(before, (kv.k_cache, kv.v_cache, kv.block_table, kv.held, kv.free_pages)):
        assert torch.equal(a, b)
    kv.status.zero_()
    kv.plan(_i64([0, 20, 0]), _i64([0, 12, 30]), tokens=60)       # the first request ends: three pages come back
    assert kv.device_status() == 0 and kv.held.tolist() == [0, 2, 2] and kv.n_free.item() == 1


def test_a_tree_over_a_request_that_fills_its_last_page():
    """max_len 40 in pages of 16: the table holds 48, and a tree may use them."""
    from dforktree_b200.paged_kv import PagedKV
    kv = PagedKV(1, 40, 1, 2, 256, page_size=16, device=DEV)
    kv.plan(_i64([0]), _i64([40]), tokens=40)
    new = torch.randn(2, 48, 2, 256, device=DEV).to(BF)
    kv.append(0, new[0][:40], new[1][:40])
    kv.plan(_i64([40]), _i64([8]), tokens=8)
    kv.append(0, new[0][40:], new[1][40:])
    anc = torch.tril(torch.ones(8, 8, dtype=torch.bool, device=DEV))[None]
    q = torch.randn(8, 4, 256, device=DEV).to(BF)
    o = kv.tree(anc, 4).run(q, (kv.k_cache[0], kv.v_cache[0]))
    a = kv.attend(0, q)                                           # a chain is causal
    assert kv.device_status() == 0
    c = dict(q=q, k=new[0], v=new[1], qo=[0, 8], kv=[0, 48], idx=np.arange(48), scale=1 / 16)
    _held(c, a)
    _held(c, o.view(8, 4, 256))


# ------------------------------------- short units beside long ones, row copies --
def _in_runs(c, share, seed):
    """c's key slots once more: of each request's blocks of 16 keys a share lies in
    consecutive slots and the rest anywhere among that rest's slots."""
    rng = np.random.default_rng(seed)
    idx = np.arange(len(c["idx"]))
    loose = [j for a, b in zip(c["kv"][:-1], c["kv"][1:]) for j0 in range(a, b, 16) if rng.random() >= share
             for j in range(j0, min(j0 + 16, b))]
    idx[loose] = rng.permutation(idx[loose])
    return dict(c, idx=idx)


@pytest.mark.parametrize("lens", [
    [2000, 30], [2000, 30, 30], [30, 2000, 64, 1, 65], [1, 64, 65, 128, 129, 3000], [3000, 129, 128, 65, 64, 1],
    [1500] + [40] * 20 + [1500] + [100] * 20, [64, 2500] * 12, [128, 1, 900] * 16, [200, 33] * 40, [700] * 40 + [5] * 90,
    [4000] + [7] * 63,
], ids=lambda x: f"{len(x)}-{x[0]}-{x[-1]}")
@pytest.mark.parametrize("slots", ["page1", "page4", "page8", "page16", "runs"])
def test_short_requests_beside_long_ones(lens, slots):
    """Single tokens whose units are one tile or many, in every order of the two:
    the pair form hands K and V of a tile over on their own times."""
    page = int(slots[4:]) if slots != "runs" else 1
    c = _attn_case([1] * len(lens), [n - 1 for n in lens], 16, 4, 256, BF, page, seed=len(slots))
    for seed in range(1 if slots != "runs" else 3):
        d = _in_runs(c, (0.2, 0.5, 0.8)[seed], seed) if slots == "runs" else c
        st = _status()
        o = _attend(d, st)
        assert st.item() == 0
        _held(d, o)


@pytest.mark.parametrize("page", [1, 16])
def test_many_one_tile_units_of_a_pair(page):
    rng = np.random.default_rng(page)
    for fresh, cached in (([1] * 300, rng.integers(0, 128, 300)), ([1] * 300, rng.integers(60, 256, 300)),
                          (rng.integers(0, 6, 200), rng.integers(0, 200, 200))):
        c = _attn_case([int(x) for x in fresh], [int(x) for x in cached], 8, 4, 256, HF, page)
        st = _status()
        o = _attend(c, st)
        assert st.item() == 0
        _held(c, o)


# ------------------------------------------------------ scores of -infinity --
@pytest.mark.parametrize("fresh,dead", [(1, (0, 128)), (1, (0, 500)), (1, (300, 600)), (40, (0, 256)), (40, (130, 520)),
                                        (3, (5, 9))])
@pytest.mark.parametrize("D,dtype", [(256, BF), (128, HF), (64, BF)])
def test_keys_whose_scores_are_minus_infinity_weigh_nothing(D, dtype, fresh, dead):
    """K of -infinity in a dim where q is positive, over whole tiles or parts of
    them: the rows are those of the other keys."""
    c = _attn_case([fresh, 2], [700, 90], 8, 2, D, dtype, 16, seed=9)
    q, k = c["q"].clone(), c["k"].clone()
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    gone = c["idx"][dead[0]:dead[1]]
    k[torch.from_numpy(gone).to(DEV), :, 0] = -float("inf")
    st = _status()
    o = _attend(dict(c, q=q, k=k), st)
    assert st.item() == 0
    n = dead[1] - dead[0]
    _held(dict(c, q=q, idx=np.delete(c["idx"], slice(*dead)), kv=c["kv"] - n * (np.arange(3) > 0)), o)


@pytest.mark.parametrize("D,dtype", [(256, BF), (128, HF), (64, BF)])
def test_a_row_of_scores_of_minus_infinity_alone_is_zero(D, dtype):
    for cached in (20, 127, 128, 900):
        c = _attn_case([2, 1], [cached, 50], 8, 2, D, dtype, 16, seed=cached)
        q, k = c["q"].clone(), c["k"].clone()
        q[:, :, 0] = q[:, :, 0].abs() + 0.5
        k[torch.from_numpy(c["idx"][:cached + 2]).to(DEV), :, 0] = -float("inf")
        o = _attend(dict(c, q=q, k=k))
        assert (o[:2] == 0).all()
        _held(dict(c, q=q), o, rows=slice(2, 3))


# ------------------------------------------------------------- paged cycle --
def _small_cycle(**kw):
    from dforktree_b200 import synth
    from dforktree_b200.cycle import CycleConfig, DraftTreeCycle
    from dforktree_b200.ngram_gpu import load_npz_arrays
    V = 2048
    cfg = CycleConfig(**{**dict(B=3, V=V, N=16, layers=3, Hk=2, Hv=4, attn_layers=1, Hq=8, Hkv=2, Da=256, prefix=64,
                                P=8, page_size=16, max_len=64), **kw})
    table = _K().Table(load_npz_arrays(synth.make_ngram_table(V, 20000, 60000, seed=1)), beta3=60.0)
    return DraftTreeCycle(cfg, table, DEV)


def test_a_step_whose_plan_cannot_be_made_moves_no_state():
    """One request's tree does not fit max_len: recurrent, conv and KV state of
    every request stay, nothing counts as accepted, and the step after it is
    that of a cycle which never met it."""
    from dforktree_b200.workload import cycle_inputs, path_target
    g = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = (torch.randn(1, 90, h, 256, device=DEV, generator=g).to(BF) for h in (8, 2, 2))
    kt, vt = (torch.randn(1, 3, 16, 2, 256, device=DEV, generator=g).to(BF) for _ in range(2))
    got = []
    for early in (True, False):
        cyc = _small_cycle()
        cyc.extend(_i64([50, 10, 30]), q, k, v)
        inp = cycle_inputs(cyc.cfg, DEV, seed=70)

        def step():
            cyc.step(inp["logits"], inp["root"], inp["pre1"], inp["x"], inp["a"], inp["b"],
                     lambda tree: path_target(tree, inp["acc_len"]), inp["q"], kt, vt)

        if early:
            names = ("pool", "conv_state", "kv_len")
            before = [getattr(cyc, n).clone() for n in names] + [cyc.kv.k_cache.clone(), cyc.kv.v_cache.clone()]
            step()                                   # 50 + 16 tokens: past max_len
            assert int(cyc.status.item()) == BAD_INDEX
            for a, b in zip(before, [getattr(cyc, n) for n in names] + [cyc.kv.k_cache, cyc.kv.v_cache]):
                assert torch.equal(a, b)
            assert cyc.accept_len.tolist() == [0, 0, 0] and (cyc.path == -1).all()
            assert (cyc.last == -1).all() and (cyc.bonus == -1).all()
            cyc.status.zero_()
        cyc.kv_len[0] = 20                           # the long request is cut back
        step()
        assert int(cyc.status.item()) == 0 and (cyc.accept_len > 0).all()
        assert cyc.kv_len.tolist() == [n + a for n, a in zip((20, 10, 30), cyc.accept_len.clamp(max=8).tolist())]
        got.append([x.clone() for x in (cyc.pool, cyc.conv_state, cyc.kv.k_cache, cyc.kv.v_cache, cyc.o_attn, cyc.path,
                                        cyc.last, cyc.bonus)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_an_accepted_path_longer_than_the_rows_kept_ends_there():
    """P below the tree's depth: what counts as accepted is what every state holds,
    as in a cycle with room whose target agrees with the first P nodes only."""
    from dforktree_b200.workload import cycle_inputs
    g = torch.Generator(device=DEV).manual_seed(7)
    q, k, v = (torch.randn(1, 90, h, 256, device=DEV, generator=g).to(BF) for h in (8, 2, 2))
    kt, vt = (torch.randn(1, 3, 16, 2, 256, device=DEV, generator=g).to(BF) for _ in range(2))
    got, deepest = [], []
    for P in (3, 16):
        cyc = _small_cycle(P=P, max_len=128, chain_first=True)
        cyc.extend(_i64([50, 10, 30]), q, k, v)
        inp = cycle_inputs(cyc.cfg, DEV, seed=70)

        def target(tree):
            # every node agrees with its first child; past the third node of a path only where P has room
            nxt = tree["nxt"].view(3, 16)
            t = torch.where(nxt >= 0, tree["tokens"].view(3, 16).gather(1, nxt.clamp(min=0)), -7)
            depth = tree["anc"].view(3, 16, 16).sum(-1)
            deepest.append(depth.max().item())
            return t if P == 3 else torch.where(depth >= 3, t + 10 ** 6, t)

        cyc.step(inp["logits"], inp["root"], inp["pre1"], inp["x"], inp["a"], inp["b"], target, inp["q"], kt, vt)
        assert int(cyc.status.item()) == 0 and cyc.accept_len.tolist() == [3, 3, 3]
        assert cyc.kv_len.tolist() == [53, 13, 33] and (cyc.path[:, :3] >= 0).all()
        got.append([x.clone() for x in (cyc.pool, cyc.conv_state, cyc.path[:, :3], cyc.last,
                                        cyc.bonus + (10 ** 6 if P == 3 else 0))])
        got[-1] += [cyc.kv.k_cache[0][cyc.tree_maps["slot_map"].view(3, 16)[:, :3]],
                    cyc.kv.v_cache[0][cyc.tree_maps["slot_map"].view(3, 16)[:, :3]]]
    assert min(deepest) > 4 and all(torch.equal(a, b) for a, b in zip(*got))


# ------------------------------------------------- one tree wrapper, many steps --
@pytest.mark.parametrize("kind", ["float32", "bool", "half", "strided"])
@pytest.mark.parametrize("captured", [False, True])
def test_a_tree_wrapper_follows_its_ancestor_matrix(kind, captured):
    """One tree() for several steps: the matrix and the maps change in place."""
    from dforktree_b200 import synth
    from dforktree_b200.paged_kv import PagedKV
    Hq, Hkv, D, N = 8, 2, 256, 16
    rng, g = np.random.default_rng(3), torch.Generator(device=DEV).manual_seed(3)
    kv = PagedKV(2, 200, 1, Hkv, D, page_size=16, device=DEV)
    maps, cached, fresh = kv.outputs(2, 2 * N), _i64([0, 0]), _i64([N, N])
    anc = {"float32": lambda: torch.zeros(2, N, N, device=DEV), "half": lambda: torch.zeros(2, N, N, device=DEV, dtype=HF),
           "bool": lambda: torch.zeros(2, N, N, device=DEV, dtype=torch.bool),
           "strided": lambda: torch.zeros(N, N, 2, device=DEV).permute(2, 0, 1)}[kind]()
    q, o = torch.zeros(2, N, Hq, D, device=DEV, dtype=BF), torch.zeros(2, N, Hq, D, device=DEV, dtype=BF)
    k, v = (torch.zeros(2 * N, Hkv, D, device=DEV, dtype=BF) for _ in range(2))
    kv.plan(cached, fresh, out=maps)
    tree = kv.tree(anc, Hq)

    def body():
        kv.plan(cached, fresh, out=maps)
        kv.append(0, k, v)
        tree.run(q, (kv.k_cache[0], kv.v_cache[0]), out=o)

    if captured:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            body()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            body()
    hist = [[np.zeros((0, Hkv, D))] * 2 for _ in range(2)]
    for step in range(3):
        want = np.stack([OB.tree_struct(synth.random_tree_parents(N, rng), 4)[0] for _ in range(2)])
        anc.copy_(torch.from_numpy(want).to(DEV))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device=DEV, generator=g))
        graph.replay() if captured else body()
        for b in range(2):
            rows = [_np(x[b * N:(b + 1) * N]) for x in (k, v)]
            kk, vv = (np.concatenate([x, y]) for x, y in zip(hist[b], rows))
            n0 = len(hist[b][0])
            for n in range(N):
                see = np.concatenate([np.arange(n0), n0 + np.nonzero(want[b][n] > 0.5)[0]])
                r, bound = OP.chunk_attention(_np(q[b, n:n + 1]), kk, vv, [0, 1], [0, len(see)], see, D ** -0.5, 2.0 ** -8)
                assert (np.abs(_np(o[b, n]) - r[0]) <= bound[0]).all(), (step, b, n)
            hist[b] = [x[:n0 + 5] for x in (kk, vv)]      # the first five nodes stay
        cached += 5
    assert kv.device_status() == 0


def test_a_tree_refuses_matrices_that_it_cannot_read_at_every_run():
    from dforktree_b200 import _lib as L
    from dforktree_b200.paged_kv import PagedKV
    kv = PagedKV(2, 64, 1, 2, 256, page_size=16, device=DEV)
    kv.plan(_i64([0, 0]), _i64([8, 8]), tokens=16)
    for anc in (torch.zeros(2, 8, 8), torch.zeros(1, 8, 8, device=DEV), torch.zeros(2, 8, 9, device=DEV),
                torch.zeros(2, 64, device=DEV)):
        with pytest.raises(L.DFTError):
            kv.tree(anc, 8)


def test_a_paged_step_checks_its_tensors_before_it_plans():
    from dforktree_b200 import _lib as L
    from dforktree_b200.workload import cycle_inputs, path_target
    g = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = (torch.randn(1, 60, h, 256, device=DEV, generator=g).to(BF) for h in (8, 2, 2))
    kt, vt = (torch.randn(1, 3, 16, 2, 256, device=DEV, generator=g).to(BF) for _ in range(2))
    cyc = _small_cycle(max_len=128)
    cyc.extend(_i64([20, 10, 30]), q, k, v)
    inp = cycle_inputs(cyc.cfg, DEV, seed=70)
    held, tokens = cyc.kv.held.clone(), cyc.tree["tokens"].clone()
    for bad in (dict(k=None), dict(v=None), dict(k=None, v=None), dict(q=None), dict(k=kt[:, :2]), dict(v=vt[:0]),
                dict(q=inp["q"][:, :, :8]), dict(k=kt[..., :128], v=vt[..., :128])):
        a = {**dict(q=inp["q"], k=kt, v=vt), **bad}
        with pytest.raises(L.DFTError):
            cyc.step(inp["logits"], inp["root"], inp["pre1"], inp["x"], inp["a"], inp["b"],
                     lambda tree: path_target(tree, inp["acc_len"]), **a)
        with pytest.raises(L.DFTError):
            cyc.verify(inp["x"], inp["a"], inp["b"], **a)
    with pytest.raises(L.DFTError):
        cyc.attend_layer(0, inp["q"][0])
    for bad in (dict(k=k[:, :59]), dict(v=v[:, :, :1]), dict(q=q[0]), dict(q=q[:, :, :4]), dict(fresh=_i64([1, 2]))):
        with pytest.raises(L.DFTError):
            cyc.extend(**{**dict(fresh=_i64([1, 1, 1]), q=q, k=k, v=v), **bad})
    assert torch.equal(held, cyc.kv.held) and torch.equal(tokens, cyc.tree["tokens"])
    assert cyc.kv_len.tolist() == [20, 10, 30] and int(cyc.status.item()) == 0


# ------------------------------------------------ int64 offsets and slots --
def test_int64_offsets_and_slots():
    """Taken as they are; values past 32 bits are reported, not wrapped."""
    c = _attn_case([4, 5], [30, 20], 8, 2, 128, BF, 1)
    call = lambda qo, kv, idx, o, st: _K().chunk_attention(c["q"], c["k"], c["v"], _i64(qo), _i64(kv), _i64(idx),
                                                           sm_scale=c["scale"], o=o, status=st)
    qo, kv, idx = (x.tolist() for x in (c["qo"], c["kv"], c["idx"]))
    st, clean = _status(), torch.empty_like(c["q"])
    call(qo, kv, idx, clean, st)
    assert st.item() == 0
    _held(c, clean)
    big = 2 ** 32
    for bad in (dict(qo=[0, 4, 9 + big]), dict(kv=[0, 34, 59 + big]), dict(idx=idx[:40] + [idx[40] + big] + idx[41:]),
                dict(idx=idx[:40] + [idx[40] - big] + idx[41:])):
        a = {**dict(qo=qo, kv=kv, idx=idx), **bad}
        st, o = _status(), torch.full_like(clean, 5.0)
        call(a["qo"], a["kv"], a["idx"], o, st)
        assert st.item() == BAD_INDEX and torch.equal(o[:4], clean[:4])
        assert "idx" in bad or (o[4:] == 5.0).all()
    kc, vc = (torch.randn(20, 2, 64, device=DEV).to(BF) for _ in range(2))
    k0, v0 = kc.clone(), vc.clone()
    tree = [3, 1, 4, 2]
    for kv, idx in (([0, 4 + big], tree), ([0, 4], [3, 1 + big, 4, 2]), ([0, 4], [3, 1, 4, 2 - big])):
        st = _status()
        _K().kv_commit(kc, vc, _i64(kv), _i64(idx), _i64([[0, 2, 3]]), _i64([3]), 4, status=st)
        assert st.item() == BAD_INDEX and torch.equal(kc, k0) and torch.equal(vc, v0)
    st = _status()
    _K().kv_commit(kc, vc, _i64([0, 4]), _i64(tree), _i64([[0, 2, 3]]), _i64([3]), 4, status=st)
    assert st.item() == 0 and torch.equal(kc[tree[:3]], k0[[3, 4, 2]]) and torch.equal(vc[tree[:3]], v0[[3, 4, 2]])
