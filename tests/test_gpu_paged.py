"""GPU: the paged-cache operators (append with rotation, attention of new tokens over pages) against
64-bit results, at the sizes, masks and layouts where they can go wrong. Every slot of the cache that
no sequence holds is NaN unless a test says otherwise."""
import math

import numpy as np
import pytest
import torch

from paged_ref import DT, TINY, U, Batch, rope_tables, rotate, rounding

pytestmark = pytest.mark.gpu


def _say(*a):
    print(*a, flush=True)


def _attn(gpu, bt, scale=None, window=0, prefix=None, out_t=None, max_keys=None, max_new=None, check=True, ws=None):
    scale = scale or 1.0 / math.sqrt(bt.hd)
    scale = float(np.float32(scale))
    kv = bt.device(gpu)
    out_t = out_t or bt.t
    out = torch.full((bt.tokens, bt.nh, bt.hd), 77.0, dtype=DT[out_t], device="cuda")
    lse = torch.full((bt.tokens, bt.nh), 77.0, device="cuda")
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    gpu.op_attn_paged(kv, bt.q.cuda(), scale, out, max_new=max(bt.new + [1]) if max_new is None else max_new,
                      max_keys=max_keys, lse=lse, window=window, prefix=pre, ws=ws)
    torch.cuda.synchronize()
    got, gl = out.cpu().double().numpy(), lse.cpu().double().numpy()
    if check:
        _compare(bt, got, gl, bt.attn(scale, window, prefix), out_t)
    return got, gl


def _compare(bt, got, gl, want, out_t):
    ref, rl, dout, dlse = want
    assert np.all(got[bt.T:] == 77.0) and np.all(gl[bt.T:] == 77.0)   # rows behind the last sequence
    g, l = got[:bt.T], gl[:bt.T]
    assert np.isfinite(g).all()
    tol = dout + rounding(np.abs(ref) + dout, out_t)
    bad = np.abs(g - ref) > tol
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), float(np.max(np.abs(g - ref) / np.maximum(tol, 1e-30))))
    empty = np.isneginf(rl)
    assert np.array_equal(empty, np.isneginf(l))
    assert np.all(g[empty] == 0.0)
    d = np.abs(l[~empty] - rl[~empty])
    assert np.all(d <= dlse[~empty]), float((d / dlse[~empty]).max())


# lens: (new tokens, keys in all): single tokens, chunks, ragged mixes, empty sequences, pages that end
# inside every tile
FORMS = {
    "one": [(1, 1)],
    "steps": [(1, 1), (1, 2), (1, 15), (1, 16), (1, 17), (1, 33), (1, 64), (1, 65), (1, 127), (1, 300)],
    "draft": [(3, 3), (5, 70), (2, 129), (4, 64), (7, 200)],
    "chunk": [(40, 40), (33, 97), (129, 300), (64, 64), (65, 66)],
    "long": [(257, 600)],
    "mixed": [(1, 300), (0, 40), (150, 150), (1, 1), (70, 333), (0, 0), (1, 64)],
}


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("form", list(FORMS))
def test_attention(gpu, form, hd, t):
    nh, nkv = {32: (4, 4), 64: (6, 2), 128: (8, 1)}[hd]
    bt = Batch(hd + len(form), FORMS[form], nh, nkv, hd, 16, t, tail=2)
    _attn(gpu, bt)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 512])
@pytest.mark.parametrize("form", ["steps", "mixed"])
def test_page_sizes(gpu, page, form):
    _attn(gpu, Batch(page, FORMS[form], 4, 2, 64, page, "bf16"))


@pytest.mark.parametrize("nh,nkv", [(1, 1), (3, 3), (5, 1), (10, 2), (16, 1), (17, 1), (32, 1), (40, 1), (33, 3)])
@pytest.mark.parametrize("form", ["steps", "draft", "mixed"])
def test_groups(gpu, nh, nkv, form):
    _attn(gpu, Batch(nh * 7 + nkv, FORMS[form], nh, nkv, 32, 32, "f16"))


@pytest.mark.parametrize("window", [1, 2, 16, 50, 64, 100, 1000])
@pytest.mark.parametrize("form", ["steps", "draft", "chunk", "mixed"])
def test_window(gpu, form, window):
    _attn(gpu, Batch(window, FORMS[form], 4, 2, 64, 16, "f16"), window=window)


@pytest.mark.parametrize("form", ["draft", "chunk", "mixed"])
@pytest.mark.parametrize("window", [0, 40])
def test_prefix(gpu, form, window):
    """A bidirectional prefix: shorter than the old keys, inside the chunk, the whole sequence, past its
    end, zero and negative."""
    lens = FORMS[form]
    prefix = [(tot * f) // 4 + a for (n, tot), f, a in zip(lens, [3, 4, 2, 8, 0, 1, 4], [0, 0, 1, 5, -3, 2, 0])]
    _attn(gpu, Batch(11, lens, 4, 2, 32, 16, "f16"), prefix=prefix, window=window)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("form", ["steps", "chunk"])
def test_fp32_output(gpu, form, t):
    _attn(gpu, Batch(3, FORMS[form], 4, 2, 64, 16, t), out_t="f32")


@pytest.mark.parametrize("form", ["steps", "mixed"])
def test_rows_that_see_nothing(gpu, form):
    """More new tokens than keys (the first rows lie before the sequence), no keys at all, negative lengths."""
    lens = [(n + 3 if i % 2 else n, max(0, tot - 1) if i % 3 else 0) for i, (n, tot) in enumerate(FORMS[form])]
    bt = Batch(5, lens, 4, 4, 32, 16, "f16")
    _attn(gpu, bt)
    bt.kv_len[0] = -5
    bt.K[0], bt.V[0] = bt.K[0][:0], bt.V[0][:0]
    _attn(gpu, bt)


@pytest.mark.parametrize("form", ["steps", "chunk", "mixed"])
def test_pages_that_do_not_exist(gpu, form):
    """Table entries outside the cache hide their keys: negative, n_pages and far beyond."""
    bt = Batch(6, [(n, tot + 90) for n, tot in FORMS[form]], 4, 2, 64, 16, "bf16")
    bt.table[0, 0] = -1
    bt.table[1 % bt.B, 2] = bt.n_pages
    bt.table[2 % bt.B, 1] = 2 ** 31 - 1
    bt.table[3 % bt.B, :] = -7
    _attn(gpu, bt)


@pytest.mark.parametrize("form", ["steps", "chunk"])
def test_keys_past_the_table(gpu, form):
    """kv_len beyond table_cols * page_size: the keys that have no entry do not exist."""
    _attn(gpu, Batch(7, [(n, tot + 100) for n, tot in FORMS[form]], 4, 2, 32, 16, "f16", cols=5))


@pytest.mark.parametrize("form", ["steps", "draft", "chunk", "mixed"])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_unseen_values_do_not_matter(gpu, form, what):
    """Keys and values of later tokens of the same chunk, of keys left of a window, of slots behind the
    sequence: set to NaN or infinity, the rows that do not see them are the same bits as before."""
    bt = Batch(8, FORMS[form], 4, 2, 64, 16, "f16", stale=0.5)
    want, wl = _attn(gpu, bt, window=60)
    poisoned = []
    for b, (n, tot) in enumerate(bt.lens):
        if n > 1:       # the chunk's last token: seen by its own row alone
            bt.K[b][tot - 1, 0] = what
            bt.V[b][tot - 1] = what
            poisoned.append(int(bt.seq_start[b + 1]) - 1)
        if tot - n - 60 >= 0 and n:   # the last key left of the first row's window
            bt.K[b][tot - n - 60] = what
            bt.V[b][tot - n - 60] = what
    bt.kc[:], bt.vc[:] = what, what
    bt.write()
    got, gl = _attn(gpu, bt, window=60, check=False)
    clean = [r for r in range(bt.T) if r not in poisoned]
    assert np.array_equal(got[clean], want[clean]) and np.array_equal(gl[clean], wl[clean])
    for r in poisoned:
        assert not np.isfinite(got[r]).all()


@pytest.mark.parametrize("hd", [32, 128])
def test_seen_infinities_and_nans(gpu, hd):
    """A value of infinity that a row sees gives infinity in that element, NaN gives NaN, and in no other
    element, row or head."""
    bt = Batch(9, [(70, 100), (1, 90)], 4, 2, hd, 16, "bf16")
    want, _ = _attn(gpu, bt)
    bt.V[0][50, 0, 3] = float("inf")
    bt.V[0][60, 1, 5] = float("nan")
    bt.V[1][10, 0, 7] = -float("inf")
    bt.write()
    got, _ = _attn(gpu, bt, check=False)
    exp = want.copy()
    exp[20:70, 0:2, 3] = math.inf      # rows at 30 + i see key 50 from i = 20 on
    exp[30:70, 2:4, 5] = math.nan
    exp[70, 0:2, 7] = -math.inf
    assert np.array_equal(got, exp, equal_nan=True)


def test_scores_of_minus_infinity_and_large(gpu):
    """Scores near the type's largest values and keys that score -inf: no NaN where the sum is defined."""
    bt = Batch(10, [(1, 70), (40, 90)], 2, 2, 64, 16, "f16")
    for b in range(2):
        bt.K[b][3] = 0.0
        bt.K[b][3, :, 0] = -math.inf
    bt.q[:, :, 0] = 1.0
    bt.write()
    got, gl = _attn(gpu, bt, check=False)
    for b in range(2):
        bt.K[b][3, :, 0] = -60000.0    # the same probability of zero
    want = bt.attn(float(np.float32(1 / 8.0)))
    _compare(bt, got, gl, want, "f16")
    bt = Batch(10, [(1, 70), (40, 90)], 2, 2, 64, 16, "f16", q_scale=200.0)
    _attn(gpu, bt, scale=1.0)


@pytest.mark.parametrize("hd", [32, 128])
def test_strides(gpu, hd):
    """q and out inside wider rows, pages apart from each other, table rows inside a wider table."""
    bt = Batch(12, FORMS["mixed"], 4, 2, hd, 16, "f16", page_pad=24)
    bt.device(gpu)
    wide = torch.full((bt.tokens, 3 * bt.nh * hd + 8), float("nan"), dtype=DT["f16"], device="cuda")
    q = wide.as_strided((bt.tokens, bt.nh, hd), (wide.shape[1], hd, 1), 8)
    q.copy_(bt.q)
    o = torch.full((bt.tokens, 2 * bt.nh * hd), 5.0, dtype=DT["f16"], device="cuda")
    out = o.as_strided((bt.tokens, bt.nh, hd), (o.shape[1], hd, 1), bt.nh * hd)
    table = torch.full((bt.B, bt.cols + 7), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, 3:3 + bt.cols] = bt.dtable
    kv = gpu.PagedKV(bt.dkc, bt.dvc, table[:, 3:3 + bt.cols], bt.dss, bt.dlen)
    lse = torch.full((bt.tokens, bt.nh), 77.0, device="cuda")
    scale = float(np.float32(1 / math.sqrt(hd)))
    gpu.op_attn_paged(kv, q, scale, out, max_new=max(bt.new), lse=lse)
    torch.cuda.synchronize()
    assert bool((o[:, :bt.nh * hd] == 5.0).all())
    _compare(bt, out.cpu().double().numpy(), lse.cpu().double().numpy(), bt.attn(scale), "f16")


@pytest.mark.parametrize("lens,nh,nkv,hd", [([(1, 5000)], 8, 1, 128), ([(1, 3001), (1, 7)], 2, 2, 32),
                                            ([(4, 4099)], 16, 4, 64), ([(60, 5001)], 4, 2, 128),
                                            ([(1, 3000), (2, 1801)], 64, 32, 64)])
def test_long_sequences_split(gpu, lens, nh, nkv, hd):
    """Few rows over long sequences: the work is split over the keys and joined."""
    bt = Batch(13, lens, nh, nkv, hd, 32, "bf16")
    a, la = _attn(gpu, bt)
    # planned for fewer and for more keys than there are: right either way
    _attn(gpu, bt, max_keys=1)
    _attn(gpu, bt, max_keys=1 << 20)
    b, lb = _attn(gpu, bt)
    assert np.array_equal(a, b) and np.array_equal(la, lb)


# Calls whose keys are divided among workgroups: a long chunk beside short ones, a single token, a draft,
# nothing, and a chunk without old keys
CUT = [(130, 5200), (1, 4000), (0, 0), (70, 900), (3, 2500), (33, 33), (0, 77)]


@pytest.mark.parametrize("hd,nh,nkv,t", [(32, 3, 3, "f16"), (64, 4, 1, "bf16"), (128, 4, 2, "f16")])
@pytest.mark.parametrize("kind", ["plain", "window", "prefix", "pages", "f32"])
def test_chunks_cut_into_runs(gpu, hd, nh, nkv, t, kind):
    bt = Batch(hd + len(kind), CUT, nh, nkv, hd, 32, t, tail=3)
    if kind == "pages":
        bt.table[0, ::9] = -1
        bt.table[1, 3] = bt.n_pages
        bt.table[3, :] = 2 ** 31 - 1
    kv = bt.device(gpu)
    assert gpu.attn_paged_workspace_bytes(kv, bt.tokens, nh, 130, 5200) > 0
    a = _attn(gpu, bt, window=2222 if kind == "window" else 0,
              prefix=[5150, 100, 3, 900, 0, 40, 5] if kind == "prefix" else None, out_t="f32" if kind == "f32" else None)
    b = _attn(gpu, bt, window=2222 if kind == "window" else 0, check=False,
              prefix=[5150, 100, 3, 900, 0, 40, 5] if kind == "prefix" else None, out_t="f32" if kind == "f32" else None)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_unseen_values_do_not_matter_when_cut(gpu):
    """As test_unseen_values_do_not_matter, with the keys divided among workgroups."""
    bt = Batch(17, CUT, 4, 2, 128, 32, "f16", stale=0.5)
    want, wl = _attn(gpu, bt)
    for b, (n, tot) in enumerate(bt.lens):
        if n > 1:
            bt.K[b][tot - 1], bt.V[b][tot - 1] = math.nan, math.nan
    bt.kc[:], bt.vc[:] = math.nan, math.inf
    bt.write()
    got, gl = _attn(gpu, bt, check=False)
    last = [int(bt.seq_start[b + 1]) - 1 for b, (n, _) in enumerate(bt.lens) if n > 1]
    clean = [r for r in range(bt.T) if r not in last]
    assert np.array_equal(got[clean], want[clean]) and np.array_equal(gl[clean], wl[clean])
    assert all(np.isnan(got[r]).any() for r in last)


def test_unequal_chunks(gpu):
    """Enough row tiles of unequal length for the launch to take them by length: long chunks over old
    keys, a single token and a draft beside them."""
    bt = Batch(19, [(700, 2600), (1, 1900), (540, 1500), (380, 900), (5, 40), (0, 9)], 32, 8, 32, 16, "f16", tail=1)
    bt.table[2, 11] = -1
    _attn(gpu, bt)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("form", ["steps", "chunk"])
def test_small_values(gpu, form, t):
    """Keys and values below the type's normal range (fp16 subnormals), queries large: nothing is flushed."""
    bt = Batch(20, FORMS[form], 4, 2, 64, 16, t, v_scale=2.0 ** -17, q_scale=2.0 ** 9)
    for b in range(bt.B):
        bt.K[b] = (bt.K[b].float() * 2.0 ** -16).to(DT[t])
    bt.write()
    _attn(gpu, bt, scale=2.0 ** 7)


@pytest.mark.parametrize("B", [300, 520])
def test_many_sequences(gpu, B):
    """More sequences than a workgroup has threads (and than the lists of equal runs hold), a long chunk
    among them."""
    lens = [(1 + (b % 3 == 0) * (b % 5), 1 + b % 70) for b in range(B)]
    lens = [(n, max(n, t)) for n, t in lens]
    lens[B // 2] = (150, 4000)
    lens[B - 1] = (60, 1700)
    lens[3] = (0, 5)
    _attn(gpu, Batch(B, lens, 2, 1, 128, 16, "bf16", tail=1))


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("chunks", [1, 3])
def test_chunks_among_many_sequences(gpu, chunks, window):
    """Prompts beside so many single tokens that whole row tiles are taken from a list (a grid of every sequence's
    row tiles would be empty but for a few): in the order of their lengths, and as they come where they are many."""
    lens = [(1, 1 + b % 90) for b in range(256)]
    for i in range(chunks):
        lens[100 * i + 7] = (1500 - i, 1500)
    _attn(gpu, Batch(21, lens, 8, 1, 32, 16, "f16", tail=1), window=window)


def test_more_row_tiles_than_are_summed(gpu):
    """More row tiles of a head than a workgroup has sums for (wide groups), taken whole from the list."""
    lens = [(1, 1 + b % 50) for b in range(300)]
    for i in range(6):
        lens[40 * i + 3] = (1100 + 10 * i, 1200)
    _attn(gpu, Batch(22, lens, 32, 1, 32, 16, "bf16", tail=1))


def test_nothing_to_do(gpu):
    """No rows, no sequences, sequences without rows: nothing is written and nothing fails."""
    bt = Batch(18, [(0, 20), (0, 0)], 4, 2, 64, 16, "f16", tail=4)
    _attn(gpu, bt)
    kv = bt.device(gpu)
    e = torch.empty((0, 4, 64), dtype=DT["f16"], device="cuda")
    gpu.op_attn_paged(kv, e, 0.1, e, max_new=0)
    gpu.op_paged_append(kv, e[:, :2], e[:, :2])
    gpu.op_paged_append(kv, e[:, :2], e[:, :2], q=e, q_out=e.clone())
    none = gpu.PagedKV(bt.dkc, bt.dvc, bt.dtable[:0], bt.dss[:1], bt.dlen[:0])
    q = torch.full((4, 4, 64), 3.0, dtype=DT["f16"], device="cuda")
    out = q.clone()
    gpu.op_attn_paged(none, q, 0.1, out, max_new=4)
    gpu.op_paged_append(none, q[:, :2], q[:, 2:])
    torch.cuda.synchronize()
    assert bool((out == 3.0).all()) and torch.equal(bt.dkc.cpu().nan_to_num(7.0), bt.kc.nan_to_num(7.0))


def test_two_graphs_share_a_workspace(gpu):
    """Two captured calls over one workspace, replayed in turn: nothing in it outlives a call."""
    scale, sets = 0.125, []
    bts = [Batch(71, CUT, 4, 1, 64, 32, "bf16"), Batch(72, [(1, 9000), (1, 30)], 4, 1, 64, 32, "bf16")]
    need = [gpu.attn_paged_workspace_bytes(bt.device(gpu), bt.T, 4, max(bt.new), 9000) for bt in bts]
    assert min(need) > 0
    ws = torch.full((max(need),), 255, dtype=torch.uint8, device="cuda")
    for bt in bts:
        q, out = bt.q.cuda(), torch.zeros((bt.T, 4, 64), dtype=DT["bf16"], device="cuda")
        call = lambda kv=bt.kv, q=q, out=out, bt=bt: gpu.op_attn_paged(kv, q, scale, out, max_new=max(bt.new), max_keys=9000, ws=ws)
        call()
        torch.cuda.synchronize()
        want = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        sets.append((bt, out, want, g, q))       # (a graph reads the q that it was captured with)
    for bt, out, want, _, _ in sets:
        ref, _, dout, _ = bt.attn(scale)
        assert np.all(np.abs(want.cpu().double().numpy() - ref) <= dout + rounding(np.abs(ref) + dout, "bf16"))
    for _ in range(3):
        for _, out, want, g, _ in sets:
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        for _, out, want, g, _ in sets:
            assert torch.equal(out, want)


def test_max_new_bounds_the_rows(gpu):
    """Rows past max_new are not computed and keep what they held."""
    bt = Batch(14, [(5, 40)], 2, 2, 32, 16, "f16")
    got, gl = _attn(gpu, bt, max_new=3, check=False)
    want = bt.attn(float(np.float32(1 / math.sqrt(32))))
    assert np.all(got[3:] == 77.0) and np.all(gl[3:] == 77.0)
    assert np.abs(got[:3] - want[0][:3]).max() < 1e-2


def test_offsets_past_32_bits(gpu):
    """Pages whose elements lie past 2^32 elements of the cache."""
    hd, nkv, page = 128, 8, 256
    n_pages = (1 << 32) // (nkv * page * hd) + 40      # 17.3 GB of K and as much of V
    bt = Batch(15, [(1, 700), (70, 600)], 8, 8, hd, page, "f16", spare=1)
    kc = torch.empty((n_pages, nkv, page, hd), dtype=DT["f16"], device="cuda")
    vc = torch.empty_like(kc)
    far = n_pages - bt.n_pages
    kc[far:], vc[far:] = bt.kc.cuda(), bt.vc.cuda()
    table = torch.from_numpy(np.where(bt.table >= 0, bt.table + far, -1).astype(np.int32)).cuda()
    kv = gpu.PagedKV(kc, vc, table, torch.from_numpy(bt.seq_start).cuda(), torch.from_numpy(bt.kv_len).cuda())
    out = torch.full((bt.tokens, 8, hd), 77.0, dtype=DT["f16"], device="cuda")
    lse = torch.full((bt.tokens, 8), 77.0, device="cuda")
    scale = float(np.float32(1 / math.sqrt(hd)))
    gpu.op_attn_paged(kv, bt.q.cuda(), scale, out, max_new=70, lse=lse)
    k = torch.randn((bt.T, 8 * hd), device="cuda")
    gpu.op_paged_append(kv, k, k * 2)
    torch.cuda.synchronize()
    _compare(bt, out.cpu().double().numpy(), lse.cpu().double().numpy(), bt.attn(scale), "f16")
    pg, off = int(table[1, 599 // page]), 599 % page
    assert torch.equal(kc[pg, :, off], k[bt.T - 1].view(8, hd).half()) and torch.equal(vc[pg, :, off], (2 * k[bt.T - 1]).view(8, hd).half())


# ---- append -----------------------------------------------------------------------------------

def _append_case(gpu, seed, lens, nh, nkv, hd, page, t, x, rot, pairs, pos=None, tables=None, tail=0, packed=True, edit=None):
    bt = Batch(seed, lens, nh, nkv, hd, page, t, stale=3.0, tail=tail)
    if edit:
        edit(bt)
    rng = np.random.default_rng(seed + 1)
    w = (nh + 2 * nkv) * hd
    qkv = torch.from_numpy((rng.standard_normal((bt.tokens, w)) * 3).astype(np.float32)).to(DT[x])
    kv = bt.device(gpu)
    d = qkv.cuda()
    q, k, v = d[:, :nh * hd], d[:, nh * hd:(nh + nkv) * hd], d[:, (nh + nkv) * hd:]
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    q_out = torch.full((bt.tokens, nh, hd), 55.0, dtype=DT[t], device="cuda")
    cos = sin = None
    if rot:
        cos, sin = tables if tables is not None else rope_tables(max(tot for _, tot in lens) + 1, rot)
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    gpu.op_paged_append(kv, k, v, q=q if nh else None, q_out=q_out if nh else None,
                        cos=None if cos is None else cos.cuda(), sin=None if sin is None else sin.cuda(), pairs=pairs,
                        pos=None if pos is None else torch.tensor(pos, dtype=torch.int32, device="cuda"), n_bad=bad)
    torch.cuda.synchronize()
    X = qkv.double().numpy().reshape(bt.tokens, nh + 2 * nkv, hd)
    ek, ev = bt.kc.double().numpy(), bt.vc.double().numpy()
    dk, dq = np.zeros_like(ek), np.zeros((bt.tokens, nh, hd))
    eq = np.full((bt.tokens, nh, hd), 55.0)
    nbad = 0
    for b in range(bt.B):
        for i in range(bt.new[b]):
            r = int(bt.seq_start[b]) + i
            slot = int(bt.kv_len[b]) - bt.new[b] + i
            p = slot if pos is None else pos[r]
            pg = int(bt.table[b, slot // page]) if 0 <= slot < bt.cols * page else -1
            if not 0 <= pg < bt.n_pages or (rot and not 0 <= p < cos.shape[0]):
                nbad += 1
                continue
            x, dx = X[r:r + 1, :nh + nkv], np.zeros((1, nh + nkv, hd))
            if rot:
                x, dx = rotate(x, cos, sin, np.array([p]), pairs)
            eq[r], dq[r] = x[0, :nh], dx[0, :nh]
            ek[pg, :, slot % page], dk[pg, :, slot % page] = x[0, nh:], dx[0, nh:]
            ev[pg, :, slot % page] = X[r, nh + nkv:]
    gk, gv, gq = (z.cpu().double().numpy() for z in (bt.dkc, bt.dvc, q_out))
    assert np.all(np.abs(gk - ek) <= dk + rounding(np.abs(ek) + dk, t))
    assert np.all(np.abs(gv - ev) <= rounding(ev, t))
    assert np.all(np.abs(gq - eq) <= dq + rounding(np.abs(eq) + dq, t))
    untouched = (dk == 0) & (ek == 3.0)
    assert np.all(gk[untouched] == 3.0)
    assert int(bad.item()) == nbad
    return bt, gk, gv, gq


@pytest.mark.parametrize("t,x", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("hd,rot", [(32, 32), (32, 16), (64, 64), (64, 0), (128, 128), (128, 64), (128, 48)])
@pytest.mark.parametrize("pairs", [False, True])
def test_append(gpu, hd, rot, pairs, t, x):
    _append_case(gpu, hd + rot, FORMS["mixed"], 6, 2, hd, 16, t, x, rot, pairs, tail=3)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("page", [16, 64])
def test_append_forms(gpu, form, page):
    _append_case(gpu, page, FORMS[form], 3, 1, 64, page, "f16", "f32", 64, True, packed=form != "chunk")


def test_append_keys_and_values_only(gpu):
    _append_case(gpu, 1, FORMS["mixed"], 0, 2, 32, 16, "f16", "f32", 0, False)


def test_append_positions_of_their_own(gpu):
    """Positions apart from the key index, some outside the tables: those rows are not written."""
    lens = [(5, 20), (3, 9)]
    _append_case(gpu, 2, lens, 2, 2, 64, 16, "bf16", "bf16", 64, False, pos=[0, 7, 7, 39, 40, -1, 3, 2 ** 31 - 1],
                 tables=rope_tables(40, 64, seed=4))


def test_append_rows_without_a_page(gpu):
    def edit(bt):
        bt.table[0, 1] = -1
        bt.table[1, 0] = bt.n_pages
        bt.kv_len[2] = 2          # more new rows than keys: the first ones have a negative index
        bt.kv_len[3] = 400        # past the table
    _append_case(gpu, 3, [(20, 40), (4, 4), (5, 5), (6, 6)], 2, 2, 32, 16, "f16", "f16", 32, False, edit=edit,
                 tables=rope_tables(500, 32))


def test_append_in_place(gpu):
    """q_out may be q itself."""
    bt = Batch(21, FORMS["mixed"], 4, 2, 64, 16, "f16")
    kv = bt.device(gpu)
    cos, sin = (z.cuda() for z in rope_tables(400, 64))
    k = torch.randn((bt.T, 2 * 64), device="cuda").half()
    for pairs in (False, True):
        q = bt.q.cuda()
        out = torch.empty_like(q)
        gpu.op_paged_append(kv, k, k, q=q, q_out=out, cos=cos, sin=sin, pairs=pairs)
        gpu.op_paged_append(kv, k, k, q=q, q_out=q, cos=cos, sin=sin, pairs=pairs)
        torch.cuda.synchronize()
        assert torch.equal(q, out)


# ---- the two together ---------------------------------------------------------------------------

@pytest.mark.parametrize("hd,nh,nkv,t,pairs", [(32, 4, 4, "f16", True), (128, 6, 2, "bf16", False)])
def test_steps_of_a_server(gpu, hd, nh, nkv, t, pairs):
    """Prompts in chunks of uneven length, then single tokens, sequences joining on the way: every step
    appends and attends; the outputs are those of attention over the rotated history in 64 bits."""
    rng = np.random.default_rng(31)
    page, B = 16, 3
    steps = [[37, 0, 0], [20, 5, 0], [1, 70, 0], [1, 1, 33], [1, 1, 1], [1, 1, 40], [0, 1, 1]]
    total = np.sum(steps, 0)
    cols = -(-int(total.max()) // page)
    kc = torch.full((B * cols, nkv, page, hd), float("nan"), dtype=DT[t], device="cuda")
    vc = torch.full_like(kc, float("nan"))
    table = torch.from_numpy(rng.permutation(B * cols).reshape(B, cols).astype(np.int32)).cuda()
    dss = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    dlen = torch.zeros(B, dtype=torch.int32, device="cuda")
    kv = gpu.PagedKV(kc, vc, table, dss, dlen)
    cos, sin = rope_tables(400, hd)
    scale = float(np.float32(1 / math.sqrt(hd)))
    K = [np.zeros((0, nkv, hd)) for _ in range(B)]
    V = [np.zeros((0, nkv, hd)) for _ in range(B)]
    have = np.zeros(B, int)
    for new in steps:
        T = sum(new)
        have += new
        dss.copy_(torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)))
        dlen.copy_(torch.from_numpy(have.astype(np.int32)))
        qkv = torch.from_numpy(rng.standard_normal((T, (nh + 2 * nkv) * hd)).astype(np.float32))
        d = qkv.cuda()
        q = torch.empty((T, nh, hd), dtype=DT[t], device="cuda")
        gpu.op_paged_append(kv, d[:, nh * hd:(nh + nkv) * hd], d[:, (nh + nkv) * hd:], q=d[:, :nh * hd], q_out=q,
                            cos=cos.cuda(), sin=sin.cuda(), pairs=pairs)
        out = torch.empty((T, nh, hd), device="cuda")
        gpu.op_attn_paged(kv, q, scale, out, max_new=max(new), max_keys=int(have.max()))
        torch.cuda.synchronize()
        got = out.cpu().double().numpy()
        X = qkv.double().numpy().reshape(T, nh + 2 * nkv, hd)
        r = 0
        for b in range(B):
            pos = np.arange(have[b] - new[b], have[b])
            y, _ = rotate(X[r:r + new[b], :nh + nkv], cos, sin, pos, pairs)
            K[b] = np.concatenate([K[b], y[:, nh:]])
            V[b] = np.concatenate([V[b], X[r:r + new[b], nh + nkv:]])
            for i in range(new[b]):
                n = pos[i] + 1
                for h in range(nh):
                    s = K[b][:n, h // (nh // nkv)] @ y[i, h] * scale
                    e = np.exp(s - s.max())
                    p = e / e.sum()
                    ref = p @ V[b][:n, h // (nh // nkv)]
                    # q and k are each rounded once (the score's error), v and the probabilities too
                    mag = (np.abs(K[b][:n, h // (nh // nkv)]) @ np.abs(y[i, h])).max() * scale
                    tol = (p @ np.abs(V[b][:n, h // (nh // nkv)])) * (2 * U[t] + 2 * 2.1 * U[t] * mag + 1e-4)
                    assert np.all(np.abs(got[r + i, h] - ref) <= tol + 1e-6)
            r += new[b]


@pytest.mark.parametrize("lens", [[(1, 3000), (1, 50)], [(90, 200), (1, 2000), (0, 5)]])
def test_graph_replays_follow_the_batch(gpu, lens):
    """One captured step (append, attention), replayed while lengths, tables and inputs change and other
    work runs in between, equals the eager calls to the bit every time."""
    hd, nh, nkv, page = 64, 4, 2, 16
    bt = Batch(41, lens, nh, nkv, hd, page, "f16", stale=0.25, cols=200, tail=5)
    kv = bt.device(gpu)
    scale = 0.125
    cos, sin = (z.cuda() for z in rope_tables(3300, hd))
    qkv = torch.randn((bt.tokens, (nh + 2 * nkv) * hd), device="cuda")
    q = torch.zeros((bt.tokens, nh, hd), dtype=DT["f16"], device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros((bt.tokens, nh), device="cuda")
    max_new = max(bt.new)
    ws = torch.empty(max(16, gpu.attn_paged_workspace_bytes(kv, bt.tokens, nh, max_new, 3200)), dtype=torch.uint8, device="cuda")

    def step():
        gpu.op_paged_append(kv, qkv[:, nh * hd:(nh + nkv) * hd], qkv[:, (nh + nkv) * hd:], q=qkv[:, :nh * hd], q_out=q,
                            cos=cos, sin=sin)
        gpu.op_attn_paged(kv, q, scale, out, max_new=max_new, max_keys=3200, lse=lse, ws=ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for k in range(4):
        qkv.normal_()
        bt.dlen.copy_(torch.tensor([max(n, tot - 37 * k) for n, tot in lens], dtype=torch.int32))
        if k == 2:
            bt.dtable.copy_(bt.dtable[:, torch.randperm(bt.cols, device="cuda")])
        kc, vc = bt.dkc.clone(), bt.dvc.clone()
        for z in (q, out, lse):
            z.fill_(9.0)                # (rows whose table entry is no page keep this)
        step()
        want = [z.clone() for z in (q, out, lse, bt.dkc, bt.dvc)]
        bt.dkc.copy_(kc)
        bt.dvc.copy_(vc)
        for z in (q, out, lse):
            z.fill_(9.0)
        rest = [z[bt.T:].clone() for z in (q, out, lse)]
        ws.fill_(255)                   # another user of the workspace
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for have, w in zip((q, out, lse, bt.dkc, bt.dvc), want):
            n = bt.T if have.shape[0] == bt.tokens else have.shape[0]
            assert torch.equal(have[:n], w[:n])
        for z, w in zip((q, out, lse), rest):
            assert torch.equal(z[bt.T:], w)
        _say("replay", k)


def test_another_stream(gpu):
    """The calls run on the stream that they are given, two streams at once with a workspace each."""
    scale = 0.125
    sets = []
    for s in range(2):
        bt = Batch(51 + s, [(1, 4000), (3, 900)], 8, 2, 64, 32, "bf16")
        kv = bt.device(gpu)
        out = torch.zeros((bt.T, 8, 64), dtype=DT["bf16"], device="cuda")
        ws = torch.empty(max(16, gpu.attn_paged_workspace_bytes(kv, bt.T, 8, 3, 4000)), dtype=torch.uint8, device="cuda")
        sets.append((bt, kv, bt.q.cuda(), out, ws, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(3):
        for bt, kv, q, out, ws, st in sets:
            gpu.op_attn_paged(kv, q, scale, out, max_new=3, max_keys=4000, ws=ws, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for bt, kv, q, out, ws, st in sets:
        ref, _, dout, _ = bt.attn(scale)
        assert np.all(np.abs(out.cpu().double().numpy() - ref) <= dout + rounding(np.abs(ref) + dout, "bf16"))
    bt, kv, q, out, ws, st = sets[0]
    with pytest.raises(ValueError):      # a workspace of torch's current stream on another one
        gpu.op_attn_paged(kv, q, scale, out, max_new=3, max_keys=4000, stream=st.cuda_stream)


def test_wrong_tensors_are_refused(gpu):
    bt = Batch(61, FORMS["draft"], 4, 2, 64, 16, "f16")
    kv = bt.device(gpu)
    q = bt.q.cuda()
    out = torch.empty_like(q)
    k = torch.zeros((bt.T, 128), dtype=DT["f16"], device="cuda")
    bad = [lambda: gpu.op_attn_paged(kv, q.float(), 0.1, out, 7), lambda: gpu.op_attn_paged(kv, q, 0.1, out[:, :2], 7),
           lambda: gpu.op_attn_paged(kv, q.transpose(0, 1), 0.1, out.transpose(0, 1), 7),
           lambda: gpu.op_attn_paged(kv, bt.q, 0.1, out, 7), lambda: gpu.op_attn_paged(kv, q, 0.1, out.double(), 7),
           lambda: gpu.op_attn_paged(kv, q, 0.1, out, 7, lse=torch.zeros(3, 4, device="cuda")),
           lambda: gpu.op_attn_paged(kv, q, 0.1, out, 7, prefix=torch.zeros(4, dtype=torch.int32, device="cuda")),
           lambda: gpu.op_paged_append(kv, k, k.float()), lambda: gpu.op_paged_append(kv, k[:, :64], k[:, :64]),
           lambda: gpu.op_paged_append(kv, k, k[:3]), lambda: gpu.op_paged_append(kv, k, k, q=q),
           lambda: gpu.op_paged_append(kv, k, k, q=q, q_out=out.float()),
           lambda: gpu.op_paged_append(kv, k, k, sin=torch.zeros(9, 32, device="cuda")),
           lambda: gpu.PagedKV(bt.dkc, bt.dvc[:, :1], bt.dtable, bt.dss, bt.dlen),
           lambda: gpu.PagedKV(bt.dkc.transpose(1, 2), bt.dvc.transpose(1, 2), bt.dtable, bt.dss, bt.dlen),
           lambda: gpu.PagedKV(bt.dkc, bt.dvc, bt.dtable.long(), bt.dss, bt.dlen),
           lambda: gpu.PagedKV(bt.dkc, bt.dvc, bt.dtable, bt.dss[:-1], bt.dlen),
           lambda: gpu.PagedKV(bt.dkc, bt.dvc, bt.dtable.cpu(), bt.dss, bt.dlen)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, gpu.GsvkError)):
            f()
            _say("not refused:", i)
