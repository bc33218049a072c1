"""Draft-tree attention, attention weight, cache eviction and path commit (include/jinf/kv_ops.h)
on the GPU against their plain 64-bit forms (kv_ops_ref.py).

Tolerances, u the unit roundoff of the 16-bit type (2^-11 fp16, 2^-8 bf16):
  out   the result is rounded once, u |out|; each probability once before it meets v, u sum p |v|, or
        2^-25 absolutely where fp16 is subnormal (relative to the largest, so over sum e^(s - m));
        the fp32 scores' dot of up to 128 products is off by at most 128 2^-24 sum |q k| scale, which is
        below 1e-4 for these inputs and moves every p by that share;
  lse   the same 1e-4, and a few 2^-24 of its own size;
  mass  1e-4 of what is added, from the scores, and 2^-22 of the sum."""
import math

import pytest
import torch

import kv_ops_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_cache(g, S, nkv, ctx, hd, dtype, layout="shrd", fill=None):
    """K, V as [S, nkv, ctx, hd] views; layout: order of the axes seq, head, row in memory."""
    dims = {"s": S, "h": nkv, "r": ctx}
    order = [c for c in layout if c != "d"]
    out = []
    for _ in range(2):
        t = torch.randn(*[dims[c] for c in order], hd, generator=g, device="cuda", dtype=dtype)
        if fill is not None:
            t.fill_(fill)
        out.append(t.permute(*[order.index(c) for c in "shr"], 3))
    return out


def random_parents(seed, nodes):
    g = torch.Generator()
    g.manual_seed(seed)
    u = torch.rand(nodes, generator=g).tolist()
    return [-1] + [int(t * u[t]) - (1 if u[t] < 0.2 else 0) for t in range(1, nodes)]


def attend(q, k, v, n_past, max_past, mask=None, scale=None, stream=None, want_lse=True):
    from jinf import kernels as K
    kv = K.KvView(k, v)
    S, T, H, hd = q.shape
    out = torch.full((S, T, H, hd), math.nan, dtype=q.dtype, device="cuda")
    lse = torch.full((S, T, H), math.nan, device="cuda") if want_lse else None
    ws = torch.zeros(K.tree_attention_workspace_bytes(kv, H, T, max_past), dtype=torch.uint8, device="cuda")
    for _ in range(2):  # the workspace survives back-to-back calls
        K.tree_attention(out, q, kv, n_past, max_past, ws, mask=mask, lse=lse, scale=scale, stream=stream)
    return out, lse


def check_attention(q, k, v, n_past, out, lse, masks, scale):
    want, wl, mag, flat = ref.attention(q, k, v, n_past.tolist(), masks, scale)
    u = ref.UNIT[q.dtype]
    tol = u * (want.abs() + mag) + 2e-4 * mag + (2.0 ** -25 * flat + 2.0 ** -25 if q.dtype == F16 else 0.0)
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    if lse is not None:
        assert torch.equal(lse == -math.inf, wl == -math.inf)
        fin = wl > -math.inf
        assert bool(((lse.double() - wl).abs()[fin] <= 1e-4 + 2.0 ** -21 * wl.abs()[fin]).all())


# (dtype, head_dim, heads, kv heads, nodes, lengths): one and several rows per warp tile and CTA, lengths
# around the key tiles' edges, zero and one, group sizes 1 to 16, one sequence and several ragged ones
SHAPES = [
    (F16, 64, 8, 2, 1, [0]),
    (F16, 64, 8, 2, 5, [37]),
    (F16, 128, 8, 2, 1, [1, 0, 127, 128, 129]),
    (BF16, 128, 4, 4, 3, [255, 13]),
    (BF16, 64, 16, 1, 2, [640]),
    (F16, 128, 32, 8, 26, [1001]),
    (BF16, 128, 16, 2, 33, [126, 700]),
    (F16, 128, 8, 1, 17, [2049]),
    (F16, 64, 12, 4, 64, [250]),
    (BF16, 128, 8, 2, 64, [1, 513]),
    (F16, 128, 2, 2, 256, [300]),
    (BF16, 64, 4, 2, 129, [0, 90]),
    (F16, 128, 4, 1, 100, [1500]),
]


@pytest.mark.parametrize("dtype,hd,nh,nkv,nodes,lengths", SHAPES)
@pytest.mark.parametrize("tree", [True, False])
def test_tree_attention(cuda, dtype, hd, nh, nkv, nodes, lengths, tree):
    from jinf import kernels as K
    g = gen(nodes + hd)
    S, mp = len(lengths), max(lengths)
    k, v = make_cache(g, S, nkv, mp + nodes + 3, hd, dtype)
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=dtype)
    n_past = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mask = K.tree_mask(random_parents(nodes, nodes)).cuda() if tree else None
    out, lse = attend(q, k, v, n_past, mp, mask)
    check_attention(q, k, v, n_past, out, lse, [mask] * S, hd ** -0.5)


@pytest.mark.parametrize("layout", ["shrd", "srhd", "rshd", "hsrd"])
@pytest.mark.parametrize("nodes", [3, 70])
def test_tree_attention_strides_masks_and_scale(cuda, layout, nodes):
    """Every axis order, q as part of a wider row, a mask per sequence, a scale of its own, no lse, and a
    bound on the lengths above the lengths themselves."""
    from jinf import kernels as K
    S, nkv, nh, hd, lengths = 3, 2, 6, 128, [200, 31, 130]
    g = gen(5)
    k, v = make_cache(g, S, nkv, 400, hd, F16, layout)
    wide = torch.randn(S, nodes, nh * hd + 64, generator=g, device="cuda", dtype=F16)
    q = wide[:, :, :nh * hd].view(S, nodes, nh, hd)
    n_past = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mask = torch.stack([K.tree_mask(random_parents(s, nodes)) for s in range(S)]).cuda()
    out, _ = attend(q, k, v, n_past, 300, mask, scale=0.21, want_lse=False)
    check_attention(q, k, v, n_past, out, None, list(mask), 0.21)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nh", [4, 40])
def test_tree_attention_ignores_what_masked_and_unused_rows_hold(cuda, dtype, bad, nh):
    """Rows behind the tree, and rows a node does not see, may hold anything; a row it sees counts."""
    S, nkv, hd, nodes, past = 2, 2, 64, 7, 59
    g = gen(9)
    k, v = make_cache(g, S, nkv, 200, hd, dtype)
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=dtype)
    n_past = torch.tensor([past, past - 40], dtype=torch.int32, device="cuda")
    words = torch.zeros(nodes, 1, dtype=torch.int32)
    for t in range(nodes):
        words[t, 0] = (1 << t) if t != 4 else 0b10011  # node 4 sees 0 and 1 as well
    words[2, 0] = 0  # nothing of the tree
    mask = words.cuda()
    clean, lse0 = attend(q, k, v, n_past, past, mask)
    for s, n in enumerate(n_past.tolist()):
        k[s, :, n + nodes:], v[s, :, n + nodes:] = bad, bad
        k[s, :, n + 6], v[s, :, n + 6] = bad, bad        # only node 6 sees it
        v[s, :, n + 1, 5] = bad                          # nodes 1 and 4 see it, in one column
    out, lse = attend(q, k, v, n_past, past, mask)
    assert torch.equal(out[:, [0, 2, 3, 5]], clean[:, [0, 2, 3, 5]])
    assert torch.equal(lse[:, :6], lse0[:, :6])
    cols = [c for c in range(hd) if c != 5]
    assert torch.equal(out[:, [1, 4]][..., cols], clean[:, [1, 4]][..., cols])
    hit = out[:, [1, 4], :, 5]
    assert bool(torch.isnan(hit).all()) if math.isnan(bad) else bool((hit == bad).all())
    assert not bool(torch.isfinite(out[:, 6]).all())


def test_tree_attention_empty_rows(cuda):
    """No cached row and an empty mask: out 0, lse -inf; the other nodes are not affected."""
    g = gen(3)
    k, v = make_cache(g, 1, 2, 40, 128, F16)
    q = torch.randn(1, 4, 4, 128, generator=g, device="cuda", dtype=F16)
    n_past = torch.zeros(1, dtype=torch.int32, device="cuda")
    mask = torch.tensor([[1], [0], [5], [0]], dtype=torch.int32, device="cuda")
    out, lse = attend(q, k, v, n_past, 0, mask)
    assert bool((out[0, [1, 3]] == 0).all()) and bool((lse[0, [1, 3]] == -math.inf).all())
    check_attention(q, k, v, n_past, out, lse, [mask], 128 ** -0.5)


@pytest.mark.parametrize("nodes,nh", [(1, 4), (40, 4), (40, 16)])
def test_tree_attention_large_and_peaked_scores(cuda, nodes, nh):
    """Scores in the hundreds, growing along the cache, so that the running maximum moves all the time."""
    g = gen(4)
    k, v = make_cache(g, 1, 2, 900, 128, BF16)
    k.mul_(torch.linspace(0.5, 12, 900, device="cuda").to(BF16)[None, None, :, None])
    q = torch.randn(1, nodes, nh, 128, generator=g, device="cuda", dtype=BF16) * 4
    n_past = torch.tensor([850], dtype=torch.int32, device="cuda")
    out, lse = attend(q, k, v, n_past, 850)
    want, wl, mag, _ = ref.attention(q, k, v, [850], [None], 128 ** -0.5)
    # scores of a few hundred: 128 2^-24 sum |q k| scale is up to 4e-3 here, and moves p by that share
    assert bool(((lse.double() - wl).abs() <= 4e-3).all())
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * (want.abs() + mag) + 8e-3 * mag).all())


def test_tree_attention_clamps_lengths(cuda):
    """Device lengths outside 0..max_past are taken as the nearest bound."""
    g = gen(8)
    k, v = make_cache(g, 2, 1, 150, 64, F16)
    q = torch.randn(2, 2, 4, 64, generator=g, device="cuda", dtype=F16)
    got, _ = attend(q, k, v, torch.tensor([-5, 10 ** 6], dtype=torch.int32, device="cuda"), 140)
    want, _ = attend(q, k, v, torch.tensor([0, 140], dtype=torch.int32, device="cuda"), 140)
    assert torch.equal(got, want)


def test_offsets_past_32_bits(cuda):
    """Sequences 2^31 elements apart: attention, mass, eviction and commit of the second one."""
    from jinf import kernels as K
    far, ctx, hd, nkv, nodes, past = (1 << 31) + 64, 64, 64, 2, 3, 50
    g = gen(12)
    store = [torch.empty(far + nkv * ctx * hd, dtype=F16, device="cuda") for _ in range(2)]
    k, v = (t.as_strided((2, nkv, ctx, hd), (far, ctx * hd, hd, 1)) for t in store)
    for t in (k, v):
        t.copy_(torch.randn(2, nkv, ctx, hd, generator=g, device="cuda", dtype=F16))
    q = torch.randn(2, nodes, 4, hd, generator=g, device="cuda", dtype=F16)
    n_past = torch.tensor([past, past], dtype=torch.int32, device="cuda")
    out, lse = attend(q, k, v, n_past, past)
    check_attention(q, k, v, n_past, out, lse, [None, None], hd ** -0.5)
    kv = K.KvView(k, v)
    m = torch.rand(2, nkv, ctx, generator=g, device="cuda")
    want, add = ref.mass(m, q, k, [past, past], [None, None], lse, None, hd ** -0.5)
    K.attention_mass(m, q, kv, n_past, past, lse)
    assert bool(((m.double() - want).abs() <= 1e-4 * add + 2.0 ** -22 * want.abs()).all())
    k0, v0, m0 = k.clone(), v.clone(), m.clone()
    acc = torch.tensor([[1, 2], [0, 2]], dtype=torch.int32, device="cuda")
    K.tree_commit(kv, m, n_past, past, acc, torch.tensor([2, 2], dtype=torch.int32, device="cuda"), nodes)
    assert torch.equal(k[1, :, past + 1], k0[1, :, past + 2]) and torch.equal(v[0, :, past], v0[0, :, past + 1])
    ids = torch.empty(2, nkv, 10, dtype=torch.int32, device="cuda")
    k0, v0, m0 = k.clone(), v.clone(), m.clone()
    K.kv_evict(kv, None, m, m, torch.tensor([52, 52], dtype=torch.int32, device="cuda"), ids, None, 10, 1, 2)
    for s in range(2):
        for h in range(nkv):
            want_ids = ref.evict_ids(m0[s, h].tolist(), 52, 10, 1, 2)
            assert ids[s, h].tolist() == want_ids
            assert torch.equal(k[s, h, :10], k0[s, h, want_ids]) and torch.equal(v[s, h, :10], v0[s, h, want_ids])


@pytest.mark.parametrize("dtype,hd,nh,nkv,nodes,lengths", SHAPES)
@pytest.mark.parametrize("weighted", [True, False])
def test_attention_mass(cuda, dtype, hd, nh, nkv, nodes, lengths, weighted):
    from jinf import kernels as K
    g = gen(nodes * 3 + hd)
    S, mp = len(lengths), max(lengths)
    ctx = mp + nodes + 3
    k, v = make_cache(g, S, nkv, ctx, hd, dtype, "srhd" if weighted else "shrd")
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=dtype)
    n_past = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mask = K.tree_mask(random_parents(nodes, nodes)).cuda() if weighted else None
    _, lse = attend(q, k, v, n_past, mp, mask)
    weight = None
    if weighted:  # some nodes, one of them by half
        weight = (torch.rand(S, nodes, generator=g, device="cuda") < 0.4).float()
        weight[:, 0] = 0.5
    m = torch.rand(S, nkv, ctx, generator=g, device="cuda")
    m[0, 0, lengths[0]] = math.nan  # the tree's rows are set, whatever they held
    before = m.clone()
    want, add = ref.mass(before, q, k, lengths, [mask] * S, lse, weight, hd ** -0.5)
    K.attention_mass(m, q, K.KvView(k, v), n_past, mp, lse, mask=mask, node_weight=weight)
    assert bool(((m.double() - want).abs() <= 1e-4 * add + 2.0 ** -22 * want.abs()).all())
    for s in range(S):  # rows behind the tree are not touched
        assert torch.equal(m[s, :, lengths[s] + nodes:], before[s, :, lengths[s] + nodes:])
    again = before.clone()
    K.attention_mass(again, q, K.KvView(k, v), n_past, mp, lse, mask=mask, node_weight=weight)
    assert torch.equal(again.nan_to_num(7.0), m.nan_to_num(7.0))


@pytest.mark.parametrize("nodes", [4, 90])
def test_attention_mass_ignores_rejected_nodes_empty_rows_and_masked_keys(cuda, nodes):
    from jinf import kernels as K
    g = gen(21)
    S, nkv, nh, hd, past = 1, 2, 8, 128, 140
    k, v = make_cache(g, S, nkv, 300, hd, F16)
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=F16)
    n_past = torch.tensor([past], dtype=torch.int32, device="cuda")
    words = (nodes + 31) // 32
    mask = torch.zeros(nodes, words, dtype=torch.int32)
    for t in range(nodes):
        mask[t, t // 32] = -(1 << 31) if t % 32 == 31 else 1 << (t % 32)
    mask = mask.cuda()
    _, lse = attend(q, k, v, n_past, past, mask)
    weight = torch.ones(S, nodes, device="cuda")
    weight[0, 1], weight[0, 3] = 0.0, 0.0
    m = torch.zeros(S, nkv, 300, device="cuda")
    want, add = ref.mass(m, q, k, [past], [mask], lse, weight, hd ** -0.5)
    q[0, 1], lse[0, 3] = math.nan, math.nan       # rejected
    k[0, :, past + 1] = math.nan                  # seen by a rejected node only
    k[0, :, past + nodes:] = math.inf             # unused
    K.attention_mass(m, q, K.KvView(k, v), n_past, past, lse, mask=mask, node_weight=weight)
    assert bool(((m.double() - want).abs() <= 1e-4 * add + 2.0 ** -22 * want.abs()).all())
    assert bool((m[0, :, past + 1] == 0).all())
    # no accepted node at all, and a row that attended nothing
    m1 = m.clone()
    K.attention_mass(m1, q, K.KvView(k, v), n_past, past, lse, mask=mask, node_weight=torch.zeros_like(weight))
    assert torch.equal(m1[:, :, :past], m[:, :, :past]) and bool((m1[:, :, past:past + nodes] == 0).all())
    lse.fill_(-math.inf)
    m2 = m.clone()
    K.attention_mass(m2, q, K.KvView(k, v), n_past, past, lse, mask=mask, node_weight=weight)
    assert torch.equal(m2[:, :, :past], m[:, :, :past])


EVICT = [  # (dtype, hd, kv heads, lengths, ctx, keep, sink, recent)
    (F16, 64, 2, [200], 256, 64, 4, 16),
    (BF16, 128, 3, [1000, 64, 0, 63, 65], 1000, 64, 1, 0),
    (F16, 128, 1, [5000], 5003, 4999, 4, 1000),
    (BF16, 64, 2, [3000, 2999], 3100, 700, 0, 700),
    (F16, 128, 8, [2048], 2048, 1, 0, 0),
    (F16, 128, 2, [40000], 40000, 3001, 4, 256),
    (F16, 64, 1, [140001], 140001, 1025, 0, 1),
    (F16, 64, 1, [400000, 1000, 70000], 400000, 990, 3, 5),  # slices too long for shared memory, and short ones
    (BF16, 64, 3, [16384, 16385, 1], 16385, 4000, 100, 0),
]


@pytest.mark.parametrize("dtype,hd,nkv,lengths,ctx,keep,sink,recent", EVICT)
@pytest.mark.parametrize("in_place", [False, True])
def test_kv_evict(cuda, dtype, hd, nkv, lengths, ctx, keep, sink, recent, in_place):
    from jinf import kernels as K
    S = len(lengths)
    g = gen(keep)
    k, v = make_cache(g, S, nkv, ctx, hd, dtype, "srhd" if in_place else "shrd")
    m = torch.rand(S, nkv, ctx, generator=g, device="cuda") ** 3
    m[:, :, ::3] = torch.round(m[:, :, ::3] * 8) / 8  # many equal ones, zeros among them
    m[:, :, 5::11] = math.nan
    m[:, :, 7::13] *= -1.0
    m[:, :, 3::17] = -0.0
    m[:, 0, 2::501] = math.inf
    k0, v0, m0 = k.clone(), v.clone(), m.clone()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    ids = torch.empty(S, nkv, keep, dtype=torch.int32, device="cuda")
    n_out = torch.empty(S, dtype=torch.int32, device="cuda")
    if in_place:
        ko, vo, mo = k, v, m
        K.kv_evict(K.KvView(k, v), None, m, m, n, ids, n_out, keep, sink, recent)
    else:
        ko, vo = make_cache(g, S, nkv, keep + 5, hd, dtype, "hsrd", fill=7.0)
        mo = torch.full((S, nkv, keep + 5), 7.0, device="cuda")
        K.kv_evict(K.KvView(k, v), K.KvView(ko, vo), m, mo, n, ids, n_out, keep, sink, recent)
        assert torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(m.isnan(), m0.isnan())
    assert n_out.tolist() == [min(x, keep) for x in lengths]
    for s in range(S):
        for h in range(nkv):
            want = ref.evict_ids(m0[s, h].tolist(), lengths[s], keep, sink, recent)
            c = len(want)
            assert ids[s, h].tolist() == want + [-1] * (keep - c)
            assert torch.equal(ko[s, h, :c], k0[s, h, want]) and torch.equal(vo[s, h, :c], v0[s, h, want])
            assert torch.equal(mo[s, h, :c].nan_to_num(9e9), m0[s, h, want].nan_to_num(9e9))
            if not in_place:
                assert bool((ko[s, h, c:] == 7).all()) and bool((mo[s, h, c:] == 7).all())
            else:
                assert torch.equal(ko[s, h, keep:], k0[s, h, keep:])


@pytest.mark.parametrize("dtype,hd,layout", [(F16, 128, "shrd"), (BF16, 64, "srhd")])
@pytest.mark.parametrize("with_mass", [True, False])
def test_tree_commit(cuda, dtype, hd, layout, with_mass):
    from jinf import kernels as K
    S, nkv, nodes, ctx = 5, 3, 40, 200
    g = gen(hd)
    k, v = make_cache(g, S, nkv, ctx, hd, dtype, layout)
    m = torch.rand(S, nkv, ctx, generator=g, device="cuda")
    k0, v0, m0 = k.clone(), v.clone(), m.clone()
    past = [0, 1, 100, 160, 33]
    paths = [[0], [], [0, 2, 3, 9, 11, 12, 20, 21, 22, 30, 31, 38, 39], list(range(40)), [39]]
    acc = torch.full((S, 41), 77, dtype=torch.int32)
    for s, p in enumerate(paths):
        acc[s, :len(p)] = torch.tensor(p, dtype=torch.int32)
    n_out = torch.empty(S, dtype=torch.int32, device="cuda")
    K.tree_commit(K.KvView(k, v), m if with_mass else None, torch.tensor(past, dtype=torch.int32, device="cuda"), 160,
                  acc.cuda(), torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda"), nodes, n_out)
    assert n_out.tolist() == [a + len(p) for a, p in zip(past, paths)]
    for s, p in enumerate(paths):
        rows = list(range(ctx))
        for i, node in enumerate(p):
            rows[past[s] + i] = past[s] + node
        assert torch.equal(k[s], k0[s][:, rows]) and torch.equal(v[s], v0[s][:, rows])
        assert torch.equal(m[s], m0[s][:, rows] if with_mass else m0[s])


def test_tree_commit_skips_numbers_out_of_range(cuda):
    from jinf import kernels as K
    g = gen(2)
    k, v = make_cache(g, 1, 1, 20, 64, F16)
    k0 = k.clone()
    n_out = torch.empty(1, dtype=torch.int32, device="cuda")
    K.tree_commit(K.KvView(k, v), None, torch.tensor([15], dtype=torch.int32, device="cuda"), 15,
                  torch.tensor([[1, 5, 2 ** 30, -7]], dtype=torch.int32, device="cuda"),
                  torch.tensor([99], dtype=torch.int32, device="cuda"), 4, n_out)
    assert torch.equal(k[0, 0, 15], k0[0, 0, 16]) and torch.equal(k[0, 0, 16:], k0[0, 0, 16:])
    assert n_out.item() == 19


def test_operators_on_another_stream_and_in_a_graph(cuda):
    """One step of the four on a side stream, captured and replayed with new lengths on the device."""
    from jinf import kernels as K
    S, nkv, nh, hd, nodes, ctx = 2, 2, 8, 128, 9, 500
    g = gen(77)
    k, v = make_cache(g, S, nkv, ctx, hd, F16)
    kv = K.KvView(k, v)
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=F16)
    n_past = torch.tensor([300, 20], dtype=torch.int32, device="cuda")
    out, lse = torch.empty(S, nodes, nh, hd, dtype=F16, device="cuda"), torch.empty(S, nodes, nh, device="cuda")
    mass = torch.zeros(S, nkv, ctx, device="cuda")
    ws = torch.zeros(K.tree_attention_workspace_bytes(kv, nh, nodes, 400), dtype=torch.uint8, device="cuda")
    acc = torch.tensor([[0, 4, 7]] * S, dtype=torch.int32, device="cuda")
    n_acc = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    n_new, n_kept = (torch.empty(S, dtype=torch.int32, device="cuda") for _ in range(2))
    ids = torch.empty(S, nkv, 64, dtype=torch.int32, device="cuda")

    def step(stream):
        K.tree_attention(out, q, kv, n_past, 400, ws, lse=lse, stream=stream)
        K.attention_mass(mass, q, kv, n_past, 400, lse, stream=stream)
        K.tree_commit(kv, mass, n_past, 400, acc, n_acc, nodes, n_new, stream=stream)
        K.kv_evict(kv, None, mass, mass, n_new, ids, n_kept, 64, 2, 8, stream=stream)

    k0, v0 = k.clone(), v.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    step(side)
    side.synchronize()
    first = (out.clone(), lse.clone(), ids.clone())
    check_attention(q, k0, v0, n_past, out, lse, [None] * S, hd ** -0.5)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream())
    for lengths in ([300, 20], [5, 399]):
        k.copy_(k0), v.copy_(v0), mass.zero_(), n_past.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_attention(q, k0, v0, n_past, out, lse, [None] * S, hd ** -0.5)
        assert n_kept.tolist() == [min(64, lengths[0] + 3), min(64, lengths[1] + 2)]
        if lengths == [300, 20]:
            assert all(torch.equal(a, b) for a, b in zip(first, (out, lse, ids)))


def test_wrappers_refuse_what_does_not_fit(cuda):
    from jinf import kernels as K
    from jinf import JinfError
    g = gen(1)
    k, v = make_cache(g, 2, 2, 50, 64, F16)
    kv = K.KvView(k, v)
    q = torch.zeros(2, 3, 4, 64, dtype=F16, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(2, 3, 4, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    ws = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError):
        K.KvView(k, v.to(BF16))
    with pytest.raises(ValueError):
        K.KvView(k.float(), v.float())
    with pytest.raises(ValueError):
        K.KvView(k.cpu(), v.cpu())
    with pytest.raises(ValueError):
        K.tree_attention(out, q.to(BF16), kv, n, 40, ws)
    with pytest.raises(ValueError):
        K.tree_attention(out, q, kv, n.long(), 40, ws)
    with pytest.raises(ValueError):
        K.tree_attention(out, q, kv, n, 40, ws[:8])
    with pytest.raises(ValueError):
        K.tree_attention(out, q, kv, n, 40, ws, mask=torch.zeros(3, 2, dtype=torch.int32, device="cuda"))
    with pytest.raises(JinfError):
        K.tree_attention(out, q, kv, n, 48, ws)  # 48 + 3 nodes > 50 rows
    with pytest.raises(ValueError):
        K.attention_mass(torch.zeros(2, 2, 49, device="cuda"), q, kv, n, 40, lse)
    with pytest.raises(JinfError):
        K.kv_evict(kv, None, torch.zeros(2, 2, 50, device="cuda"), None, n,
                   torch.empty(2, 2, 51, dtype=torch.int32, device="cuda"), None, 51)
    with pytest.raises(ValueError):
        K.tree_commit(kv, None, n, 40, torch.zeros(2, dtype=torch.int32, device="cuda"), n, 3)


@pytest.mark.parametrize("dtype,hd,nh,nkv,nodes,lengths", [
    (F16, 128, 8, 1, 33, [40000, 17]), (BF16, 128, 4, 1, 30, [33333]), (F16, 64, 4, 2, 64, [30000, 29999, 12345])])
def test_long_caches_many_tiles_per_cta(cuda, dtype, hd, nh, nkv, nodes, lengths):
    """Dozens of key tiles pass through each CTA's ring, with values that are not finite behind the tree, many
    times over: out, lse and mass stay the same bits, and the first of them right."""
    from jinf import kernels as K
    g = gen(31)
    S, mp = len(lengths), max(lengths)
    k, v = make_cache(g, S, nkv, mp + nodes + 200, hd, dtype)
    for s, n in enumerate(lengths):
        k[s, :, n + nodes:], v[s, :, n + nodes:] = math.nan, math.inf
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=dtype) * 1.5
    n_past = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mask = K.tree_mask(random_parents(4, nodes)).cuda()
    out, lse = attend(q, k, v, n_past, mp, mask)
    check_attention(q, k, v, n_past, out, lse, [mask] * S, hd ** -0.5)
    kv = K.KvView(k, v)
    want, add = ref.mass(torch.zeros(S, nkv, kv.max_ctx, device="cuda"), q, k, lengths, [mask] * S, lse, None, hd ** -0.5)
    first = None
    ws = torch.zeros(K.tree_attention_workspace_bytes(kv, nh, nodes, mp), dtype=torch.uint8, device="cuda")
    for _ in range(60):
        o, e, m = torch.empty_like(out), torch.empty_like(lse), torch.zeros(S, nkv, kv.max_ctx, device="cuda")
        K.tree_attention(o, q, kv, n_past, mp, ws, mask=mask, lse=e)
        K.attention_mass(m, q, kv, n_past, mp, lse, mask=mask)
        if first is None:
            first = m
            assert bool(((m.double() - want).abs() <= 1e-4 * add + 2.0 ** -22 * want.abs()).all())
        assert torch.equal(o, out) and torch.equal(e, lse) and torch.equal(m, first)
    K.kv_ops_status()


def test_tree_decode_example(cuda):
    """The example's steps against the same model in 32 bits with its attention written out: the logits of the
    accepted nodes over the rows that the cache kept, and as many accepted tokens as a good draft brings."""
    from jinf import tree_decode as E
    from jinf.model import TINY
    model = E.StandIn(TINY, seed=3)
    seen = []

    def check(cache, tokens, parents, path, logits):
        # the last accepted node again, in plain torch: cached rows, then the path's own rows
        n, group = cache.n, TINY.n_heads // TINY.n_heads_kv
        rows = list(range(n)) + [n + t for t in path]
        for i, (q, lse) in enumerate(cache.queries):
            k, v = cache.k[i][:, rows].float(), cache.v[i][:, rows].float()
            qq = q[path[-1]].float().view(TINY.n_heads_kv, group, -1)
            s = torch.einsum("hgd,hrd->hgr", qq, k) * TINY.head_dim ** -0.5
            want = torch.logsumexp(s, -1).flatten()
            assert torch.allclose(lse[path[-1]], want, atol=1e-3)
        seen.append((n, len(path)))

    out, steps = E.decode(model, list(range(1, 9)), 250, nodes=12, right=0.9, limit=160, keep=96, recent=32, check=check)
    assert len(out) == 250 and steps < 200
    assert max(n for n, _ in seen) <= 160 and min(n for n, _ in seen[20:]) >= 96


def test_one_workspace_for_calls_of_several_shapes(cuda):
    """Calls of other node counts, and of both kernels, in turn over one workspace of the largest's size."""
    from jinf import kernels as K
    g = gen(55)
    k, v = make_cache(g, 1, 4, 3000, 128, F16)
    kv = K.KvView(k, v)
    n_past = torch.tensor([2500], dtype=torch.int32, device="cuda")
    ws = torch.zeros(max(K.tree_attention_workspace_bytes(kv, 16, t, 2600) for t in (1, 3, 40, 70)), dtype=torch.uint8,
                     device="cuda")
    want = {}
    for t in (40, 1, 70, 3, 1, 40, 3, 70):
        q = torch.randn(1, t, 16, 128, generator=gen(t), device="cuda", dtype=F16)
        out, lse = torch.empty_like(q), torch.empty(1, t, 16, device="cuda")
        K.tree_attention(out, q, kv, n_past, 2600, ws, lse=lse)
        if t in want:
            assert torch.equal(out, want[t])
        else:
            check_attention(q, k, v, n_past, out, lse, [None], 128 ** -0.5)
        want[t] = out


# (dtype, head_dim, heads, kv heads, nodes, lengths): several units' parts in most CTAs. Up to 128 rows a unit, with
# units of a single key tile in a row and between longer ones; and units of two row tiles.
MANY_UNITS = [
    (F16, 128, 32, 8, 26, [(37 * i) % 301 for i in range(60)]),
    (F16, 128, 32, 8, 5, [(1, 90, 200, 700, 3)[i % 5] + i for i in range(80)]),
    (BF16, 128, 16, 4, 12, [0, 1, 101, 102, 103, 116, 117, 245, 1200] * 9),
    (F16, 64, 16, 4, 26, [(53 * i) % 500 for i in range(90)]),
    (BF16, 128, 32, 8, 17, [8000 - 311 * i for i in range(8)]),
    (F16, 128, 32, 8, 64, [(37 * i) % 301 for i in range(40)]),
    (BF16, 64, 8, 2, 40, [(91 * i) % 640 for i in range(100)]),
]


@pytest.mark.parametrize("dtype,hd,nh,nkv,nodes,lengths", MANY_UNITS)
def test_several_units_in_a_ctas_share(cuda, dtype, hd, nh, nkv, nodes, lengths):
    """Parts of several units one behind the other in a CTA, whose roles run ahead of one another: the results
    are right and bit for bit the same in every call."""
    from jinf import kernels as K
    g = gen(nodes)
    S, mp = len(lengths), max(lengths)
    kv_pair = make_cache(g, S, nkv, mp + nodes, hd, dtype)
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=dtype)
    n_past = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mask = K.tree_mask(random_parents(nodes, nodes)).cuda()
    out, lse = attend(q, *kv_pair, n_past, mp, mask)
    K.kv_ops_status()
    kv = K.KvView(*kv_pair)
    ws = torch.zeros(K.tree_attention_workspace_bytes(kv, nh, nodes, mp), dtype=torch.uint8, device="cuda")
    again, differ = torch.empty_like(out), torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(100):
        again.fill_(math.nan)
        K.tree_attention(again, q, kv, n_past, mp, ws, mask=mask)
        differ += (again != out).sum()
    K.kv_ops_status()
    assert int(differ) == 0
    mass = torch.zeros(S, nkv, kv.max_ctx, device="cuda")
    first = None
    for _ in range(20):
        mass.zero_()
        K.attention_mass(mass, q, kv, n_past, mp, lse, mask=mask)
        first = mass.clone() if first is None else first
        differ += (mass != first).sum()
    K.kv_ops_status()
    assert int(differ) == 0
    at = [0, S // 3, S - 1]  # a few sequences in 64 bits
    check_attention(q[at], kv_pair[0][at], kv_pair[1][at], n_past[at], out[at], lse[at], [mask] * 3, hd ** -0.5)
    want, add = ref.mass(torch.zeros(3, nkv, kv.max_ctx, device="cuda"), q[at], kv_pair[0][at], [lengths[i] for i in at],
                         [mask] * 3, lse[at], None, hd ** -0.5)
    assert bool(((mass[at].double() - want).abs() <= 1e-4 * add + 2.0 ** -22 * want.abs()).all())


@pytest.mark.parametrize("dtype,hd,nh,nkv,nodes,lengths", [
    (F16, 128, 8, 8, 1, [6100]), (BF16, 64, 32, 8, 4, [1800, 0, 513, 1801, 1, 1290, 127, 1799]),
    (F16, 64, 12, 4, 5, [13001, 40]), (BF16, 128, 14, 2, 2, [24001])])
@pytest.mark.parametrize("weighted", [True, False])
def test_attention_mass_of_few_rows_over_many_tiles(cuda, dtype, hd, nh, nkv, nodes, lengths, weighted):
    """Up to 16 query rows over hundreds of key tiles, some nodes without weight and a sequence without any."""
    from jinf import kernels as K
    g = gen(nodes)
    S, mp = len(lengths), max(lengths)
    k, v = make_cache(g, S, nkv, mp + nodes, hd, dtype)
    for s, n in enumerate(lengths):
        k[s, :, n + nodes:] = math.nan
    q = torch.randn(S, nodes, nh, hd, generator=g, device="cuda", dtype=dtype)
    n_past = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    mask = K.tree_mask(random_parents(nodes, nodes)).cuda()
    _, lse = attend(q, k, v, n_past, mp, mask)
    weight = None
    if weighted:
        weight = torch.rand(S, nodes, generator=g, device="cuda")
        weight[:, 1::2] = 0.0
        weight[S - 1] *= float(S == 1)
    kv, before = K.KvView(k, v), torch.rand(S, nkv, mp + nodes, generator=g, device="cuda")
    want, add = ref.mass(before, q, k, lengths, [mask] * S, lse, weight, hd ** -0.5)
    first = None
    for _ in range(20):
        m = before.clone()
        K.attention_mass(m, q, kv, n_past, mp, lse, mask=mask, node_weight=weight)
        first = m if first is None else first
        assert torch.equal(m, first)
    K.kv_ops_status()
    assert bool(((first.double() - want).abs() <= 1e-4 * add + 2.0 ** -22 * want.abs()).all())
