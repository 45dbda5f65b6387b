"""Graph.paged, its append and select_pages, and attention over it, on host
tensors against the formulas in float64; and what they refuse."""

import ctypes

import numpy as np
import pytest
import torch

import tiga as tg
from tiga import _native

import paged_reference as want


class Attention(tg.MessagePassing):
    reducer = tg.online_softmax()

    def edge(self, src, dst, edge, scale):
        return self.reducer((src.key * dst.query).sum(dim=-1) * scale, src.value)


class Sum(tg.MessagePassing):
    reducer = tg.sum()

    def edge(self, src, dst, edge):
        return src.x


SIZE, PAGES = 4, 12
TABLE = torch.tensor([[3, 0, 7], [5, -1, 9], [1, 2, 12], [4, 6, 8]], dtype=torch.int32)
# (empty, ending on a page, behind a page that is not there, more than the table holds)
LENGTHS = torch.tensor([0, 8, 11, 40], dtype=torch.int32)


def graph(queries=1, table=TABLE, lengths=LENGTHS):
    return tg.Graph.paged(table, lengths, page_size=SIZE, num_pages=PAGES, queries=queries)


@pytest.mark.parametrize("queries", [1, 3])
@pytest.mark.parametrize("heads,group", [(2, 1), (2, 3), (1, 4), (1, 1)])
def test_attention_with_grouped_heads_matches_the_formula(queries, heads, group):
    rng = np.random.default_rng(queries + 10 * group)
    g = graph(queries)
    q = rng.standard_normal((4 * queries, heads, group, 8))
    k, v = rng.standard_normal((2, PAGES * SIZE, heads, 8))
    out = Attention()(graph=g, src={"key": torch.tensor(k)[:, :, None],
                                    "value": torch.tensor(v)[:, :, None]},
                      dst={"query": torch.tensor(q)}, scale=0.3)
    exp = want.attention(TABLE.numpy(), LENGTHS.numpy(), SIZE, PAGES, queries, q, k, v, 0.3)
    assert out.shape == q.shape
    # 64-bit sums of at most 12 products of 8: far below 1e-12 of the values.
    assert np.abs(out.numpy() - exp).max() <= 1e-12


def test_a_table_per_head_counts_a_row_for_every_head():
    rng = np.random.default_rng(3)
    table = torch.tensor(rng.integers(0, PAGES, size=(3, 2, 2)), dtype=torch.int32)
    lengths = torch.tensor([5, 8, 1], dtype=torch.int32)
    g = tg.Graph.paged(table, lengths, page_size=SIZE, num_pages=PAGES, queries=2)
    assert (g.schema.num_dst, g.schema.num_src) == (3 * 2 * 2, PAGES * SIZE * 2)
    q = rng.standard_normal((12, 3, 8))
    k, v = rng.standard_normal((2, PAGES * SIZE, 2, 1, 8))
    flat = lambda t: torch.tensor(t).reshape(-1, 1, 8)
    out = Attention()(graph=g, src={"key": flat(k), "value": flat(v)},
                      dst={"query": torch.tensor(q)}, scale=0.5)
    exp = want.attention(table.numpy(), lengths.numpy(), SIZE, PAGES, 2, q[:, None], k, v, 0.5)
    assert np.abs(out.numpy() - exp[:, 0]).max() <= 1e-12


def test_the_tables_are_read_as_they_stand():
    table, lengths = TABLE.clone(), LENGTHS.clone()
    g = graph(table=table, lengths=lengths)
    x = torch.arange(PAGES * SIZE, dtype=torch.float64)
    kernel = Sum()

    def expected():
        out = []
        for b in range(4):
            n = want.length_of(lengths, b, 3, SIZE)
            at, named = want.slots(table[b], n, SIZE, PAGES)
            out.append(x.numpy()[at[named]].sum())
        return np.array(out)

    for _ in range(2):
        got = kernel(graph=g, src={"x": x}, dst={})
        assert np.array_equal(got.numpy(), expected())
        assert g.num_edges == g.snapshot().num_edges
        lengths += 1
        table[1, 1] = 11
    assert g.schema.lifecycle == "live" and "paged" in repr(g)
    assert g.degree_statistics() == g.snapshot().degree_statistics()
    assert g.transpose().num_edges == g.num_edges


def test_block_pruning_and_prepare_are_refused_on_the_host():
    class Pruned(Attention):
        reducer = tg.online_softmax(block_prune_threshold=0.5)

    q = torch.randn(4, 2, 8)
    k = torch.randn(PAGES * SIZE, 2, 8)
    call = dict(graph=graph(), src={"key": k, "value": k}, dst={"query": q}, scale=1.0)
    with pytest.raises(NotImplementedError):
        Pruned()(**call)
    with pytest.raises(NotImplementedError):
        Attention().prepare(**call)


@pytest.mark.parametrize("queries", [1, 2, 6])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_append_writes_the_newest_rows_and_sums_the_pages(queries, dtype):
    rng = np.random.default_rng(queries)
    table, lengths = TABLE.numpy(), np.array([1, 5, 11, 40], dtype=np.int32)
    g = graph(queries, lengths=torch.tensor(lengths))
    mk = lambda *s: torch.tensor(rng.standard_normal(s)).to(dtype)
    kc, vc = mk(PAGES * SIZE, 2, 4), mk(PAGES * SIZE, 2, 4)
    k, v = mk(4 * queries, 2, 4), mk(4 * queries, 2, 4)
    sums = torch.full((PAGES, 2, 4), 7.0)
    exp = want.append(table, lengths, SIZE, PAGES, queries, *(t.numpy() for t in (kc, k, vc, v)),
                      sums.numpy())
    g.append(kc, k, vc, v, page_sums=sums)
    assert np.array_equal(kc.numpy(), exp[0]) and np.array_equal(vc.numpy(), exp[1])
    # Sums of at most 4 values in 32 bits: 4 roundings of 2^-24 of at most 4 * max.
    assert np.abs(sums.numpy() - exp[2]).max() <= 16 * 2 ** -24 * np.abs(exp[2]).max()


@pytest.mark.parametrize("queries,count", [(1, 1), (1, 2), (1, 5), (3, 2)])
def test_select_pages_takes_the_newest_and_the_best(queries, count):
    rng = np.random.default_rng(count)
    g = graph(queries)
    q = rng.standard_normal((4 * queries, 2, 3, 8))
    sums = rng.standard_normal((PAGES, 2, 8)).astype(np.float32)
    sums[4], sums[6] = sums[6], sums[4]
    sums[6] = sums[4]           # equal scores
    sums[3, 0, 0] = np.nan
    chosen = g.select_pages(torch.tensor(q), torch.tensor(sums), count)
    table, lengths = want.select(TABLE.numpy(), LENGTHS.numpy(), SIZE, PAGES, queries, q, sums,
                                 count)
    assert np.array_equal(chosen.page_table.numpy(), table)
    assert np.array_equal(chosen.lengths.numpy(), lengths)
    before = chosen.page_table.data_ptr()
    assert g.select_pages(torch.tensor(-q), torch.tensor(sums), count, out=chosen) is chosen
    table, _ = want.select(TABLE.numpy(), LENGTHS.numpy(), SIZE, PAGES, queries, -q, sums, count)
    assert chosen.page_table.data_ptr() == before
    assert np.array_equal(chosen.page_table.numpy(), table)


def test_paged_refusals():
    ok = dict(page_size=SIZE, num_pages=PAGES)
    mk = tg.Graph.paged
    with pytest.raises(TypeError, match="int32"):
        mk(TABLE.long(), LENGTHS, **ok)
    with pytest.raises(TypeError, match="int32"):
        mk(TABLE, LENGTHS.long(), **ok)
    with pytest.raises(TypeError, match="torch.Tensor"):
        mk(TABLE.tolist(), LENGTHS, **ok)
    with pytest.raises(ValueError, match="page_table must be"):
        mk(TABLE[0], LENGTHS, **ok)
    with pytest.raises(ValueError, match=r"lengths must be \[4\]"):
        mk(TABLE, LENGTHS[:3], **ok)
    with pytest.raises(ValueError, match="dense"):
        mk(TABLE.t().contiguous().t(), LENGTHS, **ok)
    for bad in (dict(page_size=0), dict(num_pages=-1), dict(queries=0), dict(page_size=True),
                dict(page_size=2.0)):
        with pytest.raises(ValueError, match="integer of at least"):
            mk(TABLE, LENGTHS, **{**ok, **bad})
    with pytest.raises(ValueError, match="2\\*\\*31"):
        mk(TABLE, LENGTHS, page_size=SIZE, num_pages=2 ** 30)
    with pytest.raises(ValueError, match="2\\*\\*30"):
        mk(TABLE[:, :0], LENGTHS, page_size=2 ** 30, num_pages=1)
    with pytest.raises(ValueError, match="validate must be"):
        mk(TABLE, LENGTHS, validate="some", **ok)
    with pytest.raises(ValueError, match="more tokens"):
        mk(TABLE, LENGTHS, validate="full", **ok)
    with pytest.raises(ValueError, match="out-of-range page"):
        mk(TABLE, LENGTHS.clamp(max=12), validate="full", **ok)
    mk(TABLE, torch.tensor([12, 4, 8, 12], dtype=torch.int32), validate="full", **ok)


def test_append_refusals():
    g = graph()
    kc, k, sums = torch.zeros(PAGES * SIZE, 2, 4), torch.zeros(4, 2, 4), torch.zeros(PAGES, 2, 4)
    with pytest.raises(TypeError, match="paged relation"):
        tg.Graph.dense(3).append(kc, k, kc, k)
    with pytest.raises(ValueError, match="not one per head"):
        tg.Graph.paged(TABLE[:, None], LENGTHS, page_size=SIZE, num_pages=PAGES).append(
            kc, k, kc, k)
    with pytest.raises(TypeError, match="key must be a torch.Tensor"):
        g.append(kc, None, kc, k)
    with pytest.raises(ValueError, match="key_cache must have shape"):
        g.append(kc[:-1], k, kc, k)
    with pytest.raises(ValueError, match="value must have shape"):
        g.append(kc, k, kc, k[:, :1])
    with pytest.raises(TypeError, match="one floating type"):
        g.append(kc, k.half(), kc, k)
    with pytest.raises(ValueError, match="expanded"):
        g.append(torch.zeros(1, 2, 4).expand(PAGES * SIZE, 2, 4), k, kc, k)
    with pytest.raises(ValueError, match="dense"):
        g.append(torch.zeros(PAGES * SIZE, 4, 2).transpose(1, 2), k, kc, k)
    with pytest.raises(TypeError, match="float32"):
        g.append(kc, k, kc, k, page_sums=sums.double())
    with pytest.raises(ValueError, match="contiguous"):
        g.append(kc, k, kc, k, page_sums=sums[:, :1])
    with pytest.raises(NotImplementedError, match="no gradient"):
        g.append(kc, k.clone().requires_grad_(), kc, k)
    with torch.no_grad():
        g.append(kc, k.clone().requires_grad_(), kc, k)


def test_select_pages_refusals():
    g = graph()
    q, sums = torch.zeros(4, 2, 3, 8), torch.zeros(PAGES, 2, 8)
    with pytest.raises(TypeError, match="paged relation"):
        tg.Graph.dense(3).select_pages(q, sums, 2)
    with pytest.raises(ValueError, match="query must be"):
        g.select_pages(q[:3], sums, 2)
    with pytest.raises(ValueError, match="query must be"):
        g.select_pages(q.long(), sums, 2)
    with pytest.raises(ValueError, match="page_sums must be"):
        g.select_pages(q, sums.double(), 2)
    with pytest.raises(ValueError, match="page_sums must be"):
        g.select_pages(q, sums[:, :1], 2)
    for count in (0, -1, 2.0, True):
        with pytest.raises(ValueError, match="count"):
            g.select_pages(q, sums, count)
    chosen = g.select_pages(q, sums, 2)
    with pytest.raises(ValueError, match="out must be"):
        g.select_pages(q, sums, 3, out=chosen)
    with pytest.raises(ValueError, match="out must be"):
        g.select_pages(q, sums, 2, out=g)
    with pytest.raises(ValueError, match="not one per head"):
        chosen.select_pages(q, sums, 2)


def test_forward_mode_over_host_tensors():
    """Attention and norm_rotary of host tensors carry tangents."""
    make_dual, unpack = torch.autograd.forward_ad.make_dual, torch.autograd.forward_ad.unpack_dual
    rng = np.random.default_rng(31)
    g = graph()
    mk = lambda *s: torch.tensor(rng.standard_normal(s))
    q, k, v, dq = mk(4, 2, 8), mk(PAGES * SIZE, 2, 8), mk(PAGES * SIZE, 2, 8), mk(4, 2, 8)
    attend = lambda q: Attention()(graph=g, src={"key": k, "value": v}, dst={"query": q},
                                   scale=0.5)
    rotate = lambda q: tg.nn.norm_rotary(q, None, torch.arange(4), torch.ones(4))
    for f in (attend, rotate):
        with torch.autograd.forward_ad.dual_level():
            got = unpack(f(make_dual(q, dq))).tangent
        assert got is not None
        # Central differences in 64 bits: h^2 times third derivatives of order 10.
        assert ((f(q + 1e-5 * dq) - f(q - 1e-5 * dq)) / 2e-5 - got).abs().max() <= 1e-8


def paged_attention_workspace(n_seqs, heads, group, queries, D, dtype, pages=64, size=16):
    """Status of the native launch's size check."""
    p = _native.Paged(1, pages, 0, 1, n_seqs, 1, pages, size, pages, queries)
    need = ctypes.c_size_t()
    status = _native.lib().tgx_paged_attn_workspace(ctypes.byref(p), heads, group, D, dtype,
                                                    ctypes.byref(need))
    return status, need.value


def test_launches_that_need_no_workgroup_per_query_take_prompts():
    """16 sequences of 32768 new tokens on matrix tiles of 128 queries; what a
    workgroup a query cannot be launched for is told as uncovered."""
    assert paged_attention_workspace(16, 8, 4, 32768, 128, 0, pages=4096) == (0, 0)
    # A join of more queries than a launch has workgroups is left out.
    assert paged_attention_workspace(600, 8, 4, 1024, 128, 0, pages=4096) == (0, 0)
    unsupported = 2
    assert paged_attention_workspace(16, 8, 4, 32768, 128, 2, pages=4096)[0] == unsupported
    assert paged_attention_workspace(16, 8, 4, 32768, 96, 0, pages=4096)[0] == unsupported
    assert paged_attention_workspace(1 << 20, 64, 1, 1, 128, 0)[0] == unsupported


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,lost", [(20000, 320), (3000, 256)])
def test_the_bound_of_the_kernels_rejects_what_is_lost(n, lost, dtype):
    """Zeros, and an output without one piece of the keys, lie outside of what
    rounding may do; the rounded formula lies inside."""
    rng = np.random.default_rng(30)
    size, D = 16, 128
    pages = -(-n // size)
    table, mk = np.arange(pages)[None], rng.standard_normal
    q, k, v = mk((1, 2, 4, D)), mk((pages * size, 2, D)), mk((pages * size, 2, D))
    args = (table, [n], size, pages, 1, q, k)
    exp = want.attention(*args, v, D ** -0.5)
    lim = want.attention_bound(*args, v, D ** -0.5, dtype, dtype != "f32")
    rounded = torch.tensor(exp).to({"bf16": torch.bfloat16, "f16": torch.float16,
                                    "f32": torch.float32}[dtype]).double().numpy()
    assert (np.abs(rounded - exp) <= lim).all()
    assert (np.abs(exp) > lim).mean() > 0.9             # zeros
    for first in (0, n // 2 // lost * lost, n - lost):
        short = np.delete(np.arange(n), np.arange(first, first + lost))
        kk, vv = (np.concatenate([x[short], x[:lost]]) for x in (k, v))
        without = want.attention(table, [n - lost], size, pages, 1, q, kk, vv, D ** -0.5)
        assert (np.abs(without - exp) > lim).mean() > 0.25


def test_tables_are_advanced_in_place_not_replaced():
    """The launches are sized by the tables a relation was made of."""
    g = graph()
    for name, value in (("page_table", TABLE[:, :1]), ("lengths", LENGTHS[:1]), ("page_size", 1),
                        ("num_pages", 99), ("queries", 2)):
        with pytest.raises(AttributeError):
            setattr(g.paged_state, name, value)
