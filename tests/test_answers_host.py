"""The batched step over pages, on the host: the argument blocks of its graph."""
import struct

import pytest

torch = pytest.importorskip("torch")

from etx_megakernel_b200.models import batched as BT  # noqa: E402
from etx_megakernel_b200.models import qwen as Q  # noqa: E402
from etx_megakernel_b200.ops import attn as op_attn  # noqa: E402
from etx_megakernel_b200.ops import batch as op_batch  # noqa: E402
from etx_megakernel_b200.passes import compile_graph, verify_plan  # noqa: E402
from etx_megakernel_b200.runtime import Sampling  # noqa: E402
from etx_megakernel_b200.sim.protocol import simulate  # noqa: E402


def _ptr(name):
    return 0x100000000 + 65536 * (sum(map(ord, name)) % 4096)


def block(pool, name, n):
    return pool.bytes()[{r[0]: r for r in pool.rows}[name][4]:][:n]


def test_graph_over_pages():
    """One prologue block more (over tables), layers as far apart as the pool is large, slots behind the step's own; all else as without pages."""
    d = Q.load_dims("qwen3-30b-a3b", layers=2)
    B, pages, nblk = 6, 50, -(-1072 // Q.BS)
    g, pool, _ = BT.build_graph(d, _ptr, B, 1072)
    gp, poolp, _ = BT.build_graph(d, _ptr, B, 1072, pages=pages)
    assert [x.name for x in g.grids] == [x.name for x in gp.grids]
    plan = compile_graph(gp, "b200", {"POOL": len(poolp.bytes())})
    assert verify_plan(plan) == [] and not simulate(plan).deadlock
    assert struct.unpack_from("<2i", block(pool, "prologue", 32)) == (B, nblk * 16)
    assert struct.unpack_from("<2iQ", block(poolp, "prologue", 32)) == (B | op_batch.COLS_TABLES, nblk * 16, _ptr("block_tables"))
    assert block(pool, "argmax", 32) == block(poolp, "argmax", 32)
    moved = [i for i, (x, y) in enumerate(zip(block(pool, "attn_1", op_attn.F_ARG_BYTES), block(poolp, "attn_1", op_attn.F_ARG_BYTES))) if x != y]
    page = d.NKV * d.HD * 32
    at = {n: [i for i in range(0, 160, 8) if struct.unpack_from("<Q", block(poolp, "attn_1", op_attn.F_ARG_BYTES), i)[0] == v]
          for n, v in (("kc", _ptr("kc") + (pages + 1) * page), ("vc", _ptr("vc") + (pages + 1) * page), ("slot", _ptr("slot_mapping") + 8))}
    assert all(len(v) == 1 for v in at.values()) and {i // 8 * 8 for i in moved} == {v[0] for v in at.values()}
    shapes, own = BT.buffer_shapes(d, B, 1072, 8, 9, pages), BT.buffer_shapes(d, B, 1072, 8, 9)
    assert shapes["kc"][0] == (2, pages + 1, *own["kc"][0][2:]) and shapes["vc"][0] == (2, pages + 1, *own["vc"][0][2:]) and shapes["slot_mapping"][0] == (B + 1,)
    assert all(shapes[n] == own[n] for n in own if n not in ("kc", "vc", "slot_mapping"))


def test_a_vocabulary_that_rows_of_logits_cannot_have_is_refused():
    d = Q.Dims(name="odd", H=512, NH=8, NKV=2, HD=128, INTER=0, L=1, V=1500, qk_norm=True, moe=True, E=16, TOPK=4, MI=128, norm_topk=True)
    BT.build_graph(d, _ptr, 1, 64)
    with pytest.raises(ValueError, match="no multiple of 8"):
        BT.build_graph(d, _ptr, 2, 64)


def test_given_random_numbers():
    u = torch.rand((3, 2))
    assert Sampling(given=u).numbers(3, 2, "cpu") is u and torch.equal(Sampling(seed=4).numbers(3, 2, "cpu"), Sampling(seed=4).numbers(3, 2, "cpu"))
    with pytest.raises(ValueError, match="random numbers"):
        Sampling(given=u).numbers(2, 3, "cpu")
