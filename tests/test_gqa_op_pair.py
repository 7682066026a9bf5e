"""The op pair of the GQA backend, ``_write_kv`` and ``_attn``: one that replaces either
gets K and V, with every kind of positions (CPU)."""
from types import SimpleNamespace

import pytest
import torch

from auto_infer_amd import ops
from auto_infer_amd.attention.gqa import GqaHipBackend

HQ, HKV, D, T = 4, 2, 64, 5


class Kept(GqaHipBackend):
    def _write_kv(self, layer_idx, k, v, ctx):
        self.written = (k, v)


class Seen(GqaHipBackend):
    def _attn(self, layer_idx, q, k, v, ctx):
        self.seen = (q, k, v)
        return q


def backend(cls):
    w = {"model.layers.0.self_attn.qkv_proj.weight": torch.eye((HQ + 2 * HKV) * D),
         "model.layers.0.self_attn.o_proj.weight": torch.eye(HQ * D)}
    return cls(HQ, HKV, D, 0.1, 1, torch.device("cpu"), torch.float32, w=w, rope=ops.RotaryEmbedding(D, device="cpu"))


@pytest.fixture
def calls(monkeypatch):
    """The operators, as the host side of a backend sees them."""
    made = []

    def rope_qk(qkv, hq, hkv, *a, **kw):
        made.append("rope_qk")
        q, k, v = (t.view(T, -1, D) for t in qkv.split((HQ * D, HKV * D, HKV * D), -1))
        return 2 * q, 2 * k, v

    def rope_append(qkv, *a, **kw):
        made.append("rope_append")
        return 2 * qkv[:, :HQ * D].reshape(T, HQ, D)
    monkeypatch.setattr(ops, "rope_qk", rope_qk)
    monkeypatch.setattr(ops, "rope_append", rope_append)
    monkeypatch.setattr(ops, "write_kv", lambda *a: made.append("write_kv"))
    return made


def step():
    x = torch.randn(T, (HQ + 2 * HKV) * D, generator=torch.Generator().manual_seed(0))
    ctx = SimpleNamespace(cos=None, sin=None, positions=torch.arange(T), kv_caches=[torch.zeros(2, 3, 16, HKV, D)],
                          slot_mapping=torch.arange(T, dtype=torch.int32))
    q, k, v = (t.reshape(T, -1, D) for t in x.split((HQ * D, HKV * D, HKV * D), -1))
    return x, ctx, 2 * q, 2 * k, v


def test_a_replaced_write_gets_the_turned_rows(calls):
    b, (x, ctx, q, k, v) = backend(Kept), step()
    b._attn = lambda layer, q, k, v, c: q
    assert torch.equal(b.attention(0, x, ctx), q.flatten(1))
    assert calls == ["rope_qk"] and torch.equal(b.written[0], k) and torch.equal(b.written[1], v)


def test_replaced_attention_gets_the_turned_rows(calls):
    b, (x, ctx, q, k, v) = backend(Seen), step()
    assert torch.equal(b.attention(0, x, ctx), q.flatten(1))
    assert calls == ["rope_qk", "write_kv"] and all(map(torch.equal, b.seen, (q, k, v)))


def test_the_pair_of_the_backend_writes_on_the_way(calls, monkeypatch):
    b, (x, ctx, q, _, _) = backend(GqaHipBackend), step()
    monkeypatch.setattr(GqaHipBackend, "_attn", lambda self, layer, q, k, v, c: q)
    assert torch.equal(b.attention(0, x, ctx), q.flatten(1)) and calls == ["rope_append"]
