"""The attention entry points' checks of their arguments (no GPU needed) and the
rotary tables against transformers' own frequencies."""

import ctypes
import math
import types

import pytest
import torch

from blockstreamer_b200 import _lib, attention
from oracle import attention as oatt

P, Q = 0x1000, 0x2000


def heads(ptr=P, b=512, t=256, h=64):
    return _lib.Heads(ptr, b, t, h)


def cache(**kw):
    f = dict(k=P, v=P, pages=4, page_size=16, heads=2, dim=64, k_stride_page=2048, k_stride_slot=128,
             k_stride_head=64, v_stride_page=2048, v_stride_slot=128, v_stride_head=64, page_table=P, table_width=3,
             table_stride=3, lens=P, batch=2)
    f.update(kw)
    return _lib.KVCache(*[f[n] for n, _ in _lib.KVCache._fields_])


def attend(c=None, q=None, T=2, Hq=4, window=0, ws=P, ws_bytes=1 << 30, mask_stride=0, out=P, pos=P):
    return _lib.load().bs_tree_attention(q or heads(), c or cache(), T, Hq, pos, None, mask_stride, None, window, 0.125,
                                         out, None, ws, ws_bytes, None)


def message():
    return _lib.load().bs_last_error_string().decode()


@pytest.mark.parametrize("kw,status,text", [
    (dict(out=None), _lib.BS_ERR_INVALID_ARGUMENT, "null"),
    (dict(pos=None), _lib.BS_ERR_INVALID_ARGUMENT, "null"),
    (dict(T=0), _lib.BS_ERR_INVALID_ARGUMENT, "1 to 256"),
    (dict(T=257, c=cache(table_width=300)), _lib.BS_ERR_INVALID_ARGUMENT, "1 to 256"),
    (dict(Hq=3), _lib.BS_ERR_INVALID_ARGUMENT, "multiple of the cache"),
    (dict(window=-1), _lib.BS_ERR_INVALID_ARGUMENT, "window"),
    (dict(mask_stride=-1), _lib.BS_ERR_INVALID_ARGUMENT, "mask"),
    (dict(ws_bytes=16), _lib.BS_ERR_CAPACITY, "workspace"),
    (dict(ws=None), _lib.BS_ERR_CAPACITY, "workspace"),
    (dict(q=heads(P + 2)), _lib.BS_ERR_MISALIGNED, "aligned"),
    (dict(q=heads(t=255)), _lib.BS_ERR_MISALIGNED, "multiples of 8"),
    (dict(c=cache(dim=60)), _lib.BS_ERR_INVALID_ARGUMENT, "multiple of 8"),
    (dict(c=cache(dim=136)), _lib.BS_ERR_INVALID_ARGUMENT, "up to 128"),
    (dict(c=cache(k=P + 8)), _lib.BS_ERR_MISALIGNED, "key cache"),
    (dict(c=cache(v_stride_slot=130)), _lib.BS_ERR_MISALIGNED, "strides"),
    (dict(c=cache(lens=None)), _lib.BS_ERR_INVALID_ARGUMENT, "null"),
    (dict(c=cache(page_size=0)), _lib.BS_ERR_INVALID_ARGUMENT, "cache sizes"),
    (dict(c=cache(table_width=1 << 40)), _lib.BS_ERR_INVALID_ARGUMENT, "too large"),
    (dict(T=50), _lib.BS_ERR_INVALID_ARGUMENT, "drafted tokens"),
])
def test_tree_attention_refuses(kw, status, text):
    assert attend(**kw) == status and text in message()


def test_an_empty_batch_is_fine():
    assert attend(c=cache(batch=0)) == _lib.BS_OK


def test_rope_refuses():
    lib = _lib.load()

    def rope(q=None, dtype=0, D=64, rot=64, pos_dtype=2, table=P, k=None, ko=None):
        return lib.bs_rope(q or heads(), k or heads(None), heads(Q), ko or heads(None), dtype, 2, 2, 4, 2, D, table,
                           100, rot, P, pos_dtype, 0, 0, None)

    assert rope(q=heads(None)) == _lib.BS_ERR_INVALID_ARGUMENT and "null" in message()
    assert rope(k=heads(Q)) == _lib.BS_ERR_INVALID_ARGUMENT and "k_out" in message()
    for bad in (dict(rot=63), dict(rot=66), dict(rot=0), dict(D=63, rot=32)):
        assert rope(**bad) == _lib.BS_ERR_INVALID_ARGUMENT and "even" in message()
    assert rope(dtype=2) == _lib.BS_ERR_INVALID_ARGUMENT and "dtype" in message()
    assert rope(pos_dtype=1) == _lib.BS_ERR_INVALID_ARGUMENT and "positions" in message()
    assert rope(table=P + 4) == _lib.BS_ERR_MISALIGNED
    append = lambda **kw: lib.bs_rope_append(heads(), heads(), heads(), heads(Q), cache(**kw), 2, 4, P, 100, 64, P, 2, 0, None)  # noqa: E731
    assert append(dim=68) == _lib.BS_ERR_INVALID_ARGUMENT and "multiple of 8" in message()
    assert append(k=None) == _lib.BS_ERR_INVALID_ARGUMENT and "null" in message()
    assert append(batch=0) == _lib.BS_OK


def test_upkeep_refuses():
    lib = _lib.load()
    commit = lambda T, A, acc=P: lib.bs_tree_commit(cache(), T, acc, A, None)  # noqa: E731
    assert commit(4, 5) == _lib.BS_ERR_INVALID_ARGUMENT and "at most 256" in message()
    assert commit(4, 2, None) == _lib.BS_ERR_INVALID_ARGUMENT
    scores = lambda T=2, A=2, acc=P, cap=48, Hq=4: lib.bs_kv_scores_add(heads(), cache(), T, Hq, P, acc, A, 0.1, P, P, cap, None)  # noqa: E731
    assert scores(cap=49) == _lib.BS_ERR_INVALID_ARGUMENT and "more slots" in message()
    assert scores(T=4, acc=None) == _lib.BS_ERR_INVALID_ARGUMENT and "every token" in message()
    assert scores(Hq=5) == _lib.BS_ERR_INVALID_ARGUMENT
    evict = lambda budget=16, first=0, last=0, width=1, cap=48: lib.bs_kv_evict(cache(), P, cap, budget, first, last, P, width, P, P, P, None)  # noqa: E731
    assert evict(budget=0) == _lib.BS_ERR_INVALID_ARGUMENT and "budget" in message()
    assert evict(first=10, last=7) == _lib.BS_ERR_INVALID_ARGUMENT and "keep_first" in message()
    assert evict(budget=17) == _lib.BS_ERR_INVALID_ARGUMENT and "output pages" in message()
    assert evict(cap=1000) == _lib.BS_ERR_INVALID_ARGUMENT


def test_workspace_grows_with_the_row_tile():
    size = _lib.load().bs_tree_attention_workspace_bytes
    assert size(0, 1, 8, 1, 64) == 0
    assert 0 < size(1, 1, 8, 1, 64) <= size(1, 64, 8, 1, 64)


@pytest.mark.parametrize("rot,base,scaling", [
    (64, 150000.0, dict(rope_type="yarn", factor=32.0, beta_fast=32.0, beta_slow=1.0, truncate=False,
                        original_max_position_embeddings=4096)),
    (64, 150000.0, dict(rope_type="yarn", factor=8.0, beta_fast=32.0, beta_slow=1.0,
                        original_max_position_embeddings=4096)),
    (32, 10000.0, dict(rope_type="yarn", factor=4.0, attention_factor=0.9, original_max_position_embeddings=2048)),
    (128, 500000.0, dict(rope_type="linear", factor=3.0)),
])
def test_rotary_frequencies_are_those_of_transformers(rot, base, scaling):
    hf = pytest.importorskip("transformers.modeling_rope_utils")
    full = dict(scaling, rope_theta=base)

    class Config(types.SimpleNamespace):
        def standardize_rope_params(self):
            return None

    cfg = Config(rope_theta=base, rope_scaling=full, rope_parameters=full, head_dim=rot, hidden_size=rot * 4,
                 num_attention_heads=4, max_position_embeddings=131072, partial_rotary_factor=1.0)
    want, factor = hf.ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, torch.device("cpu"))
    got, mine = attention.rotary_frequencies(rot, base, scaling)
    assert mine == pytest.approx(factor, rel=1e-6)
    assert bool(((got - want.double()).abs() <= 2e-6 * got).all())


def test_rotary_table_and_its_refusals():
    t = attention.rotary_table(131072, 64, 150000.0, device="cpu")
    assert t.shape == (131072, 32, 2) and t.dtype == torch.float32
    x = 131071 * 150000.0 ** (-2 * 5 / 64)
    assert t[131071, 5, 0].item() == pytest.approx(math.cos(x), abs=1e-7)
    assert t[131071, 5, 1].item() == pytest.approx(math.sin(x), abs=1e-7)
    with pytest.raises(ValueError, match="even"):
        attention.rotary_frequencies(33)
    with pytest.raises(ValueError, match="rope_type"):
        attention.rotary_frequencies(64, scaling=dict(rope_type="other", factor=2.0))


def test_oracle_agrees_with_torch_on_plain_attention():
    """The 64-bit definition itself, against torch's own softmax over a dense cache."""
    g = torch.Generator().manual_seed(4)
    B, T, Hq, Hkv, D, page, n = 2, 3, 4, 2, 16, 4, 9
    kc, vc = torch.randn(8, page, Hkv, D, generator=g), torch.randn(8, page, Hkv, D, generator=g)
    table = torch.tensor([[0, 2, 4], [1, 3, 5]], dtype=torch.int32)
    lens = torch.tensor([n, n], dtype=torch.int32)
    pos = (lens[:, None] + torch.arange(T)).int()
    q = torch.randn(B, T, Hq, D, generator=g)
    sinks = torch.randn(Hq, generator=g)
    out, lse, _ = oatt.tree_attention(q, kc, vc, table, lens, pos, None, sinks, 5)
    for b in range(B):
        k = kc[table[b].long()].reshape(-1, Hkv, D)[: n + T].double().repeat_interleave(Hq // Hkv, 1)
        v = vc[table[b].long()].reshape(-1, Hkv, D)[: n + T].double().repeat_interleave(Hq // Hkv, 1)
        x = torch.einsum("thd,nhd->thn", q[b].double(), k) / 4
        j = torch.arange(n + T)
        x = x.masked_fill(~((j <= pos[b][:, None]) & (j > pos[b][:, None] - 5))[:, None], -math.inf)
        x = torch.cat([x, sinks.double()[None, :, None].expand(T, -1, 1)], -1)
        w = x.softmax(-1)[..., :-1]
        assert torch.allclose(out[b], torch.einsum("thn,nhd->thd", w, v), atol=1e-12)
        assert torch.allclose(lse[b], x.logsumexp(-1), atol=1e-12)


def test_library_declares_the_structs_it_is_given():
    assert ctypes.sizeof(_lib.Heads) == 32 and ctypes.sizeof(_lib.KVCache) == 17 * 8


def test_attention_layer_has_the_parameters_of_transformers():
    hf = pytest.importorskip("transformers.models.gpt_oss.modeling_gpt_oss")
    cfg = pytest.importorskip("transformers").GptOssConfig(num_hidden_layers=2)
    for i in range(2):
        with torch.device("meta"):
            theirs = {n: tuple(p.shape) for n, p in hf.GptOssAttention(cfg, i).named_parameters()}
        ours = attention.B200GptOssAttention(cfg, i)
        assert {n: tuple(p.shape) for n, p in ours.named_parameters()} == theirs
        assert all(p.is_meta for p in ours.parameters())
        assert ours.window == (cfg.sliding_window if cfg.layer_types[i] == "sliding_attention" else 0)


def test_cpu_tensors_are_refused():
    from blockstreamer_b200 import kernels
    x = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.rope(x, None, torch.zeros(4, 32, 2), torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.tree_attention(x, x, x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                               torch.zeros(1, 1, dtype=torch.int32))
