"""The paged operators where the framework itself calls them: decode steps of a patched attention module, and
SharedPrefixBatch."""
import numpy as np
import pytest
import torch

from test_gpu_paged import attn_close, gen, rope_close, rope_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("family", ["llama", "qwen3"])
def test_patched_decode_takes_its_rows_from_the_kernel(monkeypatch, family, dtype):
    pytest.importorskip("transformers")
    from transformers.models.llama.modeling_llama import LlamaAttention, LlamaConfig, LlamaRotaryEmbedding
    from transformers.models.qwen3.modeling_qwen3 import Qwen3Attention, Qwen3Config, Qwen3RotaryEmbedding
    from tritiercache_b200.integration import patch_model
    Cfg, Attn, Rot = {"llama": (LlamaConfig, LlamaAttention, LlamaRotaryEmbedding),
                      "qwen3": (Qwen3Config, Qwen3Attention, Qwen3RotaryEmbedding)}[family]
    torch.manual_seed(3)
    hd, nq, nkv = 64, 8, 2
    cfg = Cfg(hidden_size=256, num_attention_heads=nq, num_key_value_heads=nkv, head_dim=hd, max_position_embeddings=4096,
              attention_bias=False)
    rot = Rot(config=cfg).cuda()
    layers = []
    for _ in range(2):
        torch.manual_seed(4)
        layer = Attn(cfg, layer_idx=0).cuda().to(dtype)
        if family == "qwen3":
            for n in (layer.q_norm, layer.k_norm):
                n.weight.data += 0.2 * torch.randn(hd, device="cuda", generator=gen(5)).to(dtype)
        layers.append(layer)
    prompt = torch.randn(1, 30, 256, device="cuda", generator=gen(6)).to(dtype)
    tokens = [torch.randn(1, 1, 256, device="cuda", generator=gen(7 + i)).to(dtype) for i in range(6)]
    outs = []
    seen = []
    try:
        for layer, fused in zip(layers, (False, True)):
            patch_model.apply_patch(fused_qk=fused)
            with torch.no_grad():
                pos = torch.arange(30, device="cuda")[None]
                layer(prompt, position_embeddings=rot(prompt, pos))
                if fused:
                    step = layer.tri_tier_cache.step
                    monkeypatch.setattr(layer.tri_tier_cache, "step",
                                        lambda *a: (seen.append([t.clone() for t in a[:3]]), step(*a))[1])
                got = []
                for i, x in enumerate(tokens):
                    got.append(layer(x, position_embeddings=rot(x, torch.tensor([[30 + i]], device="cuda")))[0])
            outs.append(torch.cat(got))
            assert layer.tri_tier_cache.Total_Processed_Tokens == 36
    finally:
        patch_model.remove_patch()
        patch_model.FUSED_QK = False
    # the rows are the formula's on the projections, with one rounding to float32
    layer = layers[1]
    for i, (x, rows) in enumerate(zip(tokens, seen)):
        cos, sin = (t[0, :, :hd // 2] for t in rot(x, torch.tensor([[30 + i]], device="cuda")))
        with torch.no_grad():
            q, k, v = (p(x).view(1, -1, hd) for p in (layer.q_proj, layer.k_proj, layer.v_proj))
        wq, wk = (layer.q_norm.weight, layer.k_norm.weight) if family == "qwen3" else (None, None)
        rope_close(rows[0].view(1, nq, hd), rope_ref(q, wq, 1e-6, cos, sin, hd), q, wq, torch.float32, hd)
        rope_close(rows[1].view(1, nkv, hd), rope_ref(k, wk, 1e-6, cos, sin, hd), k, wk, torch.float32, hd)
        assert torch.equal(rows[2].view(1, nkv, hd), v.float())
    assert len(seen) == 6
    # and the module's output is that of its own steps, up to their roundings: a handful of the dtype's on values of
    # this size, on each side of a softmax
    scale = float(outs[0].float().abs().max())
    assert float((outs[0].float() - outs[1].float()).abs().max()) <= 16 * torch.finfo(dtype).eps * max(scale, 1.0)


def test_shared_prefix_batch(monkeypatch):
    from tritiercache_b200 import SharedPrefixBatch, _C
    g = gen(20)
    nq, nkv, hd, P, rows = 8, 2, 64, 16, 24
    batch = SharedPrefixBatch(40, P, nkv, hd, 5, 6, rows, dtype=torch.float16)
    ang = torch.randn((400, hd // 2), generator=g, device="cuda") * 5
    cos, sin = ang.cos(), ang.sin()
    make = lambda n, h: torch.randn((n, h, hd), generator=g, device="cuda").to(torch.float16)  # noqa: E731
    slots, pos = batch.set_prefix(70)
    _C.qk_norm_rope(make(70, nq), make(70, nkv), make(70, nkv), cos, sin, torch.empty((70, nq, hd), device="cuda", dtype=torch.float16),
                    batch.k_pages, batch.v_pages, positions=pos, slots=slots)
    new = torch.tensor([5, 1, 7, 0, 2], device="cuda", dtype=torch.int32)
    q, k, v = make(rows, nq), make(rows, nkv), make(rows, nkv)
    q_out, out = torch.zeros_like(q), torch.full_like(q, 5.0)

    def step():
        batch.begin(new)
        batch.place(q, k, v, cos, sin, q_out)
        batch.attend(q_out, out)

    def check():
        live = (batch.row_seq >= 0).nonzero().flatten()
        s = dict(q=q_out[live], k=batch.k_pages, v=batch.v_pages, ptab=batch.prefix_table, prefix=70, tables=batch.tables,
                 lens=batch.row_lens[live], seq=batch.row_seq[live], P=P)
        attn_close(out[live], s, hd ** -0.5)
        return len(live)

    step()
    assert check() == 15 and batch.lens.tolist() == [5, 1, 7, 0, 2]
    # a captured step, replayed with other lengths
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
    for lens in ([1, 1, 1, 9, 1], [1, -1, 1, 1, 1], [0, 3, 1, 1, -1]):
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(make(rows, nq)), k.copy_(make(rows, nkv)), v.copy_(make(rows, nkv))
        graph.replay()
        assert check() == sum(max(n, 0) for n in lens) and int(batch.deferred) == 0
    assert batch.lens.tolist() == [7, 3, 10, 11, 0]
    pages = [p for b in range(5) for p in batch.tables[b, :-(-int(batch.lens[b]) // P)].tolist()]
    assert sorted(pages + batch.free_pages[:int(batch.free_count)].tolist() + batch.prefix_table.tolist()) == list(range(40))
    with pytest.raises(ValueError):
        batch.set_prefix(16)
    with pytest.raises(ValueError):
        SharedPrefixBatch(2, 16, 1, 64, 1, 1, 0)
    with pytest.raises(ValueError):
        SharedPrefixBatch(2, 16, 1, 64, 1, 1, 1).set_prefix(33)
