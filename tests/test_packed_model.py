"""Packed documents, embedding scale and dropout in the model and the trainer."""
import copy
import math

import pytest
import torch

from system_lab_b200 import ops
from system_lab_b200.config import Config, ConfigError
from system_lab_b200.models.simple_moe import BatchInfo, SimpleMoE
from system_lab_b200.parallel.mesh import single_process_mesh
from system_lab_b200.trainer.loop import Trainer

DENSE = ["num_experts=0", "ffn_hidden_size=256", "vocab_size=512", "seq_length=128", "micro_batch_size=2", "global_batch_size=4",
         "expert_model_parallel_size=1", "heartbeat=false"]
PACKED = ["reset_attention_mask=true", "eod_token=0"]


def config(*more):
    return Config.load(preset="simplemoe-tiny", overrides=DENSE + list(more))


def model(cfg):
    torch.manual_seed(0)
    m = SimpleMoE(cfg.model)
    m.init_weights(1)
    return m


def test_every_document_is_as_if_alone():
    """Logits of a packed row are those of its documents run one by one (rotary positions are relative)."""
    cfg = config(*PACKED, "embedding_multiplier=4.0", "num_query_groups=2")
    m = model(cfg).eval()
    tok = torch.randint(1, 512, (2, 50))
    cuts = [[0, 7, 8, 50], [0, 21, 40, 50]]
    for row, cut in zip(tok, cuts):
        for c in cut[1:-1]:
            row[c - 1] = 0
    with torch.no_grad():
        packed = m(tok)
        for row, cut, out in zip(tok, cuts, packed):
            for a, b in zip(cut[:-1], cut[1:]):
                alone = m(row[None, a:b])[0]
                torch.testing.assert_close(out[a:b], alone, rtol=2e-4, atol=2e-5)
        cfg.model.reset_attention_mask = False
        assert not torch.allclose(m(tok)[0, 8:], packed[0, 8:], atol=1e-3)


def test_embedding_multiplier():
    cfg = config("embedding_multiplier=3.0")
    m = model(cfg)
    tok = torch.randint(0, 512, (2, 9))
    assert torch.equal(m.embed(tok, torch.float32), m.embed.weight[tok] * 3.0)


def test_dropout_is_a_function_of_the_seed():
    cfg = config("hidden_dropout=0.2", "lora_rank=4", "lora_targets=attn+mlp", "lora_dropout=0.3")
    m = model(cfg)
    for p in m.parameters():
        torch.nn.init.normal_(p, std=0.05)
    tok, tgt = torch.randint(0, 512, (2, 20)), torch.randint(0, 512, (2, 20))
    loss = [m(tok, tgt, batch=m.batch_info(tok, s)).item() for s in (1, 1, 2)]
    assert loss[0] == loss[1] != loss[2]
    plain = m(tok, tgt).item()
    assert m.batch_info(tok) is None and m(tok, tgt, batch=BatchInfo()).item() == plain
    # each place draws a mask of its own
    offsets = [l.offset for l in m.layers] + [x.offset for l in m.layers for x in
                                              (l.attn.qkv_lora, l.attn.o_lora, l.ffn.w1_lora, l.ffn.w2_lora)]
    taken = {o + s for o in offsets[:len(m.layers)] for s in (0, 1)} | set(offsets[len(m.layers):]) | {0}
    assert len(taken) == 1 + 6 * len(m.layers)


def run(cfg, steps=3, device="cpu", mode="auto"):
    tr = Trainer(cfg, mesh=single_process_mesh(), device=torch.device(device))
    if mode == "reference":
        ops.set_kernel_mode("reference")
    out = [float(tr.train_step()["loss"]) for _ in range(steps)]
    held_out = tr.evaluate(1)
    params = [g.shard.clone() for g in tr.engine.all_groups()]
    tr.close()
    return out, held_out, params


@pytest.mark.parametrize("extra", [["hidden_dropout=0.1"], ["lora_rank=4", "lora_targets=attn+mlp", "lora_dropout=0.2"]])
def test_recompute_draws_the_same_masks(extra):
    """A recomputed block repeats its first run: losses and updates do not depend on what is recomputed."""
    runs = {g: run(config(*PACKED, *extra, f"recompute_granularity={g}")) for g in ("none", "selective", "full")}
    for g in ("selective", "full"):
        assert runs[g][0] == pytest.approx(runs["none"][0], rel=1e-6)
        for a, b in zip(runs[g][2], runs["none"][2]):
            torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-7)
    assert run(config(*PACKED, *extra)) [0] == runs["none"][0]                       # and the run repeats itself


def test_evaluation_drops_nothing():
    cfg = config("hidden_dropout=0.5")
    tr = Trainer(cfg, mesh=single_process_mesh(), device=torch.device("cpu"))
    still = copy.deepcopy(cfg)
    still.model.hidden_dropout = 0.0
    same = Trainer(still, mesh=single_process_mesh(), device=torch.device("cpu"))
    assert tr.evaluate(1) == same.evaluate(1)


@pytest.mark.parametrize("bad", [["reset_attention_mask=true"], ["reset_attention_mask=true", "eod_token=512"],
                                 PACKED + ["context_parallel_size=2"], PACKED + ["pipeline_model_parallel_size=2"],
                                 ["hidden_dropout=1.0"], ["hidden_dropout=-0.1"], ["lora_dropout=0.1"],
                                 ["hidden_dropout=0.1", "tensor_model_parallel_size=2"],
                                 ["hidden_dropout=0.1", "pipeline_model_parallel_size=2"]])
def test_refused_configurations(bad):
    with pytest.raises(ConfigError):
        config(*bad)


def test_latent_attention_refuses_documents():
    with pytest.raises(ConfigError):
        Config.load(preset="deepseek-v3-proxy", overrides=PACKED)


@pytest.mark.gpu
@pytest.mark.parametrize("extra", [["hidden_dropout=0.1", "embedding_multiplier=16.0"],
                                   ["lora_rank=4", "lora_targets=attn+mlp", "lora_dropout=0.1", "recompute_granularity=selective"],
                                   ["num_experts=8", "hidden_dropout=0.1", "recompute_granularity=full", "moe_pad_expert_rows_to=128"],
                                   ["num_query_groups=2", "sliding_window=40", "recompute_granularity=selective"]])
def test_training_on_packed_documents(extra):
    """The whole run on the kernels against the same run on the oracles: the masks are equal, so the losses of the first
    steps are, up to what bf16 rounds (a loss near ln 512 = 6.2 from activations with 8 bits: 2^-7 of it with room)."""
    from system_lab_b200.ops import cuda
    cfg = config(*PACKED, *extra, "params_dtype=bf16", "vocab_size=512")
    got, held, _ = run(cfg, device="cuda")
    cuda.check_status()
    again, held2, _ = run(cfg, device="cuda")
    want, held3, _ = run(cfg, device="cuda", mode="reference")
    ops.set_kernel_mode("auto")
    assert all(math.isfinite(x) for x in got)
    assert got == pytest.approx(want, rel=2 ** -7) and held == pytest.approx(held3, rel=2 ** -7)
    assert got[0] == pytest.approx(again[0], rel=1e-6)      # (the cross entropy adds its rows' losses in fp32, in any order)


@pytest.mark.gpu
def test_the_set_together():
    """Token ids to the residual stream and back, as a layer uses the operators, against 64 bits; captured and replayed."""
    from system_lab_b200.ops import cuda
    dev, b, s, hid, hq, hkv, d, v = "cuda", 2, 300, 256, 4, 2, 64, 700
    g = torch.Generator(device=dev)
    g.manual_seed(5)
    table = torch.randn(v, hid, device=dev, generator=g).bfloat16().requires_grad_(True)
    w = (torch.randn((hq + 2 * hkv) * d, hid, device=dev, generator=g) / 16).bfloat16().requires_grad_(True)
    tokens = torch.randint(0, 40, (b, s), device=dev, generator=g)
    dout = torch.randn(b, s, hid, device=dev, generator=g).bfloat16()
    seed = torch.tensor([9], device=dev)

    def step(tab, ww, low=True):
        docs = ops.documents_from_tokens(tokens, 0)
        x = ops.embedding(tokens, tab, scale=0.5)
        qkv = torch.nn.functional.linear(x, ww)
        q, k, vv = qkv.flatten(0, 1).split([hq * d, hkv * d, hkv * d], dim=-1)
        heads = [t.unflatten(-1, (-1, d)) for t in (q, k, vv)]
        a = ops.packed_attention(*heads, docs)
        y = ops.dropout(a.reshape(b, s, hid), 0.25, seed if low else int(seed), 3, residual=x)
        return (y, *torch.autograd.grad(y, (tab, ww), dout.to(y.dtype)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(table, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(table, w)
    for s_ in (9, 10):
        seed.fill_(s_)
        tokens.copy_(torch.randint(0, 40, (b, s), device=dev, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        cuda.check_status()
        ops.set_kernel_mode("reference")
        try:
            want = step(table.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True), low=False)
        finally:
            ops.set_kernel_mode("auto")
        # five roundings to bf16 follow one another on the way (x, qkv, p, a, y; their gradients likewise), each at most 2^-8:
        # together below 5 * 2^-8 of the root mean square, even if all had one sign
        for x, y in zip(got, want):
            err = (x.double() - y).pow(2).mean().sqrt()
            assert err <= 5 * 2 ** -8 * y.pow(2).mean().sqrt(), (err, y.pow(2).mean().sqrt())
