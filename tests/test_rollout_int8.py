"""The rollout with its blocks' linear layers on 8-bit rows (``Rollout(int8_linears=True)``).

Tolerance of a block: a row's code step is its largest value / 127. For near-normal activations of
1536 values (largest about 3.5 deviations) that is an error of 0.8 % of the row's norm, for uniform
weights (largest 1.7 deviations) 0.4 %: 0.9 % a product. Each sublayer has two to three products in a
row, so its output moves by about 2 %, the block's change of the stream by no more than 5 %.
"""
import pytest
import torch

from streaming_sparse_b200 import rollout as R

CFG = R.WanConfig(dim=256, ffn_dim=1024, num_heads=2, num_layers=2, text_dim=128, text_len=32, latent_h=16,
                  latent_w=16, frames=6, cache_frames=6)


def _dev():
    return torch.device("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens_frame", [64, 520])
def test_block_is_close_to_bf16(tokens_frame):
    from streaming_sparse_b200.cache import KVCache

    dev, d, frames = _dev(), 1536, 3
    cfg = R.WanConfig()
    g = torch.Generator(device=dev).manual_seed(0)
    with torch.device(dev):
        blk = R.Block(cfg)
    for lin in (blk.qkv, blk.o, blk.cq, blk.ck, blk.cv, blk.co, blk.ffn1, blk.ffn2):
        a = (6.0 / sum(lin.weight.shape)) ** 0.5
        lin.weight.data.copy_(torch.rand(lin.weight.shape, device=dev, generator=g) * 2 * a - a)
        lin.bias.data.zero_()
    blk = blk.bfloat16().eval()
    n = frames * tokens_frame
    x = torch.randn(n, d, device=dev, generator=g).bfloat16()
    e0 = torch.randn(frames, 6, d, device=dev, generator=g)
    text = torch.randn(512, d, device=dev, generator=g).bfloat16()
    cos, sin = R.rope_tables(R.rope_angles(), 0, frames, tokens_frame // 8, 8, dev)
    with torch.no_grad():
        cross = blk.cross_kv(text)
        outs = []
        blk.quantize_linears()
        for int8 in (False, True):
            cache = KVCache(n, cfg.num_heads, 128, frame_tokens=tokens_frame, device=dev)
            outs.append(blk(x.clone(), e0, (cos, sin), cache, cross, 0, int8=int8).float())
    change = (outs[0] - x.float()).norm()
    assert outs[1].isfinite().all()
    assert (outs[1] - outs[0]).norm() <= 0.05 * change, ((outs[1] - outs[0]).norm() / change).item()


@pytest.mark.gpu
@pytest.mark.parametrize("attention_int8", [False, True])
def test_rollout_runs_and_replays(attention_int8):
    from streaming_sparse_b200.plugin import RouterConfig, SparseAttention, init_router_weights

    dev = _dev()
    m = R.build_model(CFG, device=dev)
    g = torch.Generator(device=dev)
    noise = torch.randn(CFG.frames, 16, 16, 16, device=dev, generator=g.manual_seed(3))
    text = torch.randn(10, CFG.text_dim, device=dev, generator=g.manual_seed(4))
    wq, wk = init_router_weights(CFG.num_heads, device=dev)
    before = R.Rollout(m).run(noise, text, generator=g.manual_seed(5))
    sp = SparseAttention(wq, wk, RouterConfig(density=0.5, int8=attention_int8))
    ro = R.Rollout(m, sparse=sp, graphs=True, int8_linears=True)
    eager, captured, replayed = (ro.run(noise, text, generator=g.manual_seed(5)) for _ in range(3))
    assert torch.isfinite(eager).all()
    assert torch.equal(captured, replayed)
    assert (captured - eager).abs().max() < 1e-2
    # a second rollout on the same model quantises into the same buffers, which the graphs still read
    R.Rollout(m, sparse=sp, int8_linears=True)
    assert torch.equal(ro.run(noise, text, generator=g.manual_seed(5)), replayed)
    ro.release_graphs()
    # the bf16 path of the same model is what it was
    assert torch.equal(R.Rollout(m).run(noise, text, generator=g.manual_seed(5)), before)


@pytest.mark.gpu
def test_int8_needs_quantised_weights_and_fused_kernels():
    m = R.build_model(CFG, device=_dev())
    with pytest.raises(ValueError):
        m.blocks[0](torch.zeros(1, 256, device=_dev()), None, None, None, None, 0, int8=True)
    with pytest.raises(ValueError):
        R.Rollout(m, fused=False, int8_linears=True)


def test_int8_is_refused_on_the_host():
    cfg = R.WanConfig(dim=128, ffn_dim=128, num_heads=1, num_layers=1, text_dim=128, text_len=8)
    with pytest.raises(ValueError):
        R.Block(cfg)(torch.zeros(1, 128), None, None, None, None, 0, int8=True)


def _replace(lin, factor):
    lin.weight = torch.nn.Parameter(lin.weight.detach() * factor)
    lin.bias = torch.nn.Parameter(lin.bias.detach() * factor + 1)


def test_loading_again_keeps_the_buffers(monkeypatch):
    """A captured graph reads the buffers that were there at its capture: they get the new values, and no
    parameter of the layer is read in their place."""
    def quant_rows(w, out, scales):   # like the kernel, it writes whatever mode the buffers are from
        with torch.inference_mode(False), torch.no_grad():
            out = torch.empty(w.shape, dtype=torch.int8) if out is None else out
            scales = torch.empty(w.shape[0]) if scales is None else scales
            scales.copy_(w.abs().amax(1) / 127)
            return out.copy_(torch.round(w / scales[:, None])), scales

    monkeypatch.setattr(R.ops, "quant_rows", quant_rows)
    lin = torch.nn.Linear(32, 16)
    for mode in (torch.no_grad, torch.enable_grad, torch.inference_mode):
        with mode():
            layer = R.Int8Linear(lin)
        kept = layer.w, layer.ws, layer.bias
        at = [t.data_ptr() for t in kept]
        old = layer.bias.clone()
        _replace(lin, 2)
        assert torch.equal(layer.bias, old)          # until load(), as the weight
        layer.load(lin)
        assert [t.data_ptr() for t in (layer.w, layer.ws, layer.bias)] == at
        assert all(a is b for a, b in zip(kept, (layer.w, layer.ws, layer.bias)))
        assert torch.equal(layer.bias, lin.bias.detach()) and layer.bias.data_ptr() != lin.bias.data_ptr()
    layer.load(lin.bfloat16())
    assert layer.bias.dtype == torch.bfloat16 and torch.equal(layer.bias, lin.bias.detach())


@pytest.mark.gpu
def test_a_captured_layer_reads_what_is_loaded_again():
    from streaming_sparse_b200 import ops

    dev = _dev()
    with torch.no_grad():
        lin = torch.nn.Linear(256, 384, device=dev, dtype=torch.bfloat16)
        layer = R.Int8Linear(lin)
        x = ops.quant_rows(torch.randn(70, 256, device=dev, generator=torch.Generator(device=dev).manual_seed(1)))
        layer(*x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(*x)
        _replace(lin, 3)
        other = [torch.randn(384, device=dev, dtype=torch.bfloat16) for _ in range(8)]   # over memory that was freed
        layer.load(lin)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, R.Int8Linear(lin)(*x)) and len(other) == 8
