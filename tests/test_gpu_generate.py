"""generate.Generator and generate.generate: rotary positions, the 8-bit cache with its attention, and the logits'
processing run together.

Whole models are no oracle here: what rounding moves a key by moves a sharp softmax by several times as much, layer after
layer.  So every layer of every step is checked on what it was given: the attention's output on the queries, keys and
values that its projections gave, with the bar that test_gpu_kv_cache.py derives, and the rest of the layer, which is
the model's own modules, bit for bit.
"""
import pytest
import torch
from test_gpu_kv_cache import _attention, _stored

pytestmark = pytest.mark.gpu


def _model(dev, heads=2, dim=64, layers=2, vocab=503, scaling=None, seed=0):
    from sparseforge_amd.llama import LlamaDecoder, LlamaShape

    shape = LlamaShape(vocab_size=vocab, hidden_size=heads * dim, intermediate_size=256, num_hidden_layers=layers,
                       num_attention_heads=heads, rope_scaling=scaling)
    m = LlamaDecoder(shape, None, device=dev)
    m.init_random(torch.Generator(device=dev).manual_seed(seed), std=0.2)
    return m


def _packed(dev):
    """A finalized student whose projections are packed 2:4."""
    from sparseforge_amd.finalize import convert_model_to_2to4, finalize_sparse_model
    from sparseforge_amd.llama import LlamaDecoder, LlamaShape
    from sparseforge_amd.sparse_modeling import SparseLinear, SparseLinearConfig

    cfg = SparseLinearConfig(mask_type="unstructured", hard_mask_type="nm_2_4", SLoRB=False)
    m = LlamaDecoder(LlamaShape(vocab_size=503, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
                                num_attention_heads=2), cfg, device=dev)
    g = torch.Generator(device=dev).manual_seed(5)
    m.init_random(g, std=0.2)
    with torch.no_grad():
        for mod in m.modules():
            if isinstance(mod, SparseLinear):
                mod.mask.copy_(torch.rand(mod.mask.shape, generator=g, device=dev))
    finalize_sparse_model(m)
    convert_model_to_2to4(m)
    return m


class _Watched:
    """What the model's modules are given and give during a step."""

    def __init__(self, m):
        self.seen = {}
        for i, layer in enumerate(m.layers):
            for name, mod in (("h", layer.input_layernorm), ("h1", layer.post_attention_layernorm),
                              ("q", layer.self_attn.q_proj), ("k", layer.self_attn.k_proj),
                              ("v", layer.self_attn.v_proj), ("o", layer.self_attn.o_proj)):
                mod.register_forward_hook(lambda _m, x, y, key=(i, name): self.seen.__setitem__(key, (x[0], y)))
        m.norm.register_forward_hook(lambda _m, x, y: self.seen.__setitem__("norm", (x[0], y)))


def _check_step(m, watched, held, starts, counts, n, cos, sin, logits):
    """held[layer][b]: turned keys and values [T, H, D] before the step; they are extended."""
    from sparseforge_amd.llama import swiglu
    from sparseforge_amd.rotary import rotary_embed

    H, D, B = m.config.num_attention_heads, m.config.head_dim, len(starts)
    w = watched.seen
    for i, layer in enumerate(m.layers):
        q, k, v = (w[i, name][1].view(B, n, H, D) for name in "qkv")
        out = w[i, "o"][0].view(B, n, H, D).double()
        for b in range(B):
            c = counts[b]
            assert not out[b, c:].any()
            if not c:
                continue
            at = torch.arange(starts[b], starts[b] + c, device=q.device)[None]
            qt, kt = (x[0] for x in rotary_embed(q[b:b + 1, :c], k[b:b + 1, :c], cos, sin, at))
            ks, vs = (torch.cat(pair) for pair in zip(held[i][b], (kt, v[b, :c])))
            held[i][b] = [ks, vs]
            end = starts[b] + c
            assert ks.shape[0] == end
            o, bar = _attention(qt, _stored(ks, end), _stored(vs, end), starts[b], D ** -0.5, 0)
            assert bool(((out[b, :c] - o).abs() <= bar).all())
        h, x = w[i, "h"]
        assert torch.equal(w[i, "h1"][0], h + w[i, "o"][1])
        f, y = layer.mlp, w[i, "h1"][1]
        after = w[i, "h1"][0] + f.down_proj(swiglu(f.gate_proj(y), f.up_proj(y)))
        if i + 1 < len(m.layers):
            assert torch.equal(w[i + 1, "h"][0], after)
        else:
            for b in range(B):
                if counts[b]:
                    assert torch.equal(w["norm"][0][b], after[b, counts[b] - 1])
    assert torch.equal(logits, m.lm_head(w["norm"][1]))


@pytest.mark.parametrize("kind", ["heads of 64", "heads of 128", "scaled", "packed"])
def test_steps(cuda_device, kind):
    """Chunks, single tokens, ragged counts, a sequence that has ended."""
    from sparseforge_amd.generate import Generator
    from sparseforge_amd.rotary import RotaryScaling, rotary_cos_sin

    scaling = RotaryScaling("yarn", 4.0, 64) if kind == "scaled" else None
    if kind == "packed":
        m = _packed(cuda_device)
    else:
        m = _model(cuda_device, 3 if scaling else 2, 128 if kind == "heads of 128" else 64, scaling=scaling)
    watched = _Watched(m)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    B, H, D = 3, m.config.num_attention_heads, m.config.head_dim
    none = torch.empty(0, H, D, dtype=torch.bfloat16, device=cuda_device)
    cos, sin = rotary_cos_sin(512, D, m.config.rope_theta, scaling, cuda_device)
    with torch.no_grad():
        for plan in ([(70, None), (1, None), (1, None), (40, None), (17, None), (1, None), (70, None)],
                     [(100, [100, 1, 64]), (1, [0, 1, 1]), (1, [1, 1, 1]), (30, [0, 30, 7])]):
            gen = Generator(m, B, 210)
            held = [[[none, none] for _ in range(B)] for _ in m.layers]
            starts = [0] * B
            for n, counts in plan:
                idx = torch.randint(0, 503, (B, n), generator=g, device=cuda_device)
                given = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda_device)
                logits = gen.step(idx, given)
                counts = counts or [n] * B
                _check_step(m, watched, held, starts, counts, n, cos, sin, logits)
                starts = [s + c for s, c in zip(starts, counts)]
                assert gen.cache.ends.tolist() == starts
    assert torch.equal(watched.seen[0, "h"][0], m.embed_tokens(idx))


def test_scaled_model_trains_with_the_scaled_tables(cuda_device):
    """LlamaShape.rope_scaling reaches the forward: its tables are rotary_cos_sin's, each half a copy."""
    from sparseforge_amd.rotary import RotaryScaling, rotary_cos_sin

    scaling = RotaryScaling("linear", 4.0)
    cos, sin = _model(cuda_device, scaling=scaling)._tables(50, cuda_device)
    c, s = rotary_cos_sin(50, 64, 10000.0, scaling, cuda_device)
    assert torch.equal(cos, torch.cat([c, c], -1)) and torch.equal(sin, torch.cat([s, s], -1))


def test_generate_is_its_steps(cuda_device):
    """generate() against the loop written out, greedily, ragged prompts, in one chunk and in several."""
    from sparseforge_amd.generate import Generator, generate
    from sparseforge_amd.logits import process_logits

    m = _model(cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    prompts = torch.randint(0, 503, (3, 50), generator=g, device=cuda_device)
    count = [50, 7, 33]
    lengths = torch.tensor(count, dtype=torch.int32, device=cuda_device)
    for chunk in (2048, 20):
        tokens, ends = generate(m, prompts, 40, lengths, chunk=chunk, repetition=1.2)
        assert ends.tolist() == [90, 47, 73] and tokens.shape == (3, 90)
        gen = Generator(m, 3, 90)
        last = [None] * 3
        for at in range(0, 50, chunk):
            n = min(chunk, 50 - at)
            c = [min(max(x - at, 0), n) for x in count]
            out = gen.step(prompts[:, at:at + n], torch.tensor(c, dtype=torch.int32, device=cuda_device))
            last = [out[b] if c[b] else last[b] for b in range(3)]
        rows = [prompts[b, :count[b]].tolist() for b in range(3)]
        logits = torch.stack(last)
        for i in range(40):
            n = torch.tensor([len(r) for r in rows], dtype=torch.int32, device=cuda_device)
            history = torch.tensor([r + [0] * (90 - len(r)) for r in rows], device=cuda_device)
            ids = process_logits(logits, history, n, repetition=1.2).argmax(-1)
            for b in range(3):
                rows[b].append(int(ids[b]))
            if i < 39:
                logits = gen.step(ids[:, None])
        for b in range(3):
            assert tokens[b, :int(ends[b])].tolist() == rows[b]


def test_penalties_masks_and_the_end(cuda_device):
    from sparseforge_amd.generate import generate

    m = _model(cuda_device, seed=3)
    prompts = torch.arange(12, device=cuda_device).view(2, 6)
    even = torch.arange(503, device=cuda_device) % 2 == 0
    tokens, _ = generate(m, prompts, 20, allowed=even)
    assert not (tokens[:, 6:] % 2).any()
    # a token is never repeated under a penalty above any logit
    tokens, ends = generate(m, prompts, 60, presence=1e4)
    assert all(len(set(row[:n].tolist())) == n for row, n in zip(tokens, ends.tolist()))
    # a grammar: after token t only t + 1 or t + 2 may follow
    def after(tokens, lengths):
        last = tokens.gather(1, lengths.long()[:, None] - 1)
        ids = torch.arange(503, device=cuda_device)[None]
        return (ids == (last + 1) % 503) | (ids == (last + 2) % 503)

    tokens, _ = generate(m, prompts, 30, allowed=after)
    step = (tokens[:, 6:] - tokens[:, 5:-1]) % 503
    assert bool(((step == 1) | (step == 2)).all())
    # the end: each sequence stops after its first end token, whenever that is
    one = torch.full((503,), -1e4, device=cuda_device)
    one[[17, 23]] = 1e4
    full, _ = generate(m, prompts, 30, bias=one, frequency=7000.0)
    tokens, ends = generate(m, prompts, 30, bias=one, frequency=7000.0, end_token=23)
    for b in range(2):
        n = int(ends[b])
        assert torch.equal(tokens[b, :n], full[b, :n]) and tokens[b, n - 1] == 23
        assert 23 not in tokens[b, 6:n - 1].tolist()
    # a random pick
    tokens, _ = generate(m, prompts, 10, pick=lambda x: torch.multinomial(x.float().softmax(-1), 1)[:, 0])
    assert bool((tokens < 503).all())


def test_refusals(cuda_device):
    from sparseforge_amd.generate import Generator, generate
    from sparseforge_amd.llama import LlamaDecoder

    m = _model(cuda_device)
    with pytest.raises(ValueError):
        generate(m, torch.zeros(2, 0, dtype=torch.int64, device=cuda_device), 3)
    with pytest.raises(ValueError):
        generate(m, torch.zeros(2, 3, device=cuda_device), 3)
    with pytest.raises(ValueError):
        generate(m, torch.zeros(2, 3, dtype=torch.int64, device=cuda_device), -1)
    with pytest.raises(ValueError):
        generate(m, torch.zeros(2, 3, dtype=torch.int64, device=cuda_device), 3,
                 torch.ones(2, dtype=torch.int64, device=cuda_device))
    gen = Generator(m, 1, 64)
    gen.step(torch.zeros(1, 60, dtype=torch.int64, device=cuda_device))
    with pytest.raises(ValueError):
        gen.step(torch.zeros(1, 5, dtype=torch.int64, device=cuda_device))
    with pytest.raises(TypeError):
        Generator(LlamaDecoder(m.config, None, device=cuda_device, dtype=torch.float32), 1, 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        Generator(LlamaDecoder(m.config, None), 1, 8)
