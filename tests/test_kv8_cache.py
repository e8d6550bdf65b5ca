"""``KV8Cache`` and ``RotaryAdapter`` under the session: a tiny random-init
Llama through ``model.generate``.  What each layer is given and gives back is
recorded; the rows the cache reads back are checked against those it was given
(within the codes' steps, see test_kv8.py), and each attention output against
attention in 64 bits over the rows read back.
"""
import pytest
import torch

from oracle import kv8 as O

gpu = pytest.mark.gpu
VOCAB, L, HQ, H, D = 97, 2, 4, 2, 64


def _model(device, **kw):
    from transformers import LlamaConfig, LlamaForCausalLM
    torch.manual_seed(0)
    c = LlamaConfig(vocab_size=VOCAB, hidden_size=HQ * D, intermediate_size=128, num_hidden_layers=L,
                    num_attention_heads=HQ, num_key_value_heads=H, head_dim=D, max_position_embeddings=512,
                    attn_implementation="sdpa", **kw)
    return LlamaForCausalLM(c).to(torch.bfloat16).to(device).eval()


def _recording(cache):
    """The cache with everything it is handed and returns kept, on the CPU."""
    log = {"prompt": {}, "new": [], "out": []}
    prefill, attend = cache.prefill_after_attn, cache.fused_decode_attention

    def prefill_after_attn(l, ca, ph, k, v):
        log["prompt"][l] = (k.cpu(), v.cpu())
        prefill(l, ca, ph, k, v)

    def fused_decode_attention(l, q_flat, q, k_flat, v_flat, cu, scale):
        rot = cache._rotation
        k, v = cache._new[l]
        log["new"].append((l, k.cpu(), v.cpu(), None if rot is None else rot[1].cpu()))
        out = attend(l, q_flat, q, k_flat, v_flat, cu, scale)
        log["out"].append((l, q_flat.cpu(), out.cpu(), scale,
                           [[x.cpu().double() for x in cache.stores[l].dequantize(s, int(cache._next[s]))]
                            for s in range(cache.batch_size * H)]))
        return out

    cache.prefill_after_attn, cache.fused_decode_attention = prefill_after_attn, fused_decode_attention
    return log


@gpu
@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("own_rotation", [False, True])
def test_session_over_the_8_bit_cache(code, own_rotation):
    from wnw_b200 import KV8Cache, LlamaFamilyAdapter, RotaryAdapter, WnWSession
    model = _model("cuda")
    freq = model.model.rotary_emb.inv_freq.cpu()
    n, steps = 45, 40
    ids = torch.randint(1, VOCAB, (2, n), generator=torch.Generator().manual_seed(1)).cuda()
    mask = torch.ones_like(ids)
    mask[1, :13] = 0  # left padding
    cache = KV8Cache(L, H, HQ, D, "cuda", code=code, page_rows=32, max_decode_tokens=16)  # grows twice
    log = _recording(cache)
    adapter = RotaryAdapter(2, 30) if own_rotation else LlamaFamilyAdapter(2, 30)
    with WnWSession(model, adapter, cache) as sess:
        sess.setup_audio(ids, mask)
        out = sess.generate({"input_ids": ids, "attention_mask": mask}, max_new_tokens=steps + 1, do_sample=False,
                            pad_token_id=0, eos_token_id=None)
        assert out.shape == (2, n + steps + 1)
        cache.check()
    eps = torch.finfo(torch.bfloat16).eps
    pads = [0, 13]
    for l in range(L):
        news = [x for x in log["new"] if x[0] == l]
        assert len(news) == steps
        for s in range(2 * H):
            b, h = divmod(s, H)
            k = [log["prompt"][l][0][b, h, pads[b]:].double()]
            v = [log["prompt"][l][1][b, h, pads[b]:].double()]
            for _, nk, nv, pos in news:
                x = nk[b:b + 1].double()
                if own_rotation:
                    assert pos.shape == (1, 2, 1)
                    x = O.rotate(x, pos[:, b:b + 1], freq, [0] * (D // 2)).to(torch.bfloat16).double()
                k.append(x[0, h])
                v.append(nv[b, h].double())
            rows = cache.layer_rows(l, s)
            for got, want, e in ((rows[0], torch.cat(k), eps if own_rotation else 0.0), (rows[1], torch.cat(v), 0.0)):
                got = got.cpu().double()
                assert got.shape == want.shape
                for j in range(0, got.shape[0], 32):
                    blk = want[j:j + 32]
                    if blk.shape[0] < 32:
                        tol = e * blk.abs()
                    else:
                        sc = O.block_scale(blk, code)
                        tol = O.half_step(blk, sc, code) * (1 + 16 * e) + (2.0 ** -20 + 2 * e) * blk.abs() + e * sc
                    assert bool(((got[j:j + 32] - blk).abs() <= tol).all())
    for i, (l, q, out, scale, rows) in enumerate(log["out"]):
        if own_rotation:  # positions: the step's, behind each sample's padding
            pos = log["new"][i][3]
            q = O.rotate(q.reshape(2, HQ, 1, D), pos, freq, [0] * (D // 2)).to(torch.bfloat16).view(2 * H, HQ // H, D)
        for s, (k, v) in enumerate(rows):
            want, _, pv = O.attention(q[s].double(), k, v, scale)
            # the 64-bit rotation's rounding may take the other neighbour: 2^-8 of each score's terms at most
            slack = 2.0 ** -8 * scale * float((q[s].double().abs() @ k.abs().t()).max()) if own_rotation else 0.0
            tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * slack) * pv + k.shape[0] * 2.0 ** -25 * float(v.abs().max())
            assert bool(((out[s].double() - want).abs() <= tol).all())


@gpu
def test_own_rotation_matches_the_models():
    """The same prompt's logits with the model's tables (rounded to bf16) and
    with positions: as close as those roundings allow; the model is as before
    afterwards."""
    from wnw_b200 import KV8Cache, LlamaFamilyAdapter, RotaryAdapter, WnWSession
    model = _model("cuda")
    forward = model.model.rotary_emb.forward
    ids = torch.randint(1, VOCAB, (1, 60), generator=torch.Generator().manual_seed(2)).cuda()
    logits = []
    for adapter in (LlamaFamilyAdapter(2, 30), RotaryAdapter(2, 30)):
        cache = KV8Cache(L, H, HQ, D, "cuda")
        with WnWSession(model, adapter, cache) as sess:
            sess.setup_audio(ids)
            logits.append(model(ids, past_key_values=cache).logits.detach().float())
        assert model.model.rotary_emb.forward == forward
    rel = float((logits[0] - logits[1]).norm() / logits[0].norm())
    # a rounding to bf16 of tables, products and sums in each of two layers against one: a few times 2^-8
    assert rel <= 8 * 2.0 ** -8


@gpu
def test_sections_of_positions():
    """Positions of several axes reach the rotation; 2-D ones count for every
    axis."""
    from wnw_b200 import RotaryAdapter
    model = _model("cuda")
    a = RotaryAdapter(2, 30, sections=(8, 12, 12))
    state = a.prepare_for_inference(model)
    x = torch.zeros(2, 5, HQ * D, device="cuda", dtype=torch.bfloat16)
    p3 = torch.randint(0, 99, (3, 2, 5), device="cuda")
    q = torch.randn(2, HQ, 5, D, device="cuda", dtype=torch.bfloat16)
    k = torch.randn(2, H, 5, D, device="cuda", dtype=torch.bfloat16)
    pe = model.model.rotary_emb(x, p3)
    assert torch.equal(pe[0], p3)
    got = a.apply_rope(q, k, pe, None)
    axis = [0] * 8 + [1] * 12 + [2] * 12
    freq = model.model.rotary_emb.inv_freq.cpu()
    for y, z in zip(got, (q, k)):
        want = O.rotate(z.cpu(), p3.cpu(), freq, axis)
        assert bool(((y.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18).all())
    one = model.model.rotary_emb(x, torch.arange(5, device="cuda")[None])[0]
    assert one.shape == (3, 2, 5) and torch.equal(one[2, 1], torch.arange(5, device="cuda"))
    a.restore_after_inference(model, state)
    assert a.rotary is None


@gpu
def test_grown_store_keeps_its_content():
    from wnw_b200.kv8 import KV8Attention, KV8Store
    s = KV8Store(4, D, 4, 1, page_rows=64)
    s.reserve(64)
    k = torch.randn(2, 2, 61, D, device="cuda").bfloat16()
    zero = torch.zeros(4, dtype=torch.int32, device="cuda")
    s.append(k, k, zero)
    q = torch.randn(4, 2, D, device="cuda").bfloat16()
    one = KV8Attention(s, 2, 0.1)
    a = one(q, zero + 61)
    t = s.grown(500)
    two = KV8Attention(t, 2, 0.1, scratch_of=one)
    assert two.partials is one.partials
    assert torch.equal(a, two(q, zero + 61))
    t.append(k, k, zero + 61)
    for x, y in zip(t.dequantize(3, 61), s.dequantize(3, 61)):
        assert torch.equal(x[:32], y[:32])
    t.check()
    with pytest.raises(ValueError, match="scratch"):
        KV8Attention(t, 3, 0.1, scratch_of=one)


@gpu
def test_fresh_tokens():
    """The attention directly behind an append that it need not wait for in
    full: the same bits as one that waits, whether the append finishes blocks
    or not."""
    from wnw_b200.kv8 import KV8Attention, KV8Store
    g = torch.Generator().manual_seed(0)
    n = 2000
    for S, fresh in ((6, 1), (6, 40), (6, 3000), (300, 1)):
        s = KV8Store(S, D, S * 40, 40, page_rows=64)
        s.reserve(64 * 40)
        k = torch.randn(S, 1, n, D, generator=g).bfloat16().cuda()
        lens = torch.tensor([0, 1, 31, 63, 1500, 1999] * (S // 6), dtype=torch.int32, device="cuda")
        zero = torch.zeros(S, dtype=torch.int32, device="cuda")
        s.append(k, k, zero, counts=lens)
        q = torch.randn(S, 4, D, generator=g).bfloat16().cuda()
        att = KV8Attention(s, 4, 0.125)
        m = min(fresh, 60)
        x = torch.randn(S, 1, m, D, generator=g).bfloat16().cuda()
        after = lens + m
        torch.cuda.synchronize()
        s.append(x, x, lens)
        got = att(q, after, fresh=fresh)
        want = att(q, after)
        assert torch.equal(got, want)
        s.check()


def test_session_asks_no_scores_of_the_8_bit_cache():
    from wnw_b200.session import _no_scores
    from wnw_b200.kv8_cache import KV8Cache
    assert _no_scores(1, 2) == (None, None) and KV8Cache.needs_prefill_scores is False
    c = KV8Cache(2, 2, 4, 64, "cpu")
    c.setup_audio(torch.tensor([1, 2]), torch.tensor([3, 4]), torch.tensor([[0, 1, 1, 1, 1], [1, 1, 1, 1, 1]]))
    assert c._pads == [1, 0] and c.batch_size == 2
    assert c._snapshot_cache_stats() == []
    with pytest.raises(ValueError, match="one at a time"):
        c.decode_before_attn(0, torch.zeros(2, 2, 3, 64), torch.zeros(2, 2, 3, 64))
    with pytest.raises(NotImplementedError):
        c.crop(1)


def test_rotary_adapter_refuses_changing_frequencies():
    from wnw_b200 import RotaryAdapter
    model = _model("cpu", rope_parameters={"rope_type": "dynamic", "factor": 2.0, "rope_theta": 1e4})
    with pytest.raises(ValueError, match="must not depend"):
        RotaryAdapter(0, 1).prepare_for_inference(model)


def test_rotary_adapter_refuses_interleaved_sections():
    from types import SimpleNamespace
    from wnw_b200 import RotaryAdapter
    params = {"rope_type": "default", "mrope_section": [2, 3, 3], "mrope_interleaved": True}
    m = SimpleNamespace(rotary_emb=SimpleNamespace(
        rope_type="default", inv_freq=torch.ones(8), config=SimpleNamespace(rope_parameters=params), forward=None))
    with pytest.raises(ValueError, match="interleaved"):
        RotaryAdapter(0, 1).prepare_for_inference(m)
    params["mrope_interleaved"] = False
    a = RotaryAdapter(0, 1)
    a.prepare_for_inference(m)
    assert a.rotary.num_axes == 3


def test_a_session_that_cannot_be_entered_leaves_the_model_alone():
    """The second layer's patch fails: the first layer's forward and the rotary
    module's are the model's own again."""
    from wnw_b200 import KV8Cache, RotaryAdapter, WnWSession
    model = _model("cpu")

    class Failing(RotaryAdapter):
        def attention_meta(self, attn):
            if attn.layer_idx == 1:
                raise RuntimeError("no such layer")
            return super().attention_meta(attn)

    ids = torch.arange(1, 9)[None]
    with torch.no_grad():
        want = model(ids).logits
    session = WnWSession(model, Failing(2, 5), KV8Cache(L, H, HQ, D, "cpu"))
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no such layer"):
            session.__enter__()
        assert session.adapter.rotary is None and not session._orig
        with torch.no_grad():
            assert torch.equal(model(ids).logits, want)
