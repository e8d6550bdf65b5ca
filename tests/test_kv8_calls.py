"""Calls of the 8-bit cache and the rotation at the borders of what their
documentation allows: numbers near 31 bits, outputs that share memory,
derivatives, growth."""
import ctypes
import random

import pytest
import torch
from torch.autograd import forward_ad

from oracle import kv8 as O
from wnw_b200 import native as N
from wnw_b200.kv8 import KV8Attention, KV8Store
from wnw_b200.kv8_cache import KV8Cache
from wnw_b200.rotary import Apart, Rotary

gpu = pytest.mark.gpu
BF16 = torch.bfloat16


def _freq(half, base=1e4):
    return (base ** (-torch.arange(half, dtype=torch.float64) / half)).float()


@gpu
@pytest.mark.parametrize("left", [1, 40])
def test_append_behind_two_billion_rows(left):
    """A token behind almost 2^31 others: the blocks that a longer append
    would fill begin beyond 31 bits and are left alone."""
    width = (1 << 20) - 1  # pages of 2,048 rows
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    pool = torch.full((1, 64, 64 * 64 + 128), 7, dtype=torch.uint8, device="cuda")
    tk = torch.zeros(1, 2, 32, 64, dtype=BF16, device="cuda")
    s = KV8Store.wrap(pool, table, tk, torch.zeros(1, 2, 64, 32, dtype=BF16, device="cuda"))
    rows = width * 2048 - left
    k = torch.ones(1, 1, 5000, 64, dtype=BF16, device="cuda")
    s.append(k, k, torch.tensor([rows], dtype=torch.int32, device="cuda"),
             counts=torch.ones(1, dtype=torch.int32, device="cuda"))
    if left == 1:  # it fills a block whose page is none
        with pytest.raises(RuntimeError, match="out of range"):
            s.check()
    else:
        s.check()
        at = rows // 32 % 2
        want = torch.zeros_like(tk)
        want[0, at, rows % 32] = 1
        assert torch.equal(s.tail_k, want) and torch.equal(s.tail_v, want.transpose(2, 3))
    assert bool((s.pool == 7).all())


# ------------------------------------------------- derivatives of the rotation

class _OnTheCpu(Rotary):
    """The rotation with its launch replaced by the formula, for what autograd
    does around it."""

    def _launch(self, q, k, positions, inverse, out, stream):
        axis = self.axis.tolist()
        return tuple(None if x is None else O.rotate(x, positions, self.inv_freq, axis, inverse).to(x.dtype)
                     for x in (q, k))


def _forward_derivatives(rotary, device):
    g = torch.Generator().manual_seed(2)
    q, tq, gq = (torch.randn(2, 3, 5, 64, generator=g).to(device) for _ in range(3))
    k, tk, gk = (torch.randn(2, 2, 5, 64, generator=g).to(device) for _ in range(3))
    pos = torch.randint(0, 900, (2, 2, 5), generator=g).to(device)
    want = rotary(tq, tk, pos)
    for inverse in (False, True):
        turned = rotary(tq, tk, pos, inverse=inverse)
        with forward_ad.dual_level():
            for grads in (False, True):
                a, b = (x.clone().requires_grad_(grads) for x in (q, k))
                yq, yk = rotary(forward_ad.make_dual(a, tq), forward_ad.make_dual(b, tk), pos, inverse=inverse)
                assert torch.equal(forward_ad.unpack_dual(yq).tangent, turned[0])
                assert torch.equal(forward_ad.unpack_dual(yk).tangent, turned[1])
                if grads:
                    da, db = torch.autograd.grad([forward_ad.unpack_dual(y).primal for y in (yq, yk)], (a, b), (gq, gk))
                    back = rotary(gq, gk, pos, inverse=not inverse)
                    assert torch.equal(da, back[0]) and torch.equal(db, back[1])
    with forward_ad.dual_level():
        # one of the two, a broadcast tangent, no gradients recorded
        with torch.no_grad():
            yq, yk = rotary(q, forward_ad.make_dual(k, tk), pos)
        assert not forward_ad.unpack_dual(yq).tangent.any() and torch.equal(forward_ad.unpack_dual(yk).tangent, want[1])
        ones = torch.ones(1, device=device).expand(q.shape)
        y, none = rotary(forward_ad.make_dual(q, ones), None, pos)
        assert none is None and torch.equal(forward_ad.unpack_dual(y).tangent, rotary(ones.contiguous(), None, pos)[0])
        with pytest.raises(ValueError, match="gradients"):
            rotary(forward_ad.make_dual(q, tq), None, pos, out=(torch.empty_like(q), None))
        y, _ = rotary(q, None, pos)
        assert forward_ad.unpack_dual(y).tangent is None


def test_rotary_forward_derivatives_are_carried():
    _forward_derivatives(_OnTheCpu(_freq(32), sections=(10, 22)), "cpu")


@gpu
def test_rotary_forward_derivatives():
    _forward_derivatives(Rotary(_freq(32).cuda(), sections=(10, 22)), "cuda")


# -------------------------------------------------------- what calls write into

def _stale(saved, write):
    """A backward pass that needs ``saved`` as it was, after ``write``."""
    w = torch.ones(saved.shape, device=saved.device, dtype=torch.float32, requires_grad=True)
    y = (w * saved).sum() if saved.dtype is torch.float32 else (w.to(saved.dtype) * saved).sum()
    with torch.no_grad():
        write()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@gpu
def test_backward_passes_refuse_what_calls_have_overwritten():
    r = Rotary(_freq(32).cuda())
    pos = torch.arange(3, device="cuda")[None]
    q, k = torch.randn(1, 4, 3, 64, device="cuda"), torch.randn(1, 2, 3, 64, device="cuda")
    _stale(q, lambda: r(q, None, pos, out=(q, None)))
    _stale(k, lambda: r(q, k, pos, out=(torch.empty_like(q), k)))
    s = KV8Store(2, 64, 4, 2, page_rows=32)
    s.reserve(64)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    qb, kb = q.to(BF16), k.to(BF16)
    _stale(qb, lambda: s.append(kb, kb, lens, rotary=r, positions=pos, q=qb, q_out=qb))
    for held in (s.tail_k, s.tail_v, s.scales()):
        _stale(held, lambda: s.append(kb, kb, lens))
    att, out = KV8Attention(s, 2, 0.1), torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    _stale(out, lambda: att(qb[0, :, 0].reshape(2, 2, 64).contiguous(), lens, out=out))
    # what a call only reads stays good, and results made in the call are new
    w = torch.ones_like(q, requires_grad=True)
    y = (w * q).sum()
    with torch.no_grad():
        r(q, k, pos)
    y.backward()
    assert torch.equal(w.grad, q)
    with torch.inference_mode():
        x = q.clone()
        r(x, None, pos, out=(x, None))
    assert torch.equal(x, r(q, None, pos)[0])


def test_outputs_that_carry_derivatives_are_refused():
    r, q, pos = Rotary(_freq(32)), torch.zeros(1, 4, 3, 64), torch.zeros(1, 3, dtype=torch.int64)
    leaf = torch.zeros(1, 4, 3, 64, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="carries derivatives"):
            r(q, None, pos, out=(out, None))
        with pytest.raises(ValueError, match="carries derivatives"):
            r(q, q, pos, out=(torch.zeros_like(q), out))
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA device"):  # as far as the device
            r(q, None, pos, out=(out, None))
    with forward_ad.dual_level(), pytest.raises(ValueError, match="carries derivatives"):
        r(q, None, pos, out=(forward_ad.make_dual(torch.zeros_like(q), q), None))


@gpu
def test_outputs_of_the_cache_that_carry_derivatives_are_refused():
    s = KV8Store(2, 64, 2, 1, page_rows=32)
    s.reserve(32)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    kv = torch.zeros(1, 2, 3, 64, dtype=BF16, device="cuda")
    q, pos = torch.zeros(1, 4, 3, 64, dtype=BF16, device="cuda"), torch.zeros(1, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="carries derivatives"):
        s.append(kv, kv, lens, rotary=Rotary(_freq(32).cuda()), positions=pos, q=q,
                 q_out=torch.empty_like(q).requires_grad_())
    one = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="carries derivatives"):
        KV8Attention(s, 2, 0.1)(one, lens, out=torch.empty_like(one).requires_grad_())
    with torch.no_grad():
        KV8Attention(s, 2, 0.1)(one, lens, out=torch.empty_like(one).requires_grad_())
    s.check()


# ----------------------------------------------------- outputs that share memory

def test_shared_elements_are_found():
    """Against the sets of elements themselves, over random views of one buffer."""
    rnd, found = random.Random(4), [0, 0]
    buf = torch.zeros(4000)
    for _ in range(2000):
        B, H, n, D = (rnd.randint(1, 3) for _ in range(4))
        pad = [rnd.randint(0, 2) for _ in range(3)]
        order = rnd.sample(range(3), 3)
        strides, span = [0, 0, 0], D + pad[0]
        for d in order:
            strides[d] = span
            span *= (B, H, n)[d] + rnd.randint(0, 3)
        a, b = (buf.as_strided((B, h, n, D), (*strides, 1), rnd.randint(0, 40)) for h in (H, rnd.randint(1, H)))
        ids = [set((torch.arange(4000).as_strided(x.shape, x.stride(), x.storage_offset())).flatten().tolist())
               for x in (a, b)]
        share = bool(ids[0] & ids[1])
        found[share] += 1
        for x, y in ((a, b), (b, a)):
            check, at = Apart(("x", x, None), ("y", None, y)), (x.data_ptr(), None, None, y.data_ptr())
            for _ in range(2):
                if share:
                    with pytest.raises(ValueError, match="shares memory"):
                        check(*at)
                else:
                    check(*at)
    assert min(found) > 200


def test_outputs_that_share_memory_with_other_tensors_are_refused():
    r, pos = Rotary(_freq(32)), torch.zeros(2, 5, dtype=torch.int64)
    qkv = torch.zeros(2, 5, 8, 64).transpose(1, 2)
    q, k, v = qkv.split([4, 2, 2], 1)
    two = torch.zeros(2, 4, 6, 64)
    for ins, outs in (((k, v), (v, k)), ((k, v), (k, k)), ((k, v), (torch.zeros_like(k), k)),
                      ((k, v), (v, torch.zeros_like(v))),
                      ((two[:, :, :5], None), (two[:, :, 1:], None)),
                      ((two[:, :, :4], None), (two.view(-1)[:2 * 4 * 4 * 64].view(2, 4, 4, 64), None))):
        with pytest.raises(ValueError, match="shares memory"):
            r(*ins, pos[:, :ins[0].shape[2]], out=outs)
    one = torch.zeros(1, 4, 1, 64)
    for ins, outs in (((q, k), (q, k)), ((q, k), (q, torch.zeros_like(k))), ((q, None), (torch.zeros_like(q), None)),
                      ((one, None), (one.as_strided(one.shape, (7, 64, 9, 1)), None))):
        with pytest.raises(ValueError, match="CUDA device"):  # as far as the device
            r(*ins, pos[:ins[0].shape[0], :ins[0].shape[2]], out=outs)


def test_query_rows_that_share_memory_with_keys_are_refused():
    s, lens = KV8Store(4, 64, 4, 1, page_rows=64, device="cpu"), torch.zeros(4, dtype=torch.int32)
    x = torch.zeros(2, 3, 8, 64).bfloat16().transpose(1, 2)
    q, k, v = x.split([4, 2, 2], 1)
    args = dict(rotary=Rotary(_freq(32)), positions=torch.zeros(1, 2, 3, dtype=torch.int64), q=q)
    for out in (x[:, 1:5], x[:, 2:6], x[:, 4:], x[:, 3:7]):
        with pytest.raises(ValueError, match="shares memory"):
            s.append(k, v, lens, q_out=out, **args)
    for out in (q, torch.zeros_like(q)):
        with pytest.raises(ValueError, match="CUDA device"):
            s.append(k, v, lens, q_out=out, **args)


@gpu
def test_outputs_in_place_and_refused_ones_on_the_gpu():
    """In place within one packed buffer: the bits of separate outputs."""
    r, pos = Rotary(_freq(32).cuda()), torch.arange(10, device="cuda").view(2, 5)
    qkv = torch.randn(2, 5, 8, 64, device="cuda").to(BF16).transpose(1, 2)
    q, k, v = qkv.split([4, 2, 2], 1)
    want, left = r(q, k, pos), v.clone()
    with pytest.raises(ValueError, match="shares memory"):
        r(k, v, pos, out=(v, k))
    r(q, k, pos, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, left)
    s = KV8Store(4, 64, 4, 1, page_rows=32)
    s.reserve(32)
    att, lens = KV8Attention(s, 2, 0.1), torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.randn(5, 2, 64, device="cuda").to(BF16)
    with pytest.raises(ValueError, match="shares memory"):
        att(x[:4], lens, out=x[1:])
    assert not att(x[:4], lens, out=x[:4]).any()  # q itself: no rows, zeros
    s.check()


# -------------------------------------------------------------- packed queries

def test_packed_query_rows_are_taken():
    """One expanded batch may be written where samples have tokens of their
    own (as far as the device), and nowhere else."""
    s, lens = KV8Store(4, 64, 4, 1, page_rows=64, device="cpu"), torch.zeros(4, dtype=torch.int32)
    x = torch.zeros(1, 8, 9, 64).bfloat16().expand(2, -1, -1, -1)
    q, k, v = x.split([4, 2, 2], 1)
    out = torch.zeros(1, 4, 9, 64).bfloat16().expand(2, -1, -1, -1)
    args = dict(rotary=Rotary(_freq(32)), positions=torch.zeros(1, 2, 9, dtype=torch.int64), q=q)
    for to in (out, q):
        with pytest.raises(ValueError, match="CUDA device"):
            s.append(k, v, lens, counts=lens[:2], q_out=to, **args)
    with pytest.raises(ValueError, match="share memory"):
        s.append(k, v, lens, q_out=out, **args)
    with pytest.raises(ValueError, match="share memory"):
        s.append(k, v, lens, counts=lens[:2], q_out=out[:, :1].expand(2, 4, 9, 64), **args)


@gpu
def test_packed_query_rows():
    """Ragged prompts packed in one tensor, their queries into another: the
    rows of a padded output, and the rows of no sample left as they were."""
    counts, starts, total, D = [40, 1, 0, 97], [2, 42, 42, 44], 143, 128
    g = torch.Generator().manual_seed(6)
    x = torch.randn(total, 8, D, generator=g).to(BF16).cuda().transpose(0, 1)[None].expand(4, -1, -1, -1)
    q, k, v = x.split([4, 2, 2], 1)
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device="cuda")  # noqa: E731
    r, pos = Rotary(_freq(64).cuda()), torch.arange(total, device="cuda").expand(1, 4, total)
    args = dict(starts=i32(starts), counts=i32(counts), max_count=97, rotary=r, positions=pos, q=q)
    stores = [KV8Store(8, D, 32, 4, page_rows=32) for _ in range(3)]
    for s in stores:
        s.reserve(97)
    lens = i32([0] * 8)
    padded = stores[0].append(k, v, lens, **args)
    packed = torch.full((total, 4, D), 3.0, dtype=BF16, device="cuda")
    to = packed.transpose(0, 1)[None].expand(4, -1, -1, -1)
    assert stores[1].append(k, v, lens, q_out=to, **args) is to
    untouched = torch.ones(total, dtype=torch.bool)
    for b, (at, n) in enumerate(zip(starts, counts)):
        assert torch.equal(packed[at:at + n].transpose(0, 1), padded[b, :, at:at + n])
        untouched[at:at + n] = False
    assert bool((packed[untouched.cuda()] == 3).all()) and int(untouched.sum()) == 5
    own = x[0].clone()[None].expand(4, -1, -1, -1)  # in place, within the packed projection
    q, k, v = own.split([4, 2, 2], 1)
    stores[2].append(k, v, lens, q_out=q, **{**args, "q": q})
    assert torch.equal(q[0].transpose(0, 1)[~untouched.cuda()], packed[~untouched.cuda()])
    for s in stores:
        s.check()
        assert torch.equal(s.pool, stores[0].pool) and torch.equal(s.tail_k, stores[0].tail_k)


# ------------------------------------------------------------------- KV8Cache

@pytest.mark.parametrize("over,text", [
    (dict(num_q_heads=36), "group"), (dict(num_q_heads=5), "query heads"), (dict(num_q_heads=0), "group"),
    (dict(num_kv_heads=0), "query heads"), (dict(head_dim=96), "head_dim"), (dict(code="fp4"), "code"),
    (dict(page_rows=48), "page_rows"),
])
def test_cache_refuses_what_its_attention_does_not_take(over, text):
    """When it is made, not in the first decode step behind a prefill."""
    args = dict(num_layers=2, num_kv_heads=4, num_q_heads=32, head_dim=64, device="cpu")
    KV8Cache(**args)
    with pytest.raises(ValueError, match=text):
        KV8Cache(**{**args, **over})


@gpu
def test_growth_copies_seldom():
    """Steps inside the last page leave the pool where it is, and a long
    generation grows some times, not once in max_decode_tokens."""
    H, D, prompt, steps = 2, 64, 45, 700
    cache = KV8Cache(1, H, 4, D, "cuda", page_rows=128, max_decode_tokens=16)
    cache.setup_audio(torch.tensor([1]), torch.tensor([20]))
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(2, 1, H, prompt + steps, D, generator=g, device="cuda").to(BF16)
    cache.prefill_after_attn(0, None, None, *x[:, :, :, :prompt])
    cache.prefill_all_layers_done()
    q, pools, moved = torch.randn(H, 2, D, generator=g, device="cuda").to(BF16), [cache.stores[0].pool], []
    for i in range(prompt, prompt + steps):
        k, v = x[:, :, :, i:i + 1]
        cache.decode_before_attn(0, k, v)
        cache.fused_decode_attention(0, q, scale=0.125)
        cache.decode_all_layers_done()
        if cache.stores[0].pool is not pools[-1]:
            pools.append(cache.stores[0].pool)
            moved.append(i)
    cache.check()
    # pages of 128 rows: the first growth where the first page ends, the next where what it added does
    assert moved[0] == 128 and len(moved) <= 6
    whole = KV8Store(H, D, H * 6, 6, 128)
    whole.reserve(prompt + steps)
    whole.append(*x, torch.zeros(H, dtype=torch.int32, device="cuda"))
    for s in range(H):
        for a, b in zip(cache.layer_rows(0, s), whole.dequantize(s, prompt + steps)):
            assert torch.equal(a, b)


@gpu
def test_growth_within_the_pool_copies_nothing():
    s = KV8Store(2, 64, 8, 4, page_rows=32)
    s.reserve(40)
    x, lens = torch.randn(1, 2, 40, 64, device="cuda").to(BF16), torch.zeros(2, dtype=torch.int32, device="cuda")
    s.append(x, x, lens)
    t = s.grown(100)
    assert t.pool.data_ptr() == s.pool.data_ptr() and t._free == [] and int((t.page_table >= 0).sum()) == 8
    t.append(x, x, lens + 40)
    for i in range(2):
        assert torch.equal(t.dequantize(i, 40)[0][:32], s.dequantize(i, 40)[0][:32])
    u = t.grown(200)
    assert u.pool.shape[0] == 14 and torch.equal(u.pool[:8], t.pool)
    u.check()


def test_numbers_of_pages_that_wrap_around_are_refused():
    """Checked on the host: 2^58 pages of 64 blocks are 2^64."""
    for pages in (1 << 58, (1 << 57) + 1, 1 << 31):
        d = N.Kv8StoreDesc(dtype=N.BF16, head_dim=64, code=0, num_segs=2, pool=4096, num_pages=pages, page_blocks=64,
                           page_table=4096, max_pages=2, tail_k=4096, tail_v=4096, err=4096)
        a = N.Kv8AppendArgs(store=d, batch=1, num_kv_heads=2, tokens=4, max_count=4, seg_len=4096, k=4096, v=4096)
        b = N.Kv8AttnArgs(store=d, group=4, q=4096, seg_len=4096, out=4096, scale=1.0, partials=4096,
                          partial_floats=1 << 30, counters=4096)
        for call, args in ((N.lib.wnw_kv8_append, a), (N.lib.wnw_kv8_attn, b)):
            assert call(ctypes.byref(args), None) == N.WNW_ERR_INVALID
            assert "blocks" in N.lib.wnw_last_error().decode()


@pytest.mark.parametrize("hq,hk", [(1 << 30, 1 << 30), ((1 << 31) - 1, 1), ((1 << 31) - 1, (1 << 31) - 1),
                                   (1 << 20, 1)])
def test_numbers_of_heads_that_wrap_around_are_refused(hq, hk):
    a = N.RotaryArgs(dtype=N.BF16, head_dim=64, batch=1, tokens=2, num_q_heads=hq, num_kv_heads=hk, q=4096, q_out=4096,
                     k=8192, k_out=8192, err=4096,
                     rope=N.Rope(rot=64, num_axes=1, inv_freq=4096, axis=4096, pos=4096))
    assert N.lib.wnw_rotary(ctypes.byref(a), None) == N.WNW_ERR_INVALID
    assert "heads" in N.lib.wnw_last_error().decode()


# ------------------------------------------------- captured, and large and small heads

@gpu
def test_captured_steps_with_fresh_tokens():
    """A decode step as a loop runs it, the attention early behind the append,
    captured once and replayed over growing sequences that finish blocks and
    begin pages: the bits of one that waits."""
    B, H, G, D, n, steps = 3, 2, 4, 64, 57, 80
    g = torch.Generator(device="cuda").manual_seed(8)
    store = KV8Store(B * H, D, B * H * 5, 5, page_rows=32)
    store.reserve(n + steps + 2)
    r, att, other = Rotary(_freq(32).cuda()), *(KV8Attention(store, G, 0.125) for _ in range(2))
    lens = torch.tensor([0, 31, 32, 57, 5, 40], dtype=torch.int32, device="cuda")
    kv = torch.randn(B * H, 1, n, D, generator=g, device="cuda").to(BF16)
    KV8Store.wrap(store.pool, store.page_table, store.tail_k, store.tail_v).append(kv, kv, lens * 0, counts=lens)
    x = torch.randn(B, H * (G + 2), 1, D, generator=g, device="cuda").to(BF16)
    new, pos = lens + 1, torch.full((1, B, 1), 57, dtype=torch.int64, device="cuda")

    def step():
        q = store.append(x[:, H * G:H * G + H], x[:, -H:], lens, rotary=r, positions=pos, q=x[:, :H * G])
        out, lse = att(q.view(B * H, G, D), new, return_lse=True, fresh=1)
        lens.add_(1)
        new.add_(1)
        pos.add_(1)
        return q, out, lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out, lse = step()
    for _ in range(steps):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        graph.replay()
        want = other(q.view(B * H, G, D), lens, return_lse=True)  # lens: the step's new ones by now
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    store.check()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, BF16])
@pytest.mark.parametrize("D,rot,Hq,Hk,n", [(512, 512, 3, 1, 700), (512, 16, 1, 2, 9), (16, 16, 40, 0, 3000),
                                          (496, 240, 2, 2, 301), (32, 16, 1, 1, 1), (128, 128, 1, 0, 1)])
def test_rotary_large_and_small_heads(dtype, D, rot, Hq, Hk, n):
    """Tolerance as derived in test_rotary.py: the type's rounding, and 2^-22
    of both magnitudes for the fp32 cosine, sine, products and sum."""
    g = torch.Generator().manual_seed(D + n)
    r = Rotary(_freq(rot // 2).cuda())
    pos = torch.randint(0, 10 ** 6, (1, 2, n), generator=g)
    x = [torch.randn(2, h, n, D, generator=g).to(dtype) for h in (Hq, Hk)]
    got = r(x[0].cuda(), x[1].cuda() if Hk else None, pos.cuda())
    for y, z in zip(got, x[:2 if Hk else 1]):
        want = O.rotate(z, pos, r.inv_freq.cpu(), [0] * (rot // 2))
        m = z.double().abs()
        both = m[..., :rot // 2] + m[..., rot // 2:rot]
        mag = torch.cat([both, both, torch.zeros_like(m[..., rot:])], -1)
        tiny = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, BF16: 2.0 ** -134}[dtype]
        tol = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -7) + 2.0 ** -22 * mag + tiny
        assert bool(((y.cpu().double() - want).abs() <= tol).all())
    r.check()
