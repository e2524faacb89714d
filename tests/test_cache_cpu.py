"""Rotary positions and the paged cache: the CPU path, and what calls refuse."""
import math

import pytest
import torch

from gonn_b200 import nn
from gonn_b200.ops.rotary import turns_of


def test_fixed_point_angles():
    """p times the fraction of a turn, modulo 2^64, against the exact product."""
    from fractions import Fraction
    w = nn.RotaryEmbedding(64, 500000.0)._w
    for f, t in zip(w, turns_of(w).tolist()):
        turn = Fraction(f / (2 * math.pi))
        for p in (0, 1, 4095, 131071, 2 ** 31 - 1, -5):
            got = Fraction(t * p % 2 ** 64, 2 ** 64)
            want = turn * p % 1
            d = abs(got - want)
            assert min(d, 1 - d) <= Fraction(abs(p) + 1, 2 ** 65)


@pytest.mark.parametrize("inter", [False, True])
def test_rotary_keeps_lengths_and_relative_positions(inter):
    rope = nn.RotaryEmbedding(6, interleaved=inter)
    x, y = torch.randn(2, 1, 1, 1, 8, dtype=torch.float64)
    at = torch.arange(50)
    a, b = rope(x.expand(1, 50, 1, 8), at)[0, :, 0], rope(y.expand(1, 50, 1, 8), at)[0, :, 0]
    assert torch.allclose(a.norm(dim=-1), x.norm().expand(50))
    assert torch.allclose((a[3:] * b[:-3]).sum(-1), (a[3] * b[0]).sum().expand(47))
    assert torch.equal(a[:, 6:], x.view(8)[6:].expand(50, 2))
    assert torch.equal(a[0], x.view(8))


def test_rotary_gradient():
    rope = nn.RotaryEmbedding(4, interleaved=True, scaling="linear", factor=3.0, amplitude=1.2)
    x = torch.randn(2, 3, 2, 5, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: rope(t, torch.tensor([5, 9, 100])), (x,))


def test_scalings():
    plain = nn.RotaryEmbedding(64)._w
    assert nn.RotaryEmbedding(64, scaling="linear", factor=4.0)._w == [f / 4 for f in plain]
    base = nn.RotaryEmbedding(64, scaling="base", factor=4.0)._w
    assert base[0] == plain[0] and math.isclose(base[-1], plain[-1] / 4)
    bands = nn.RotaryEmbedding(64, scaling="bands", factor=4.0, original=4096)._w
    for f, g in zip(plain, bands):
        turns = 4096 * f / (2 * math.pi)
        assert g == f if turns >= 32 else math.isclose(g, f / 4) if turns <= 1 else f / 4 < g < f


def test_module():
    rope = nn.NewRotaryEmbedding(8)
    assert not list(rope.parameters()) and not rope.state_dict()
    assert rope.to(torch.bfloat16).turns.dtype == torch.int64


def steps(B, kv, H, D, page, pieces, shared=0, dtype=torch.float64):
    """Tokens appended and attended piece by piece, and the same by attention over all of them at once."""
    T = sum(pieces)
    columns = -(-T // page)
    cache = nn.KVCache(B * columns + shared, page, kv, D, dtype=dtype)
    table = torch.randperm(B * columns).view(B, columns).to(torch.int32)
    q, k, v = (torch.randn(B, T, h, D, dtype=dtype) for h in (H, kv, kv))
    if shared:
        table[1:, :shared] = table[0, :shared]
        k[1:, :shared * page], v[1:, :shared * page] = k[0, :shared * page], v[0, :shared * page]
    rope = nn.RotaryEmbedding(D // 2 * 2)
    lengths, outs = torch.zeros(B, dtype=torch.int32), []
    for n in pieces:
        at = int(lengths[0])
        piece = slice(at, at + n)
        x = cache.Append(k[:, piece], v[:, piece], table, lengths, rotary=rope, q=q[:, piece])
        outs.append(cache.Attend(x, table, lengths, shared_pages=shared if at >= shared * page else 0))
        lengths += n
    qr, kr = rope(q), rope(k).repeat_interleave(H // kv, 2)
    s = torch.einsum("bthd,bnhd->bhtn", qr, kr) / math.sqrt(D)
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), -math.inf)
    want = torch.einsum("bhtn,bnhd->bthd", torch.softmax(s, -1), v.repeat_interleave(H // kv, 2))
    return torch.cat(outs, 1), want


@pytest.mark.parametrize("pieces", [[1] * 9, [5, 1, 1, 4], [20], [16, 3]])
def test_pieces(pieces):
    got, want = steps(2, 2, 6, 8, 4, pieces)
    assert torch.allclose(got, want)


def test_shared_pages():
    got, want = steps(3, 1, 2, 6, 4, [8, 1, 2], shared=2)
    assert torch.allclose(got, want)


def test_padded_batch():
    cache = nn.KVCache(6, 4, 1, 4)
    table, lengths = torch.arange(6, dtype=torch.int32).view(3, 2), torch.tensor([0, 3, 1], dtype=torch.int32)
    counts = torch.tensor([2, 0, 3], dtype=torch.int32)
    q, k, v = (torch.randn(3, 3, 1, 4) for _ in range(3))
    before = cache.Keys.clone()
    out = cache.Append(k, v, table, lengths, counts=counts, q=q)
    assert torch.equal(out[0, :2], q[0, :2]) and not bool(out[0, 2:].any()) and not bool(out[1].any())
    assert torch.equal(cache.Keys[0, 0, :2], k[0, :2, 0]) and torch.equal(cache.Keys[2:4], before[2:4]) and not bool(cache.Keys[0, 0, 2:].any())
    y = cache.Attend(q, table, lengths, counts=counts)
    assert not bool(y[1].any()) and not bool(y[0, 2].any()) and bool(y[2].any())
    assert torch.allclose(y[0, 0], v[0, 0])                    # the first position sees itself alone


def test_refusals():
    i32 = dict(dtype=torch.int32)
    cache = nn.KVCache(4, 16, 2, 8)
    k, q = torch.zeros(2, 1, 2, 8), torch.zeros(2, 1, 4, 8)
    table, at = torch.zeros(2, 1, **i32), torch.zeros(2, **i32)
    for bad in (dict(dim=0), dict(dim=3), dict(dim=2050), dict(dim=4, scaling="other"), dict(dim=2, scaling="base"), dict(dim=4, factor=0.0),
                dict(dim=4, scaling="bands"), dict(dim=4, scaling="bands", original=8, low=4, high=4), dict(dim=4, base=-1.0)):
        with pytest.raises(ValueError):
            nn.RotaryEmbedding(**bad)
    rope = nn.RotaryEmbedding(8)
    for x, p, error in ((torch.zeros(2, 8), None, ValueError), (torch.zeros(1, 1, 1, 6), None, ValueError), (k, torch.zeros(2, 2, **i32), ValueError),
                        (k, torch.zeros(1), TypeError), (k.int(), None, TypeError)):
        with pytest.raises(error):
            rope(x, p)
    for shape in ((0, 1, 1, 1), (1, 0, 1, 1)):
        with pytest.raises(ValueError):
            nn.KVCache(*shape)
    with pytest.raises(ValueError):
        nn.KVCache.Over(torch.zeros(1, 2, 3, 4), torch.zeros(1, 2, 3, 5))
    with pytest.raises(TypeError):
        nn.KVCache(1, 1, 1, 1, dtype=torch.int8)
    for args, error in (((k[..., :4], k[..., :4], table, at), ValueError), ((k[:, :, :1], k, table, at), ValueError), ((k.double(), k, table, at), TypeError),
                        ((k, k, table.long(), at), TypeError), ((k, k, table, at[:1]), ValueError), ((k, k, table[:, :0], at), ValueError),
                        ((k, k, table, at + 16), ValueError), ((k, k, table, at - 1), ValueError), ((k, k, table + 4, at), ValueError),
                        ((k, k, torch.zeros(2, 2 ** 27, **i32).expand(2, 2 ** 27), at), ValueError)):
        with pytest.raises(error):
            cache.Append(*args)
    with pytest.raises(ValueError):
        cache.Append(k, k, table, at, rotary=nn.RotaryEmbedding(10))
    with pytest.raises(ValueError):
        cache.Append(k, k, table, at, q=q[:1])
    for kw, error in ((dict(q=q[:, :, :3]), ValueError), (dict(q=q[..., :4]), ValueError), (dict(q=q.half()), TypeError), (dict(shared_pages=2), ValueError),
                      (dict(shared_pages=-1), ValueError), (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError), (dict(scale=math.inf), ValueError),
                      (dict(lengths=at + 16), ValueError), (dict(table=table - 1), ValueError), (dict(counts=at.long()), TypeError)):
        with pytest.raises(error):
            cache.Attend(**{**dict(q=q, table=table, lengths=at), **kw})
    grad = q.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        cache.Attend(grad, table, at)
    with torch.no_grad():
        cache.Attend(grad, table, at)


# ------------------------------------------------------------------------------------------------------------------ layers and models
def test_attention_with_rotary():
    """The layer with rotary positions: relative to each other, gradients by differences, in pieces from a cache."""
    torch.manual_seed(1)
    mha = nn.MultiHeadAttention(12, 2, rotary=nn.RotaryEmbedding(4, interleaved=True), dtype=torch.float64)
    x = torch.randn(2, 5, 12, dtype=torch.float64)
    whole = mha(x, causal=True)
    assert not torch.allclose(whole, nn.MultiHeadAttention.forward(_without_rotary(mha), x, causal=True))
    assert torch.allclose(mha.ForwardMasked(x, causal=True), whole)
    assert torch.autograd.gradcheck(lambda t: mha(t, causal=True), (x[:1, :3].clone().requires_grad_(),))
    cache = nn.KVCache(4, 4, 2, 6, dtype=torch.float64)
    table, at, outs = torch.tensor([[3, 0], [1, 2]], dtype=torch.int32), torch.zeros(2, dtype=torch.int32), []
    with torch.no_grad():
        for piece in x.split([2, 1, 2], 1):
            outs.append(mha.ForwardCached(piece, cache, table, at))
            at += piece.shape[1]
    assert torch.allclose(torch.cat(outs, 1), whole)
    with pytest.raises(ValueError):
        nn.MultiHeadAttention(12, 2, rotary=nn.RotaryEmbedding(8))


def _without_rotary(mha):
    import copy
    other = copy.deepcopy(mha)
    other.__dict__["rotary"] = None
    return other


@pytest.mark.parametrize("rotary", [None, True, dict(dim=4, interleaved=True, scaling="linear", factor=2.0)])
def test_generate(rotary):
    """Greedy continuation from the cache is that of the whole sequence computed anew for every token."""
    from gonn_b200.models import GPT
    torch.manual_seed(2)
    model = GPT(vocab=31, d_model=16, n_layers=2, n_heads=2, d_ff=24, max_seq=32, rotary=rotary, dtype=torch.float64)
    assert (model.pos is None) == (rotary is not None)
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() > 1:
                p.normal_(0, 0.5)
    ids = torch.randint(0, 31, (2, 7))
    want = ids
    with torch.no_grad():
        for _ in range(9):
            want = torch.cat((want, model(want)[:, -1].argmax(-1, keepdim=True)), 1)
    assert torch.equal(model.Generate(ids, 9, page_size=4), want)
    assert torch.equal(model.Generate(ids[:1], 9, samples=3, page_size=4), want[:1].expand(3, -1))
    assert torch.equal(model.Generate(ids[:1], 9, samples=3, page_size=7), want[:1].expand(3, -1))
    drawn = model.Generate(ids[:1], 5, samples=4, temperature=1.0, page_size=4)
    assert drawn.shape == (4, 12) and torch.equal(drawn[:, :7], ids[:1].expand(4, -1))
    assert torch.equal(model.Generate(ids, 0), ids)
    for bad in (dict(new_tokens=-1), dict(new_tokens=1, samples=2), dict(new_tokens=1, samples=0)):
        with pytest.raises(ValueError):
            model.Generate(ids, **bad)
    if rotary is None:
        with pytest.raises(ValueError):
            model.Generate(ids, 26)


def test_steps_behind_the_last_learned_position():
    """Refused as ``forward`` refuses them; tokens that do not count may lie there."""
    from gonn_b200.models import GPT
    torch.manual_seed(6)
    model = GPT(vocab=31, d_model=16, n_layers=1, n_heads=2, d_ff=24, max_seq=8, dtype=torch.float64)
    ids = torch.randint(0, 31, (2, 12))
    table, at = torch.arange(6, dtype=torch.int32).view(2, 3), torch.zeros(2, dtype=torch.int32)
    with torch.no_grad():
        with pytest.raises(IndexError):
            model(ids)
        with pytest.raises(IndexError):
            model.Step(ids, model.Caches(6, 4), table, at)
        caches = model.Caches(6, 4)
        whole = model.Step(ids[:, :8], caches, table, at)
        assert torch.allclose(whole, model(ids[:, :8]))
        with pytest.raises(IndexError):
            model.Step(ids[:, 8:9], caches, table, at + 8)
        padded = model.Step(ids, model.Caches(6, 4), table, at, counts=torch.tensor([8, 3], dtype=torch.int32))
        # (attention over 3 positions and over 8 may add in another order: at most 24 terms a sum, 24 2^-53 of their magnitudes, a few sums in a row)
        assert torch.equal(padded[0, :8], whole[0]) and torch.allclose(padded[1, :3], whole[1, :3], rtol=1e-12, atol=1e-12)


def test_positions_changed_behind_the_tape(monkeypatch):
    """The gradient's turn needs the positions of the forward's: the tape tells that they have been written over."""
    from gonn_b200.ops import rotary
    rope = nn.RotaryEmbedding(4)

    def launch(x, positions, turns, interleaved, amplitude, back, out=None):       # the kernel's part, on the CPU
        return rotary.rotate_ref(x.detach(), positions, rope._w, interleaved, amplitude, back)
    monkeypatch.setattr(rotary, "_launch", launch)
    x, at = torch.randn(1, 3, 2, 4, requires_grad=True), torch.arange(3)
    call = lambda: rotary._Rotary.apply(x, at, rope.turns, False, 1.0, False)
    dx, = torch.autograd.grad(call().sum(), x)
    assert torch.allclose(dx, rotary.rotate_ref(torch.ones_like(x), at, rope._w, False, 1.0, True))
    y = call()
    at += 3
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_checkpoints_leave_frequencies_alone(tmp_path):
    """Frequencies follow from a module's options: a model saved with others, or before it had any, loads, and keeps its own."""
    from gonn_b200.utils import checkpoint

    class Layer(nn.Module):
        def __init__(self, rope):
            super().__init__()
            self.proj, self.rope = nn.Linear(4, 4), rope
    path, plain = str(tmp_path / "x"), nn.RotaryEmbedding(8)
    first, other = Layer(plain), Layer(nn.RotaryEmbedding(8, scaling="linear", factor=4.0))
    want = other.rope.turns.clone()
    for source in (first, Layer(None)):
        checkpoint.save(path, source)
        checkpoint.load(path, other)
        assert torch.equal(other.rope.turns, want) and torch.equal(other.proj.weight, source.proj.weight)


def test_steps_of_a_layer_under_a_tape_are_refused():
    """Nothing has a gradient through a cache: refused wherever the input or a projection into the cache would need one."""
    mha = nn.MultiHeadAttention(16, 2, dtype=torch.float64)
    cache, x = nn.KVCache(1, 4, 2, 8, dtype=torch.float64), torch.randn(1, 1, 16, dtype=torch.float64)
    table, at = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        mha.ForwardCached(x, cache, table, at)
    with torch.no_grad():
        want = mha.ForwardCached(x, cache, table, at)
    for p in mha.parameters():
        p.requires_grad_(False)
    with pytest.raises(RuntimeError):
        mha.ForwardCached(x.clone().requires_grad_(), cache, table, at)
    assert torch.equal(mha.ForwardCached(x, cache, table, at), want)
    mha.outproj.weight.requires_grad_(True)                            # behind the cache: a gradient like any other
    mha.ForwardCached(x, cache, table, at).sum().backward()
    assert mha.outproj.weight.grad is not None
    # the value's projection alone: its keys and queries need none
    mha.vproj.bias.requires_grad_(True)
    with pytest.raises(RuntimeError):
        mha.ForwardCached(x, cache, table, at)


def test_fused_steps_under_a_tape_are_refused(monkeypatch):
    """The product of all three projections at once, which only CUDA takes, refuses them alike: here it would not be reached."""
    from gonn_b200.nn import attention
    mha, called = nn.MultiHeadAttention(16, 2), []
    monkeypatch.setattr(attention, "fused_view", lambda parts: called.append(1))
    table, at = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        mha.ForwardCached(torch.randn(1, 1, 16), nn.KVCache(1, 4, 2, 8), table, at)
    assert not called


def test_caches_in_tensors_that_need_a_gradient():
    q, k = torch.randn(1, 1, 2, 8), torch.randn(1, 1, 2, 8)
    table, at = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for which in range(2):
        tensors = [torch.zeros(1, 2, 4, 8) for _ in range(2)]
        cache = nn.KVCache.Over(*tensors)
        tensors[which].requires_grad_()
        for call in (lambda: cache.Append(k, k, table, at), lambda: cache.Attend(q, table, at)):
            with pytest.raises(RuntimeError, match="under torch.no_grad"):
                call()
            with torch.no_grad():
                call()


def test_tables_of_nearly_2_to_the_31_positions():
    """A tile's last key is counted in 32 bits: tables whose last tile would pass them are refused, by the native library too, and so are rows of
    queries."""
    from gonn_b200 import lib
    q = torch.zeros(0, 1, 1, 8)
    table, at = torch.zeros(0, 1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    for page, fits in ((2 ** 31 - 257, True), (2 ** 31 - 256, False), (2 ** 31 - 2, False)):
        cache = nn.KVCache.Over(*(torch.zeros(1, 1, 1, 8).expand(1, 1, page, 8) for _ in range(2)))
        for call in (lambda: cache.Attend(q, table, at), lambda: cache.Append(q, q, table, at)):
            if fits:
                call()
            else:
                with pytest.raises(ValueError):
                    call()
        assert (lib.lib().gb_cache_attn_bytes(0, 1, 1, 1, 1, 8, 0, page) >= 0) == fits
        assert (lib.lib().gb_cache_attn_bytes(0, 1, page, 1, 1, 8, 0, 1024) >= 0) == fits


def test_sizes_beyond_32_bits_are_refused():
    """By the native entries, before any launch (2^32 tokens were none)."""
    from gonn_b200 import lib
    from gonn_b200.ops.rotary import words
    at, big = 256, 2 ** 32                                              # an address, looked at by nobody
    rotary = [64, 64, 64, 64, 64, 64, 1, 0, 1, 64, 0, 0, 0, 0, 0, 0]
    append = [64] * 15 + [1, 0, 1, 1, 64, 0, 0, 1, 1, 1, 1]
    attend = [64] * 9 + [1, 0, 1, 1, 64, 1, 1, 1, 1, 0]
    calls = ((rotary, range(6, 11), lambda z: lib.call("gb_rotary", 0, at, at, z, None, None, 1.0, None)),
             (append, [*range(15, 21), 23, 24, 25], lambda z: lib.call("gb_cache_append", 0, at, at, at, at, at, at, z, None, 1.0, at, at, None, None)),
             (attend, [*range(9, 14), *range(15, 19)], lambda z: lib.call("gb_cache_attn", 0, at, at, at, at, z, at, at, None, 1.0, None, 0, None)))
    for sizes, which, call in calls:
        call(words(*sizes))                                             # no tokens: nothing to do
        for i in which:
            for bad in (big, big + 1, -big):
                with pytest.raises(lib.NativeError):
                    call(words(*(bad if j == i else s for j, s in enumerate(sizes))))


def test_tangents(monkeypatch):
    """Forward-mode derivatives: the turn of the tangent; none goes through a cache."""
    from gonn_b200.ops import rotary
    fw = torch.autograd.forward_ad
    rope = nn.RotaryEmbedding(4, interleaved=True, amplitude=1.5)
    x, dx = torch.randn(2, 1, 3, 2, 6).unbind(0)
    at = torch.tensor([3, 1, 7])
    with fw.dual_level():
        want = fw.unpack_dual(rope(fw.make_dual(x, dx), at))

        def launch(x, positions, turns, interleaved, amplitude, back, out=None):   # the kernel's part, on the CPU
            return rotary.rotate_ref(x.detach(), positions, rope._w, interleaved, amplitude, back)
        monkeypatch.setattr(rotary, "_launch", launch)
        got = fw.unpack_dual(rotary._Rotary.apply(fw.make_dual(x, dx), at, rope.turns, True, 1.5, False))
        assert torch.equal(got.primal, want.primal) and torch.allclose(got.tangent, want.tangent)
        back = fw.unpack_dual(rotary._Rotary.apply(fw.make_dual(x, dx), at, rope.turns, True, 1.5, True))
        assert torch.allclose(back.tangent, rotary.rotate_ref(dx, at, rope._w, True, 1.5, True))
        cache, q = nn.KVCache(1, 4, 2, 6), x[:, :1]
        table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
        dual = fw.make_dual(q, dx[:, :1])
        for call in (lambda: cache.Append(dual, q, table, lengths), lambda: cache.Append(q, dual, table, lengths), lambda: cache.Attend(dual, table, lengths)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
        cache.Append(q, q, table, lengths)


def test_layers_pickled_without_rotary():
    """A layer pickled whole before it knew of rotary positions has none."""
    import pickle
    mha = nn.MultiHeadAttention(8, 2, dtype=torch.float64)
    x = torch.randn(1, 3, 8, dtype=torch.float64)
    old = pickle.loads(pickle.dumps(mha))
    del old.__dict__["rotary"]
    old = pickle.loads(pickle.dumps(old))
    assert old.rotary is None
    assert torch.equal(old(x, causal=True), mha(x, causal=True)) and torch.equal(old.ForwardMasked(x), mha.ForwardMasked(x))
    cache, table, at = nn.KVCache(1, 4, 2, 4, dtype=torch.float64), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with torch.no_grad():
        old.ForwardCached(x, cache, table, at)
    old.to(torch.float32)
    # and one with them keeps them
    with_rope = pickle.loads(pickle.dumps(nn.MultiHeadAttention(8, 2, rotary=nn.RotaryEmbedding(4))))
    assert with_rope.rotary.dim == 4


def test_fixed_point_angles_against_pi():
    """p times the fraction of a turn against p w / 2 pi with pi to 60 digits: off by p 2^-55 turns at most, w / 2 pi being rounded to fp64 (w up to
    1: below 0.16, off by 2^-56 and by what 2 pi in fp64 is off, 2^-54.5 of it)."""
    from fractions import Fraction
    pi = Fraction(3141592653589793238462643383279502884197169399375105820974944, 10 ** 60)
    for base, dim in ((10000.0, 128), (500000.0, 64), (1e6, 48)):
        w = nn.RotaryEmbedding(dim, base)._w
        for f, t in zip(w, turns_of(w).tolist()):
            for p in (1, 4095, 131071, 2 ** 31 - 1, -5):
                d = abs(Fraction(t * p % 2 ** 64, 2 ** 64) - Fraction(f) * p / (2 * pi) % 1)
                assert min(d, 1 - d) <= Fraction(abs(p), 2 ** 55)


def test_rotary_given_to_a_layer_later():
    """Assigned, it is a child of the layer, which uses it, pickles it and moves it."""
    import pickle
    rope = nn.RotaryEmbedding(4)
    mha, given = nn.MultiHeadAttention(8, 2), nn.MultiHeadAttention(8, 2, rotary=rope)
    given.load_state_dict(mha.state_dict())
    x = torch.randn(1, 3, 8)
    plain = mha(x, causal=True)
    mha.rotary = rope
    for layer in (mha, pickle.loads(pickle.dumps(mha)), mha.to("cpu")):
        assert torch.equal(layer(x, causal=True), given(x, causal=True)) and not torch.equal(layer(x, causal=True), plain)
