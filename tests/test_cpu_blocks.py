"""Refusals of the residual-block operators (favae_hip/blocks.py): wrong arguments raise before anything is launched, so they are
checked here without a GPU; the C entry points report theirs through favae_last_error."""
import pytest
import torch


def _b():
    from favae_hip import blocks
    return blocks


def _gn(b, **kw):
    a = dict(x=torch.zeros(2, 3, 8), groups=2, gamma=torch.ones(8), beta=torch.zeros(8))
    a.update(kw)
    return b.group_norm_act(**a)


@pytest.mark.parametrize("kw,err", [
    (dict(groups=3), ValueError), (dict(groups=0), ValueError), (dict(groups=2.0), ValueError), (dict(act="relu6"), ValueError),
    (dict(x=torch.zeros(8)), ValueError), (dict(x=torch.zeros(2, 3, 8, dtype=torch.float16)), TypeError),
    (dict(x=torch.zeros(2, 3, 8, dtype=torch.float64)), TypeError), (dict(), ValueError)])
def test_group_norm_refusals(kw, err):
    with pytest.raises(err):
        _gn(_b(), **kw)


def test_group_norm_bwd_refusals():
    b = _b()
    dy, g, st = torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(2, 2)
    for x in (torch.zeros(2, 4, 8), torch.zeros(2, 3, 8, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="as dy"):
            b.group_norm_act_bwd(dy, x, 2, g, g, st, st)
    ck = b.Ckpt8(torch.zeros(2, 3, 8, dtype=torch.int8), torch.zeros(2, 3, 1, dtype=torch.uint8), torch.bfloat16)
    with pytest.raises(ValueError, match="as dy"):
        b.group_norm_act_bwd(dy, ck, 2, g, g, st, st)


def test_linear_refusals():
    b = _b()
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError, match="GPU"):
        b.linear_act(x, w)
    for bad in (torch.zeros(6, 7), torch.zeros(8), torch.zeros(2, 6, 8)):
        with pytest.raises(ValueError):
            b.linear_act(x, bad)
    with pytest.raises(TypeError):
        b.linear_act(x, w.bfloat16())
    with pytest.raises(ValueError, match="act"):
        b.linear_act(x, w, act="tanh")
    dy = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="pre"):
        b.linear_act_bwd(dy, x, w, act="silu")
    with pytest.raises(ValueError, match="pre"):
        b.linear_act_bwd(dy, x, w, act="silu", pre=torch.zeros(4, 5))
    with pytest.raises(ValueError, match="need"):
        b.linear_act_bwd(dy, x, w, need=("r",))
    with pytest.raises(ValueError):
        b.linear_act_bwd(dy, torch.zeros(3, 8), w)
    with pytest.raises(ValueError, match="GPU"):
        b.linear_act_bwd(dy, x, w)


def test_ckpt8_refusals():
    b = _b()
    i8, u8 = torch.int8, torch.uint8
    q, e = torch.zeros(4, 40, dtype=i8), torch.zeros(4, 2, dtype=u8)
    assert b.Ckpt8(q, e, torch.float32).shape == (4, 40)
    for args, err in (((q.to(u8), e, torch.float32), TypeError), ((q, e, torch.float16), TypeError), ((q, e[:, :1], torch.float32), ValueError),
                      ((q[:, :33].clone()[:, :32], e[:, :1], torch.float32), ValueError), ((q, torch.zeros(2, 4, dtype=u8).t(), torch.float32), ValueError)):
        with pytest.raises(err):
            b.Ckpt8(*args)
    with pytest.raises(TypeError):
        b.ckpt8_pack(torch.zeros(4, 8, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        b.ckpt8_pack(torch.zeros(4, 8))
    with pytest.raises(TypeError):
        b.ckpt8_unpack(b.Ckpt8(q, e, torch.float32), torch.float64)


def test_row_strides():
    b = _b()
    t = torch.zeros(4, 6, 10)
    assert b._rows(t, "t") == 10 and b._rows(t[:, :, :7], "t") == 10 and b._rows(t[:, 2, :5], "t") == 60 and b._rows(t[:1, :, 3:], "t") == 10
    assert b._rows(t[0, 0, 2:5], "t") == 3 and b._maps(t[:, 1:4, :8], "t") == (60, 10) and b._maps(t[2:3, :, :8], "t") == (0, 10)
    for bad in (t[:, :3], t.transpose(1, 2), t[:, :, ::2], torch.zeros(10).expand(4, 10), t.permute(1, 0, 2)):
        with pytest.raises(ValueError):
            b._rows(bad, "t")


def test_c_entry_points_refuse_without_a_gpu():
    b = _b()
    from favae_hip import lib as L
    r = b._raw
    for call, text in ((lambda: r.favae_ckpt8_pack(None, 8, 4, 8, None, 8, None, 1, 0, None), "favae_ckpt8_pack"),
                       (lambda: r.favae_ckpt8_pack(None, 8, -1, 8, None, 8, None, 1, 0, None), "bad sizes"),
                       (lambda: r.favae_ckpt8_unpack(None, 8, None, 1, 4, 8, None, 8, 7, None), "dtype"),
                       (lambda: r.favae_gn_act_fwd(None, 8, 8, 1, 1, 8, 3, None, None, 1e-5, 0, None, 8, 8, None, None, None, None, None, 0, 0, None), "groups"),
                       (lambda: r.favae_gn_act_fwd(None, 8, 8, 1, 1, 8, 2, None, None, 1e-5, 9, None, 8, 8, None, None, None, None, None, 0, 0, None), "activation"),
                       (lambda: r.favae_gn_act_bwd(None, 8, 8, None, 8, 8, None, None, 1, 1, 8, 2, None, None, None, None, 0, None, 8, 8, None, None, None, 0, 0, None), "null"),
                       (lambda: r.favae_linear_act_fwd(None, 8, None, 8, None, None, 0, None, 0, None, 6, 4, 6, 8, 0, None, 0, 5, None), "dtype"),
                       (lambda: r.favae_linear_act_bwd(None, 6, None, 8, None, 0, None, 8, None, 0, None, 0, 4, 6, 8, 0, None, 8, None, 8, 0, None, None, 0, 0, None), "dy")):
        assert call() < 0 and text in L.last_error(), L.last_error()


def test_group_norm_plans_for_any_channel_count():
    """The workspace size, and with it the choice of a kernel, for channel counts around every limit of a workgroup."""
    from favae_hip import blocks as b
    from favae_hip import lib as L
    for dtype in (L.F32, L.BF16):
        for backward in (0, 1):
            for c, g in [(1047553, 1047553), (1 << 24, 1), (1 << 24, 1 << 24), ((1 << 24) - 1, 1), ((1 << 24) - 1, (1 << 24) - 1), (4097, 1), (4097 * 3, 3),
                         (1023 * 1021, 1023), (7, 7), (1, 1)]:
                for n, s in [(1, 1), (1, 5000), (300, 17), (0, 4), (2, 0)]:
                    assert b._raw.favae_gn_act_scratch(n, s, c, g, backward, dtype) >= 0
    assert L.last_error() is not None


def test_limits_are_checked_before_anything_is_launched():
    """Sizes past a limit, with pointers that no launch would survive: the argument error (-1), never that of a launch (-2)."""
    if torch.cuda.is_available():
        pytest.skip("a launch would be seen by its error, which needs a machine without a GPU")
    from favae_hip import blocks as b
    from favae_hip import lib as L
    r, p, big = b._raw, 4096, 1 << 60
    calls = {
        # groups of all samples together, backward in chunks
        "groups": lambda: r.favae_gn_act_bwd(p, 64 << 13, 64, p, 64 << 13, 64, None, None, 1 << 25, 1 << 13, 64, 64, p, p, p, p, 0, p, 64 << 13, 64, p, p, p, big, L.BF16, None),
        # workgroups of the norm, whose checkpoint goes first
        "samples": lambda: r.favae_gn_act_fwd(p, 8201, 8201, 1 << 30, 1, 8201, 8201, p, p, 1e-5, 0, p, 8201, 8201, p, p, p, p, p, big, L.BF16, None),
        # operands of the products, whose du goes first
        "too large": lambda: r.favae_linear_act_bwd(p, 1 << 20, p, 1 << 20, None, 0, p, 1 << 20, p, 1 << 20, None, 0, 1 << 22, 1 << 20, 1 << 20, 2, p, 1 << 20, p, 1 << 20,
                                                    L.BF16, p, p, big, L.BF16, None)}
    for text, call in calls.items():
        assert call() == -1 and text in L.last_error(), (text, L.last_error())
    assert r.favae_linear_act_bwd(p, 8, p, 8, None, 0, p, 8, None, 0, None, 0, 4, 8, 8, 0, p, 8, None, 8, L.BF16, None, p, big, L.BF16, None) == -2      # (a launch)


def test_outputs_beside_an_input_in_one_buffer():
    """Memory spans that meet without an element in common: columns of one buffer, and what only looks so."""
    import random
    b = _b()
    big = torch.zeros(6, 5, 40)
    x = big[:, :, :24]
    apart = lambda out, *ins: b._apart(out, "out", ins)
    for out in (big[:, :, 24:], big[:, :, 24:32], big[1:, :, 24:], big[:, 2:, 30:], big[::2, :, 24:], big[3, :, 24:]):
        apart(out, x)
        apart(x, out)
    apart(torch.zeros(3, 8)[:, 4:], torch.zeros(3, 8))
    rows = torch.zeros(64).as_strided((3, 8), (20, 1), 0)
    apart(torch.zeros(0), rows)
    for out in (big[:, :, 23:], big[:, :, 10:20], big[2:, :, 23:30], big.view(6, 200)[:, 20:50], big.view(-1)[24:60], big[..., ::2], big.transpose(1, 2)[:, 24:]):
        with pytest.raises(ValueError, match="overlaps"):
            apart(out, x)
        with pytest.raises(ValueError, match="overlaps"):
            apart(x, out)
    # another pitch, another type's view, and a pitch that is no multiple
    base = torch.zeros(400)
    a = base.as_strided((8, 4), (10, 1), 0)
    for out in (base.as_strided((4, 4), (15, 1), 5), base.as_strided((8, 4), (12, 1), 5), base.as_strided((8, 8), (10, 1), 4), base.as_strided((4, 2, 3), (20, 7, 1), 5)):
        with pytest.raises(ValueError, match="overlaps"):
            apart(out, a)
    apart(base.as_strided((3, 2, 4), (40, 20, 1), 5), a)
    apart(base.as_strided((4, 4), (20, 1), 5), a)
    apart(base.view(torch.bfloat16).as_strided((8, 8), (20, 1), 10), a)
    # never two tensors with an element in common
    rng, taken = random.Random(1), 0
    for _ in range(2000):
        pitch = rng.randint(4, 9)
        pair = []
        for _ in range(2):
            k, c = rng.choice([1, 1, 2]), rng.randint(1, 5)
            sh, st = (rng.randint(1, 4), rng.randint(1, 4), c), (pitch * rng.randint(0, 3), pitch * k + rng.choice([0, 0, 0, 1]), 1)
            pair.append(base.as_strided(sh, st, rng.randint(0, 2 * pitch)))
        one, two = (set(torch.arange(400).as_strided(t.shape, t.stride(), t.storage_offset()).flatten().tolist()) for t in pair)
        try:
            apart(*pair)
            taken += 1
            assert not one & two
        except ValueError:
            pass
    assert taken > 200


def norm_form(n, s, c, g, backward, dtype, even=1):
    """(form, vectors a thread up to the kernel's own number, groups a vector may touch, runs that end inside a vector), and what is ragged about it."""
    import ctypes
    from favae_hip import blocks as b
    from favae_hip import lib as L
    v = (ctypes.c_int * 12)()
    assert b._raw.favae_debug_gn_act_plan(ctypes.c_longlong(n), ctypes.c_longlong(s), c, g, backward, even if backward else 0, dtype, v) == 0
    form, items, gpv, tail, pieces, nsub, p, ncb, nchunk, cb, rows, _ = v
    name, vec = ("wave", "piped", "held", "chunked")[form], 4 if dtype == L.F32 else 8
    sizes = {"wave": (1, 2, 4, 8), "held": (4, 8, 12, 16) if backward else (4, 16)}.get(name, (1 << 30,))
    if name in ("held", "chunked"):
        gpv = gpv if gpv == 1 else vec
        tail = tail if gpv > 1 else 0
    ragged = {k for k, is_so in (("channels", c % cb), ("positions", p and s % p), ("samples", rows and n > rows and n % rows)) if is_so}
    return (name, min(t for t in sizes if t >= items) if name in ("wave", "held") else 0, gpv, tail), ragged


def test_every_form_of_the_norm_has_a_shape_among_the_gpu_tests():
    import test_gpu_blocks as t
    from favae_hip import lib as L
    for dtype, vec in ((L.F32, 4), (L.BF16, 8)):
        gpvs = [1, 2, 4, 8][:vec.bit_length()]
        for backward in (0, 1):
            got = [norm_form(*shape, backward, dtype) for shape in t.GN_FORMS]
            kinds = [(1, 0), (vec, 0), (vec, 1)]
            want = {("wave", i, k, 0) for i in (1, 2, 4, 8) for k in gpvs} | {("chunked", 0) + k for k in kinds}
            want |= {("held", i) + k for i in ((4, 8, 12, 16) if backward else (4, 16)) for k in kinds}
            if backward:
                want |= {("piped", 0, k, 0) for k in gpvs}
            assert want == {k for k, _ in got}, want ^ {k for k, _ in got}
            for form in ("wave", "held", "chunked") + (("piped",) if backward else ()):
                ragged = set().union(*(r for (f, *_), r in got if f == form))
                assert {"positions", "channels"} <= ragged and (form not in ("piped", "wave") or not backward or "samples" in ragged), (form, ragged)


def test_shapes_of_the_piped_backward_are_piped():
    import test_gpu_blocks as t
    from favae_hip import lib as L
    for mark in t.test_group_norm_piped_backward.pytestmark:
        for dtype, *shape in mark.args[1]:
            (form, *_), _ = norm_form(*shape, 1, L.F32 if dtype == torch.float32 else L.BF16)
            assert form == "piped", shape


def test_checkpoints_are_written_by_the_norm_where_its_runs_start_on_their_blocks():
    """Whatever the plan, a run of channels that a kernel packs starts and ends on a block of 32."""
    import ctypes
    import random
    from favae_hip import blocks as b
    rng, v, seen = random.Random(3), (ctypes.c_int * 12)(), set()
    for _ in range(20000):
        cg = rng.choice([1, 2, 4, 8, 12, 16, 24, 32, 40, 64, 2056, 2080, 4104, 4128, 8192, rng.randint(1, 9000)])
        g = rng.choice([1, 2, 4, 8, 32, rng.randint(1, 40)])
        dtype, c = rng.randint(0, 1), cg * g
        assert b._raw.favae_debug_gn_act_plan(ctypes.c_longlong(rng.choice([1, 3, 64, 700])), ctypes.c_longlong(rng.choice([0, 1, 5, 64, 1000, 5000])), c, g, 0, 1, dtype, v) == 0
        form, pieces, cb, packs = v[0], v[4], v[9], v[11]
        if packs:
            starts = [k * cg + j * cb for k in range(g) for j in range(pieces)] if pieces > 1 else range(0, c, cb)
            assert c % 32 == 0 and all(t % 32 == 0 for t in starts), (cg, g, pieces, cb)
        seen.add((bool(packs), pieces > 1, c % 32 == 0))
    assert {(True, True, True), (False, True, True), (True, False, True)} <= seen


def test_forward_form_with_a_checkpoint():
    """Held from 160 workgroups on, chunked below, where a thread would have more than 4 vectors; without a checkpoint from 96 on."""
    import ctypes
    from favae_hip import blocks as b
    from favae_hip import lib as L
    v = (ctypes.c_int * 12)()
    for shape, dtype, ckpt, form in (((64, 1024, 64, 8), L.BF16, 1, 3), ((48, 2048, 64, 8), L.BF16, 1, 3), ((200, 1500, 32, 4), L.BF16, 1, 2), ((24, 512, 256, 32), L.F32, 1, 2),
                                     ((64, 1024, 64, 8), L.BF16, 0, 2), ((8, 4096, 64, 8), L.BF16, 0, 3)):
        n, s, c, g = shape
        assert b._raw.favae_debug_gn_act_plan(ctypes.c_longlong(n), ctypes.c_longlong(s), c, g, 0, ckpt, dtype, v) == 0
        assert v[0] == form and (not ckpt or v[11]), (shape, ckpt, list(v))
