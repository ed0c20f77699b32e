"""GPU tests of the client's operators in the clear (libfhe_ssm_clear.so through clear_ops.py) against their definitions in
64 bits.

Tolerances are derived from the arithmetic, not from results.  With M the same sum taken over magnitudes, a float32 sum of n
rounded terms is off by at most about n 2^-24 M; an output in a 16-bit type is rounded once more, by the unit roundoff of 8
significant bits (2^-8 of itself) in bf16 and of 11 bits (2^-11) in f16.  Drawn tokens are whole numbers: the draws lie in the middle of a token's interval, where rounding cannot
move them to another, and have to give that token.
"""
import math

import numpy as np
import pytest

from engine_loader import load_module

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROUNDING = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LOWEST = {torch.float32: 2.0**-140, torch.bfloat16: 2.0**-130, torch.float16: 2.0**-24}  # below it results may be flushed


def ops():
    return load_module("clear_ops")


def assert_near(got, want, magnitude, terms):
    kind = got.dtype
    g = got.double()
    assert torch.isfinite(g).all()
    allowed = terms * 2.0**-24 * magnitude * (1 + ROUNDING[kind]) + ROUNDING[kind] * want.abs() + LOWEST[kind]
    worst = ((g - want).abs() / allowed).max().item() if g.numel() else 0.0
    assert worst <= 1, f"{worst} times the allowed error"


# ------------------------------------------------------------------------------------------------ linear attention
def recurrence(q, k, v, g, state, lengths, scale):
    """the definition, token by token in 64 bits: q, k [B, T, heads or fewer, dk], v [B, T, H, dv], g [B, T, H]"""
    B, T, H, dv = v.shape
    q, k = (x.double().repeat_interleave(H // x.shape[2], 2) for x in (q, k))
    v, g, S = v.double(), g.double().clamp_min(-1000.0), state.double().clone()
    out = torch.zeros(v.shape, dtype=torch.float64, device=v.device)
    for t in range(T):
        new = S * g[:, t].exp()[..., None, None] + k[:, t][..., None] * v[:, t][..., None, :]
        there = (lengths > t)[:, None, None]
        out[:, t] = torch.where(there, (q[:, t][..., None] * new).sum(-2) * scale, 0.0)
        S = torch.where(there[..., None], new, S)
    return out, S


def attention_case(B, T, H, Hq, Hk, dk, dv, kind, seed, decay=0.3):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    q, k, v = normal(B, T, Hq, dk).to(kind), normal(B, T, Hk, dk).to(kind), normal(B, T, H, dv).to(kind)
    g = -decay * torch.rand((B, T, H), generator=gen, device="cuda")
    return q, k, v, g, normal(B, H, dk, dv)


def run_prompt(q, k, v, g, state, lengths=None, scale=1.0, out=None, into=None, stream=None):
    c = ops()
    out = torch.full_like(v, 7.0) if out is None else out
    into = torch.full((v.shape[0], v.shape[2], q.shape[3], v.shape[3]), 7.0, device="cuda") if into is None else into
    need = c.linear_attention_workspace(q, k, v)
    workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda") if need else None
    c.linear_attention_prompt(q, k, v, g, state, into, out, scale=scale, lengths=lengths, workspace=workspace, stream=stream)
    torch.cuda.synchronize()
    return out, into


def check_prompt(q, k, v, g, state, lengths=None, scale=1.0, **more):
    B, T, H, dv = v.shape
    full = torch.full((B,), T, device="cuda") if lengths is None else lengths
    start = torch.zeros((B, H, q.shape[3], dv), device="cuda") if state is None else state.clone()
    wide = g.expand(B, T, H) if g.dim() == 1 else g
    want, left = recurrence(q, k, v, wide, start, full, scale)
    size, size_left = recurrence(q.abs(), k.abs(), v.abs(), wide, start.abs(), full, abs(scale))
    out, into = run_prompt(q, k, v, g, state, lengths, scale, **more)
    # a term is rounded when it is formed, decayed by a product of up to T factors (each off by 2 units, or together by the
    # size of their exponents' sum, below 2 a token here) and summed with T tokens and dk channels
    terms = 4 * T + q.shape[3] + 64
    assert_near(out, want, size, terms)
    assert_near(into, left, size_left, terms)
    return out, into


LENGTHS = [1, 2, 3, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 511, 700]


@pytest.mark.parametrize("T", LENGTHS)
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_lengths(T, kind):
    print(f"prompt of {T} tokens, {kind}", flush=True)
    check_prompt(*attention_case(2, T, 3, 3, 3, 64, 64, TYPES[kind], T), scale=0.125)


@pytest.mark.parametrize("dk, dv", [(1, 1), (8, 8), (16, 33), (31, 30), (32, 32), (40, 48), (48, 80), (64, 1), (65, 64),
                                    (96, 160), (128, 128), (127, 129)])
@pytest.mark.parametrize("kind", TYPES)
def test_prompt_head_sizes(dk, dv, kind):
    print(f"dk {dk}, dv {dv}, {kind}", flush=True)
    for T in (5, 150):
        check_prompt(*attention_case(1, T, 2, 1, 2, dk, dv, TYPES[kind], dk + dv + T), scale=dk**-0.5)


@pytest.mark.parametrize("H, Hq, Hk", [(1, 1, 1), (6, 6, 2), (6, 3, 6), (6, 1, 1), (5, 5, 1)])
def test_prompt_shared_heads(H, Hq, Hk):
    for T in (9, 140):
        check_prompt(*attention_case(2, T, H, Hq, Hk, 32, 48, torch.bfloat16, H + Hq + Hk + T))


@pytest.mark.parametrize("T", [7, 64, 300])
def test_prompt_ragged_lengths_hide_what_lies_behind(T):
    """every length from none to all, with NaN and infinities in what no lane reads"""
    lengths = torch.tensor([0, 1, T // 2, T - 1, T, T + 5, -3], dtype=torch.int32, device="cuda")
    q, k, v, g, state = attention_case(len(lengths), T, 2, 2, 1, 64, 64, torch.float32, T)
    clean = tuple(x.clone() for x in (q, k, v, g))
    for b, n in enumerate(lengths.clamp(0, T).tolist()):
        q[b, n:], k[b, n:], v[b, n:], g[b, n:] = math.nan, math.inf, math.nan, -math.inf
    want, left = check_prompt(*clean, state, lengths.clamp(0, T))
    out, into = run_prompt(q, k, v, g, state, lengths)
    assert torch.equal(out, want) and torch.equal(into, left)
    assert (out[0] == 0).all() and torch.equal(into[0], state[0])


def test_prompt_of_no_tokens_hands_the_state_on():
    q, k, v, g, state = attention_case(2, 0, 3, 3, 3, 64, 48, torch.bfloat16, 1)
    out, into = run_prompt(q, k, v, g, state)
    assert torch.equal(into, state) and out.numel() == 0
    _, into = run_prompt(q, k, v, g, None)
    assert (into == 0).all()


@pytest.mark.parametrize("T", [5, 64, 200])
def test_prompt_states(T):
    """no state before, none kept, the same buffer for both"""
    q, k, v, g, state = attention_case(2, T, 2, 2, 2, 64, 64, torch.bfloat16, T)
    check_prompt(q, k, v, g, None)
    want, left = run_prompt(q, k, v, g, state)
    kept = state.clone()
    out, into = run_prompt(q, k, v, g, kept, into=kept)
    assert torch.equal(out, want) and torch.equal(into, left)
    c = ops()
    out = torch.empty_like(v)
    need = c.linear_attention_workspace(q, k, v)
    c.linear_attention_prompt(q, k, v, g, state, None, out,
                              workspace=torch.empty(need, dtype=torch.uint8, device="cuda") if need else None)
    assert torch.equal(out, want)


@pytest.mark.parametrize("T", [6, 100, 260])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompt_decays_at_their_ends(T, kind):
    """no decay at all, states cleared by -inf and by what is as good, sums of decays far below the exponential's range,
    decays so small that only their sum counts"""
    q, k, v, g, state = attention_case(2, T, 5, 5, 5, 64, 64, TYPES[kind], T)
    g[:, :, 0] = 0.0
    g[:, ::3, 1] = -math.inf
    g[:, :, 2] = -90.0
    g[:, 1::4, 3] = -1e30
    g[:, :, 4] = -1e-6
    check_prompt(q, k, v, g, state)


@pytest.mark.parametrize("T", [20, 64, 200, 1500])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompt_values_that_are_not_finite_stay_in_their_future(T, kind):
    """an infinite value or a NaN reaches no token before its own, no other channel and no other lane or head"""
    q, k, v, g, state = attention_case(2, T, 2, 2, 2, 64, 64, TYPES[kind], T)
    want, left = run_prompt(q, k, v, g, state)
    at = [(0, T // 2, 1, 7, math.inf), (0, T - 1, 0, 3, math.nan), (1, T // 3, 0, 63, -math.inf)]
    for b, t, h, c, x in at:
        v[b, t, h, c] = x
    out, into = run_prompt(q, k, v, g, state)
    hit, hit_state = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(into, dtype=torch.bool)
    for b, t, h, c, _ in at:
        hit[b, t:, h, c], hit_state[b, h, :, c] = True, True
    assert not torch.isfinite(out[hit]).any() and not torch.isfinite(into[hit_state]).any()
    # elsewhere the same sums in another order
    size, size_left = recurrence(q.abs(), k.abs(), v.nan_to_num(0, 0, 0).abs(), g, state.abs(), torch.full((2,), T, device="cuda"), 1.0)
    allowed = (2 * (4 * T + 128) * 2.0**-24) * size + 2 * ROUNDING[out.dtype] * want.double().abs()
    assert ((out.double() - want.double()).abs() <= allowed)[~hit].all()
    assert ((into.double() - left.double()).abs() <= 2 * (4 * T + 128) * 2.0**-24 * size_left)[~hit_state].all()


@pytest.mark.parametrize("T", [4, 150])
def test_prompt_one_decay_per_head(T):
    q, k, v, _, state = attention_case(2, T, 4, 4, 2, 64, 64, torch.bfloat16, 3)
    check_prompt(q, k, v, -torch.exp2(-torch.arange(2.0, 6.0, device="cuda")), state)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("T", [6, 130])
def test_prompt_strides(T, kind):
    """slices of one projection's rows, tokens before lanes, one row shared by all lanes, an odd start, gaps in the output"""
    B, H, dk, dv = 3, 2, 64, 48
    gen = torch.Generator(device="cuda").manual_seed(T)
    wide = 3 + H * (2 * dk + dv) + 5
    rows = torch.randn((T, B, wide), generator=gen, device="cuda").to(TYPES[kind]).transpose(0, 1)
    q = rows[..., 3:3 + H * dk].unflatten(-1, (H, dk))
    k = rows[:1, :, 3 + H * dk:3 + 2 * H * dk].unflatten(-1, (H, dk)).expand(B, T, H, dk)
    v = rows[..., 3 + 2 * H * dk:-5].unflatten(-1, (H, dv))
    g = -torch.rand((H, T, B), generator=gen, device="cuda").permute(2, 1, 0)
    state = torch.randn((B, H, dk, dv), generator=gen, device="cuda")
    gaps = torch.full((T, H, B, dv + 7), 7.0, device="cuda").to(TYPES[kind])
    out = gaps[..., 3:3 + dv].permute(2, 0, 1, 3)
    assert q.storage_offset() % 2 == 1 and out.stride()[0] == dv + 7
    check_prompt(q, k, v, g, state, out=out)
    assert (gaps[..., :3] == 7).all() and (gaps[..., 3 + dv:] == 7).all()


def test_prompt_many_lanes_and_few():
    """work that fills the GPU many times over by lanes alone, and one head whose only long axis is its tokens"""
    check_prompt(*attention_case(150, 70, 8, 8, 8, 64, 64, torch.bfloat16, 1, decay=0.01))
    check_prompt(*attention_case(1, 2500, 1, 1, 1, 64, 64, torch.bfloat16, 2, decay=0.01))


def test_prompt_offsets_past_32_bits():
    """a lane whose rows begin past 2^32 bytes and past 2^31 elements"""
    B, T, H, d = 2, 70, 1, 64
    far = (1 << 31) + 4096
    pool = torch.zeros(far + T * H * d, dtype=torch.bfloat16, device="cuda")
    q, k, v, g, state = attention_case(B, T, H, H, H, d, d, torch.bfloat16, 5)
    for name, x in (("q", q), ("k", k), ("v", v)):
        view = pool.as_strided((B, T, H, d), (far, H * d, d, 1))
        view.copy_(x)
        check_prompt(view if name == "q" else q, view if name == "k" else k, view if name == "v" else v, g, state)
    view = pool.as_strided((B, T, H, d), (far, H * d, d, 1))
    check_prompt(q, k, v, g, state, out=view)


@pytest.mark.parametrize("lanes, H, Hq, Hk, dk, dv", [(1, 12, 12, 12, 64, 64), (32, 12, 12, 12, 64, 64), (3, 4, 2, 1, 48, 80),
                                                      (2, 3, 3, 3, 33, 31), (5, 2, 2, 2, 128, 130), (1, 1, 1, 1, 1, 1)])
@pytest.mark.parametrize("kind", TYPES)
def test_step(lanes, H, Hq, Hk, dk, dv, kind):
    q, k, v, g, state = attention_case(lanes, 1, H, Hq, Hk, dk, dv, TYPES[kind], lanes + dk)
    want, left = recurrence(q, k, v, g, state, torch.ones(lanes, device="cuda"), 0.25)
    size, size_left = recurrence(q.abs(), k.abs(), v.abs(), g, state.abs(), torch.ones(lanes, device="cuda"), 0.25)
    out, into = torch.full_like(v[:, 0], 7.0), torch.full_like(state, 7.0)
    ops().linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], state, into, out, scale=0.25)
    assert_near(out[:, None], want, size, dk + 68)
    assert_near(into, left, size_left, dk + 68)
    again = state.clone()  # in place, as a server keeps it
    ops().linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], again, again, out, scale=0.25)
    assert torch.equal(again, into)


def test_steps_continue_a_prompt():
    """a prompt's state carried on token by token gives what the whole text gives as one prompt"""
    T, more = 130, 9
    q, k, v, g, state = attention_case(2, T + more, 3, 3, 3, 64, 64, torch.float32, 8)
    want, left = check_prompt(q, k, v, g, state)
    _, into = run_prompt(q[:, :T], k[:, :T], v[:, :T], g[:, :T], state)
    out = torch.empty_like(v[:, 0])
    sizes, size_left = recurrence(q.abs(), k.abs(), v.abs(), g, state.abs(), torch.full((2,), T + more, device="cuda"), 1.0)
    for t in range(T, T + more):
        ops().linear_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], into, into, out)
        torch.cuda.synchronize()
        assert ((out - want[:, t]).abs() <= 2 * (4 * (T + more) + 128) * 2.0**-24 * sizes[:, t]).all()
    assert ((into - left).abs() <= 2 * (4 * (T + more) + 128) * 2.0**-24 * size_left).all()


def test_attention_results_do_not_change_from_run_to_run():
    case = attention_case(1, 3000, 2, 2, 2, 64, 64, torch.bfloat16, 4)
    first = run_prompt(*case)
    for _ in range(3):
        out, into = run_prompt(*case)
        assert torch.equal(out, first[0]) and torch.equal(into, first[1])


def test_attention_refusals():
    c = ops()
    q, k, v, g, state = attention_case(2, 3, 4, 2, 2, 64, 64, torch.bfloat16, 1)
    out, into = torch.empty_like(v), torch.empty_like(state)

    def refuse(words, **change):
        a = {**dict(q=q, k=k, v=v, log_decay=g, state_in=state, state_out=into, out=out), **change}
        with pytest.raises(c.ClearError, match=words):
            c.linear_attention_prompt(**a)

    refuse("differ in type", k=k.float())
    refuse("element type", q=q.double(), k=k.double(), v=v.double())
    refuse("differ in lanes", q=q[:1])
    refuse("cannot share", q=q[:, :, :1].expand(2, 3, 3, 64))
    refuse("contiguous", q=q.transpose(-1, -2).contiguous().transpose(-1, -2))
    refuse("float32", log_decay=g.half())
    refuse("log_decay", log_decay=g[:, :2])
    refuse("one entry per head", log_decay=g[0, 0, :2])
    refuse("like v", out=out.float())
    refuse("state_in", state_in=state[:, :, :32])
    refuse("state_out", state_out=into.transpose(-1, -2))
    refuse("lengths", lengths=torch.ones(2, dtype=torch.int64, device="cuda"))
    refuse("on the GPU", v=v.cpu())
    refuse("dk 192", q=torch.cat((q, q, q), -1), k=torch.cat((k, k, k), -1),
           state_in=None, state_out=None)
    with pytest.raises(c.ClearError, match="lanes, heads, channels"):
        c.linear_attention_step(q, k, v, g, state, into, out)


# ------------------------------------------------------------------------------------------------ 4-bit products
def product_case(rows, out, n_in, group, kind, scale_type, zeros, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-n_in // group)
    x = torch.randn((rows, n_in), generator=gen, device="cuda").to(kind)
    codes = torch.randint(0, 256, (out, -(-n_in // 2)), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (0.01 + torch.rand((out, groups), generator=gen, device="cuda") / 16).to(scale_type)
    z = torch.randint(0, 16, (out, groups), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    return x, codes, scales, z


def product_reference(x, codes, scales, zeros, group):
    """(the product, the sum of magnitudes that the kernel's sums go through: codes held as 16 + c, 16 + zero taken out)"""
    rows, n_in = x.shape
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :n_in].double()
    s = scales.double().repeat_interleave(group, 1)[:, :n_in]
    z = torch.full_like(c, 8.0) if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :n_in]
    return x.double() @ (s * (c - z)).t().contiguous(), x.double().abs() @ (s * (32 + c + z)).t().contiguous()


def check_product(x, codes, scales, zeros, group, out=None, stream=None):
    m = ops().Q4Matrix(codes, scales, zeros, in_features=x.shape[1], group=group, stream=stream)
    out = torch.full((x.shape[0], codes.shape[0]), 7.0, device="cuda").to(x.dtype) if out is None else out
    m.product(x, out, stream=stream)
    torch.cuda.synchronize()
    want, size = product_reference(x, codes, scales, zeros, group)
    # sums of a group's products (cut off rather than rounded at worst: two units each), of groups, and of waves
    assert_near(out, want, size, 2 * (min(group, x.shape[1]) + -(-x.shape[1] // group) + 16))
    return out


@pytest.mark.parametrize("rows", [1, 2, 7, 15, 16, 17, 31, 32, 33, 48, 64, 65, 130])
@pytest.mark.parametrize("kind", TYPES)
def test_product_rows(rows, kind):
    check_product(*product_case(rows, 200, 384, 64, TYPES[kind], torch.float16, False, rows), 64)


@pytest.mark.parametrize("n_in", [1, 2, 7, 31, 32, 33, 63, 65, 127, 128, 129, 255, 640, 1101, 4096, 5000])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
def test_product_columns_and_groups(n_in, group):
    for kind, zeros in ((torch.bfloat16, True), (torch.float32, False), (torch.float16, True)):
        check_product(*product_case(3, 37, n_in, group, kind, torch.float16, zeros, n_in + group), group)


@pytest.mark.parametrize("out", [1, 3, 15, 16, 17, 63, 64, 65, 255, 1000, 4099, 20011])
def test_product_outputs(out):
    for rows in (1, 20, 40):
        check_product(*product_case(rows, out, 256, 32, torch.bfloat16, torch.float16, True, out + rows), 32)


@pytest.mark.parametrize("scale_type", TYPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("zeros", [False, True])
def test_product_types(scale_type, kind, zeros):
    for rows, group in ((1, 32), (18, 64), (5, 128)):
        check_product(*product_case(rows, 130, 700, group, TYPES[kind], TYPES[scale_type], zeros, rows), group)


def test_product_every_code_and_zero_point_exactly():
    """one column at a time: y = scale (code - zero) for each of the 256 pairs, which nothing rounds"""
    c, z = torch.meshgrid(torch.arange(16), torch.arange(16), indexing="ij")
    codes = torch.zeros((256, 32), dtype=torch.uint8)
    for j in range(64):
        codes[:, j // 2] |= (c.reshape(-1) << (4 * (j % 2))).to(torch.uint8)
    zeros = z.reshape(-1, 1).to(torch.uint8).repeat(1, 2).contiguous().cuda()
    scales = torch.full((256, 2), 0.25, dtype=torch.float16, device="cuda")
    for kind in TYPES.values():
        m = ops().Q4Matrix(codes.cuda(), scales, zeros, group=32)
        x = torch.eye(64, device="cuda").to(kind)
        y = torch.empty((64, 256), device="cuda", dtype=kind)
        m.product(x, y)
        want = (0.25 * (c - z).reshape(1, -1).float()).expand(64, 256).cuda()
        assert torch.equal(y.float(), want)


def test_product_uses_all_24_bits_of_float32_rows():
    """an x whose three parts all count, against equal weights of 1: the product is x itself"""
    x = torch.tensor([[1 + 2.0**-23, -(1 + 2.0**-8 + 2.0**-16), 2.0**-100 * (1 + 2.0**-20), 1e30]], device="cuda").t().contiguous()
    codes = torch.full((16, 1), 9, dtype=torch.uint8, device="cuda")
    m = ops().Q4Matrix(codes, torch.ones((16, 1), device="cuda"), in_features=1, group=32)
    y = torch.empty((4, 16), device="cuda")
    m.product(x, y)
    # 25 x - 24 x: sums of x's size times 25, in float32
    assert ((y - x).abs() <= 64 * 2.0**-24 * x.abs()).all()


@pytest.mark.parametrize("kind", TYPES)
def test_product_strides(kind):
    """rows of x inside wider rows at an odd place, one row for all, rows of y with gaps, rows of codes with gaps; what lies
    beside a row is NaN and must not be read into it"""
    rows, out, n_in, group = 6, 90, 203, 32
    x, codes, scales, zeros = product_case(rows, out, n_in, group, TYPES[kind], torch.float16, True, 9)
    wide = torch.full((rows, n_in + 10), math.nan, device="cuda").to(TYPES[kind])
    wide[:, 3:3 + n_in] = x
    wide_codes = torch.full((out, codes.shape[1] + 13), 255, dtype=torch.uint8, device="cuda")
    wide_codes[:, 5:5 + codes.shape[1]] = codes
    gaps = torch.full((rows, out + 5), 7.0, device="cuda").to(TYPES[kind])
    want = check_product(x, codes, scales, zeros, group)
    got = check_product(wide[:, 3:3 + n_in], wide_codes[:, 5:5 + codes.shape[1]], scales, zeros, group, out=gaps[:, 1:1 + out])
    assert torch.equal(got, want) and (gaps[:, 0] == 7).all() and (gaps[:, 1 + out:] == 7).all()
    check_product(x[:1].expand(rows, n_in), codes, scales, zeros, group)


def test_product_of_no_rows_and_the_last_code():
    x, codes, scales, _ = product_case(3, 40, 65, 32, torch.bfloat16, torch.float16, False, 2)
    m = ops().Q4Matrix(codes, scales, None, in_features=65, group=32)
    y = torch.full((0, 40), 7.0, device="cuda").bfloat16()
    m.product(x[:0], y)
    want = check_product(x, codes, scales, None, 32)
    dirty = codes.clone()
    dirty[:, -1] |= 0xf0  # the half byte past the last column belongs to nothing
    assert torch.equal(check_product(x, dirty, scales, None, 32), want)


def test_product_rows_do_not_meet():
    """a row of NaN leaves the others as they are"""
    x, codes, scales, _ = product_case(20, 64, 256, 64, torch.float32, torch.float16, False, 2)
    want = check_product(x, codes, scales, None, 64)
    x[7] = math.nan
    m = ops().Q4Matrix(codes, scales, None, group=64)
    y = torch.empty((20, 64), device="cuda")
    m.product(x, y)
    assert torch.isnan(y[7]).all()
    keep = torch.arange(20) != 7
    assert torch.equal(y[keep], want[keep])


def test_product_offsets_past_32_bits():
    x, codes, scales, _ = product_case(2, 48, 256, 64, torch.bfloat16, torch.float16, False, 3)
    far = (1 << 31) + 1024
    pool = torch.zeros(far + 256, dtype=torch.bfloat16, device="cuda")
    view = pool.as_strided((2, 256), (far, 1))
    view.copy_(x)
    want = check_product(x, codes, scales, None, 64)
    assert torch.equal(check_product(view, codes, scales, None, 64), want)
    out = pool.as_strided((2, 48), (far, 1))
    assert torch.equal(check_product(x, codes, scales, None, 64, out=out), want)


def test_quantized_head_gives_the_matrix_products():
    """quantize_q4 and the product together: the product of the rounded matrix, half a step of each weight from the given one"""
    c = ops()
    w = np.random.default_rng(1).standard_normal((70, 200)).astype(np.float32)
    x = torch.randn((4, 200), generator=torch.Generator().manual_seed(1)).cuda()
    for zeros in (False, True):
        codes, scales, zero = (None if a is None else torch.from_numpy(a).cuda() for a in c.quantize_q4(w, 32, zeros))
        y = check_product(x, codes, scales, zero, 32)
        step = scales.double().repeat_interleave(32, 1)[:, :200]
        far = (1.01 if zeros else 0.51) * (x.double().abs() @ step.t().contiguous())
        assert ((y.double() - x.double() @ torch.from_numpy(w).cuda().double().t().contiguous()).abs() <= far + 1e-3).all()


def test_product_refusals():
    c = ops()
    x, codes, scales, zeros = product_case(3, 40, 64, 32, torch.bfloat16, torch.float16, True, 2)
    with pytest.raises(c.ClearError, match="group 48"):
        c.Q4Matrix(codes, scales, group=48)
    with pytest.raises(c.ClearError, match="do not hold"):
        c.Q4Matrix(codes, scales, in_features=66, group=32)
    with pytest.raises(c.ClearError, match="scales must be"):
        c.Q4Matrix(codes, scales[:, :1], group=32)
    with pytest.raises(c.ClearError, match="zeros must be"):
        c.Q4Matrix(codes, scales, zeros.int(), group=32)
    with pytest.raises(c.ClearError, match="uint8 rows"):
        c.Q4Matrix(codes.int(), scales, group=32)
    m = c.Q4Matrix(codes, scales, zeros, group=32)
    y = torch.empty((3, 40), device="cuda", dtype=torch.bfloat16)
    for bad_x, bad_y in ((x.float(), y), (x[:, :32], y), (x, y[:, :39]), (x, y[:2]), (x.double(), y)):
        with pytest.raises(c.ClearError):
            m.product(bad_x, bad_y)
    with pytest.raises(c.ClearError, match="contiguous"):
        m.product(x.t().contiguous().t(), y)
    with pytest.raises(c.ClearError, match="overlap"):
        m.product(x, y[:1].expand(3, 40))


# ------------------------------------------------------------------------------------------------ sampling
def kept_weights(x, temperature=1.0, k=0, top_p=1.0, min_p=0.0):
    """the definition in 64 bits for one row: the weight of every entry, 0 where the filters drop it"""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, dtype=np.float64)) + 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    weight = np.zeros(len(x))
    if not len(order):
        return weight
    if not temperature > 0:
        weight[order[0]] = 1.0
        return weight
    order = order[:k] if k > 0 else order
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        p = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / temperature))
    p = p / p.sum()
    kept = np.ones(len(p), dtype=bool)
    if top_p < 1:
        kept &= np.concatenate(([0.0], np.cumsum(p)[:-1])) < top_p
        kept[0] = True
    if min_p > 0:
        kept &= p >= min(min_p, 1.0) * p[0]
    weight[order[kept]] = p[kept] / p[kept].sum()
    return weight


def run_sample(logits, draws, **params):
    rows = logits.shape[0]
    tokens = torch.full((rows,), -7, dtype=torch.int64, device="cuda")
    logprobs = torch.full((rows,), 7.0, device="cuda")
    given = {}
    for name, v in params.items():
        dtype = torch.int32 if name == "top_k" else torch.float32
        given[name] = torch.as_tensor(v, dtype=dtype, device="cuda").expand(rows).contiguous()
    ops().sample(logits, torch.as_tensor(draws, dtype=torch.float32, device="cuda"), tokens, logprobs, **given)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), logprobs.cpu().numpy()


def check_row(x, kind=torch.float32, most=200, **params):
    """draws in the middle of every kept entry's interval (of `most` of them) give that entry and its log-probability"""
    x = torch.as_tensor(np.asarray(x, dtype=np.float32)).to(kind)
    params = {n: v if n == "top_k" else float(np.float32(v)) for n, v in params.items()}  # as the kernel is given them
    w = kept_weights(x.double().numpy(), params.get("temperature", 1.0), params.get("top_k", 0), params.get("top_p", 1.0),
                     params.get("min_p", 0.0))
    upto = np.cumsum(w)
    # an interval's middle is at least half its width from its ends: 2^-24 of float32 numbers, 2^-21 of the sums' rounding
    at = np.flatnonzero(w > 2.0**-18)
    at = at[np.linspace(0, len(at) - 1, min(most, len(at))).astype(int)]
    draws = (upto[at] - w[at] / 2)
    tokens, logprobs = run_sample(x.cuda()[None].expand(len(at), len(x)), draws, **params)
    assert np.array_equal(tokens, at)
    # (l - top) / temperature, a float32 exponent of up to 25, and the logarithm of a sum of 2^-22
    assert np.abs(logprobs - np.log(w[at])).max() <= 2.0**-20
    return at


def spread(vocab, seed, kind="peaked"):
    rng = np.random.default_rng(seed)
    x = 2 * rng.standard_normal(vocab)
    if kind == "peaked":
        x[rng.permutation(vocab)[:max(1, vocab // 60)]] += 6
    return x.astype(np.float32)


VOCABS = [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1025, 4097, 20000, 50277, 65536, 100001, 262144]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("kind", TYPES)
def test_sample_vocabularies(vocab, kind):
    print(f"vocabulary of {vocab}, {kind}", flush=True)
    x = spread(vocab, vocab)
    check_row(x, TYPES[kind], most=40)
    check_row(x, TYPES[kind], most=40, temperature=0.7, top_k=20)
    check_row(x, TYPES[kind], most=40, temperature=1.3, top_p=0.81234)
    check_row(x, TYPES[kind], most=40, top_k=50, top_p=0.912345, min_p=0.0123)


@pytest.mark.parametrize("k", [1, 2, 5, 63, 64, 65, 255, 999, 1000, 1001, 1 << 30])
def test_sample_top_k(k):
    at = check_row(spread(1000, 7, "flat") / 8, most=1000, top_k=k)
    assert len(at) == min(k, 1000)


@pytest.mark.parametrize("vocab", [700, 5000, 70000])
def test_sample_large_nuclei(vocab):
    """filters that keep hundreds and thousands of entries, from flat rows and from rows of equal entries"""
    x = spread(vocab, 3, "flat") / 4
    for top_p in (0.101, 0.5003, 0.9907):
        check_row(x, most=60, top_p=top_p)
    check_row(x, most=60, top_k=vocab // 2, top_p=0.7003)
    check_row(x, most=60, min_p=0.31)
    check_row(np.zeros(600), most=600, top_k=333)
    check_row(np.zeros(600), most=600, top_p=100.5 / 600)


def test_sample_ties_go_to_the_lowest_index():
    x = np.zeros(300)
    x[[7, 50, 200]] = 2.0
    x[[9, 60, 61, 299]] = 1.0
    for k, want in ((1, [7]), (2, [7, 50]), (3, [7, 50, 200]), (4, [7, 9, 50, 200]), (6, [7, 9, 50, 60, 61, 200]),
                    (8, [0, 7, 9, 50, 60, 61, 200, 299])):
        for kind in TYPES.values():
            assert check_row(x, kind, top_k=k).tolist() == want
    # top-p that ends inside the ties: 2 of the 4 ones, whose first has 3 e^2 before it
    total = 3 * math.e**2 + 4 * math.e + 293
    assert check_row(x, top_p=(3 * math.e**2 + 1.5 * math.e) / total).tolist() == [7, 9, 50, 60, 200]
    # and of both filters the shorter
    six = 3 * math.e**2 + 3 * math.e
    assert check_row(x, top_k=6, top_p=(3 * math.e**2 + 0.5 * math.e) / six).tolist() == [7, 9, 50, 200]
    assert check_row(x, top_k=5, top_p=0.999).tolist() == [7, 9, 50, 60, 200]
    assert check_row([0.0, -0.0, 0.0, -0.0], top_k=3).tolist() == [0, 1, 2]


def test_sample_greedy():
    x = spread(5000, 1)
    x[[41, 4000]] = 30.0
    for temperature in (0.0, -1.0, math.nan):
        tokens, logprobs = run_sample(torch.from_numpy(x).cuda()[None].expand(3, 5000), [0.0, 0.5, 0.999],
                                      temperature=temperature, top_k=40, top_p=0.9, min_p=0.1)
        assert (tokens == 41).all() and (logprobs == 0).all()


def test_sample_masks_infinities_and_nan():
    x = spread(3000, 2)
    x[::2] = -np.inf
    x[1::6] = np.nan
    for params in ({}, dict(top_k=7), dict(top_p=0.612345), dict(top_k=2000, min_p=0.03), dict(temperature=3.0)):
        check_row(x, most=50, **params)
    lowest = spread(500, 3)
    lowest[::3] = np.finfo(np.float32).min
    check_row(lowest, most=50)
    check_row(np.full(70, np.finfo(np.float32).min))  # all at the type's lowest value: equal, and drawn
    infinite = spread(500, 3)
    infinite[[3, 77, 400]] = np.inf
    assert check_row(infinite).tolist() == [3, 77, 400]
    assert check_row(infinite, top_k=2).tolist() == [3, 77]
    empty = torch.full((4, 900), -math.inf, device="cuda")
    empty[1] = math.nan
    empty[2, 899] = 1.0
    empty[3, 0] = -3e38
    tokens, logprobs = run_sample(empty, [0.0, 0.5, 0.9, 0.2], top_k=5, top_p=0.9, min_p=0.1)
    assert tokens.tolist() == [-1, -1, 899, 0]
    assert logprobs[0] == logprobs[1] == -math.inf and logprobs[2] == logprobs[3] == 0


def test_sample_draws_and_parameters_at_their_ends():
    x = np.array([0.0, -np.inf, 1.0, 0.5, -50.0], dtype=np.float32)
    row = torch.from_numpy(x).cuda()[None]
    tokens, _ = run_sample(row.expand(6, 5), [0.0, -1.0, math.nan, 1.0 - 2.0**-24, 1.0, 7.0])
    assert tokens.tolist()[:3] == [0, 0, 0]  # the first that may be drawn
    assert tokens.tolist()[3:] == [3, 3, 3]  # the last with a mass that counts: e^-51 is below 2^-24 of the sum
    check_row(x, top_k=0)
    check_row(x, top_k=-4, top_p=1.0, min_p=0.0)
    check_row(x, top_p=math.nan)
    check_row(x, min_p=math.nan)
    check_row(x, top_p=2.0, min_p=-1.0)
    assert check_row(x, top_p=0.0).tolist() == [2] and check_row(x, top_p=-1.0).tolist() == [2]
    assert check_row([1.0, 0.0, 1.0], min_p=1.0).tolist() == [0, 2] and check_row([1.0, 0.0, 1.0], min_p=9.0).tolist() == [0, 2]
    tokens, logprobs = run_sample(row, [0.5], temperature=1e-40)
    assert tokens.tolist() == [2] and logprobs[0] == 0
    tokens, logprobs = run_sample(row.expand(4, 5), [0.1, 0.4, 0.6, 0.9], temperature=math.inf)  # four equal entries
    assert tokens.tolist() == [0, 2, 3, 4] and np.abs(logprobs + math.log(4)).max() < 1e-6


def test_sample_rows_have_parameters_of_their_own():
    """a batch of rows, each with its own filters and its own draw, in a strided block of logits with NaN in the gaps"""
    rows, vocab = 67, 3001
    rng = np.random.default_rng(4)
    block = torch.full((rows, vocab + 13), math.nan, device="cuda")
    logits = block[:, 5:5 + vocab]
    params = dict(temperature=[], top_k=[], top_p=[], min_p=[])
    draws, want, logs = [], [], []
    for r in range(rows):
        x = spread(vocab, 100 + r)
        p = dict(temperature=[0.0, 0.5, 1.0, 1.7][r % 4], k=[0, 1, 17, 400][r // 4 % 4], top_p=[1.0, 0.512345, 0.95321][r % 3],
                 min_p=[0.0, 0.0123, 0.2345][r // 3 % 3])
        p = {n: float(np.float32(v)) if n != "k" else v for n, v in p.items()}
        w = kept_weights(x, **p)
        at = rng.choice(np.flatnonzero(w > 1e-5))
        draws.append(np.cumsum(w)[at] - w[at] / 2)
        want.append(at)
        logs.append(math.log(w[at]))
        logits[r] = torch.from_numpy(x).cuda()
        for n, v in p.items():
            params["top_k" if n == "k" else n].append(v)
    tokens, logprobs = run_sample(logits, draws, **{n: np.array(v) for n, v in params.items()})
    assert tokens.tolist() == want
    assert np.abs(logprobs - np.array(logs)).max() <= 2.0**-20


def test_sample_offsets_past_32_bits_and_no_logprobs():
    vocab, far = 500, (1 << 31) + 64
    pool = torch.zeros(far + vocab, dtype=torch.bfloat16, device="cuda")
    logits = pool.as_strided((2, vocab), (far, 1))
    logits.copy_(torch.from_numpy(spread(vocab, 1)).cuda()[None].expand(2, vocab))
    logits[1, 123] = 60.0
    tokens = torch.empty(2, dtype=torch.int64, device="cuda")
    ops().sample(logits, torch.tensor([0.5, 0.5], device="cuda"), tokens)
    assert tokens[1].item() == 123 and tokens[0].item() != 123


def test_sample_follows_the_distribution():
    """many draws on a grid: each kept token as often as its probability says, to within one draw"""
    x, n = spread(40, 9), 4096
    params = dict(temperature=1.1, top_k=25, top_p=0.93)
    w = kept_weights(x, 1.1, 25, 0.93, 0.0)
    draws = (np.arange(n) + 0.5) / n
    tokens, _ = run_sample(torch.from_numpy(x).cuda()[None].expand(n, 40), draws, **params)
    assert np.abs(np.bincount(tokens, minlength=40) - n * w).max() <= 1.001
    assert (np.diff(tokens) >= 0).all()  # in the order of the vocabulary


def test_sample_refusals():
    c = ops()
    x = torch.zeros((3, 10), device="cuda")
    u, tokens = torch.zeros(3, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (dict(draws=u.double()), dict(draws=u[:2]), dict(tokens=tokens.int()), dict(top_k=tokens),
                dict(temperature=u.half()), dict(logits=x.double()), dict(logits=x.t().contiguous().t()),
                dict(logprobs=tokens), dict(min_p=torch.zeros(6, device="cuda")[::2])):
        with pytest.raises(c.ClearError):
            c.sample(**{**dict(logits=x, draws=u, tokens=tokens), **bad})
    c.sample(x[:0], u[:0], tokens[:0])  # no rows: nothing to do


# ------------------------------------------------------------------------------------------------ streams and graphs
def together(stream=None):
    """all operators on one stream, as a client runs them: prompt, head, draw"""
    c = ops()
    q, k, v, g, state = attention_case(2, 200, 3, 3, 3, 64, 64, torch.float32, 3)
    x, codes, scales, zeros = product_case(1, 777, 192, 32, torch.float32, torch.float16, True, 4)
    need = c.linear_attention_workspace(q, k, v)
    bufs = dict(out=torch.zeros_like(v), into=torch.zeros_like(state), logits=torch.zeros((2, 777), device="cuda"),
                tokens=torch.zeros(2, dtype=torch.int64, device="cuda"), logprobs=torch.zeros(2, device="cuda"))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    head = c.Q4Matrix(codes, scales, zeros, in_features=192, group=32)
    draws = torch.tensor([0.3, 0.8], device="cuda")
    torch.cuda.synchronize()

    def go(stream):
        c.linear_attention_prompt(q, k, v, g, state, bufs["into"], bufs["out"], scale=0.125, workspace=ws, stream=stream)
        c.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], bufs["into"], bufs["into"], bufs["out"][:, -1],
                                scale=0.125, stream=stream)
        head.product(bufs["out"][:, -1].flatten(1), bufs["logits"], stream=stream)
        c.sample(bufs["logits"], draws, bufs["tokens"], bufs["logprobs"], stream=stream)

    return go, bufs


def test_operators_on_another_stream():
    go, bufs = together()
    go(None)
    torch.cuda.synchronize()
    want = {n: b.clone() for n, b in bufs.items()}
    side = torch.cuda.Stream()
    for b in bufs.values():
        b.zero_()
    side.wait_stream(torch.cuda.current_stream())
    go(side.cuda_stream)
    side.synchronize()
    for n in bufs:
        assert torch.equal(bufs[n], want[n]), n


def test_operators_in_a_graph():
    go, bufs = together()
    go(None)
    torch.cuda.synchronize()
    want = {n: b.clone() for n, b in bufs.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        for b in bufs.values():
            b.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for n in bufs:
            assert torch.equal(bufs[n], want[n]), n
        go(None)
        torch.cuda.synchronize()
