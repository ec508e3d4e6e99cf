"""Full-attention operators of a serving step (block tables, rotary positions with norm and cache write, paged decode) against
the 64-bit oracle, their refusals, and a run of them together.

Tolerances. ``half(t)`` is the half step of one rounding to type t, relative to the value. A rotated channel is one rounding of
a 32-bit value whose error is within 2^-20 of the length of the pair it comes from (frequency reduced in 64 bits; sine and cosine
within 2 units in the last place, 2^-22; two products and a sum, 2^-23; with the norm also the sum of at most 256 squares, each lane
adding eight and five shuffle steps, 13 * 2^-24, its root and two products: 2^-20 in all, so 2^-19 is allowed there). Attention: the
scores are 32-bit sums of D products, off by at most D * 2^-24 * scale * sum |q| |k| =: e; the weights are rounded to the activations'
type for the product with v, and the 32-bit sums over n tokens are off by at most (n + 64) * 2^-24, so an output is
within (half + 2 e + 2 (n + 64) 2^-24 + 2^-20) * sum p |v|, plus its own rounding; the log of the sum within e + (n + 64) 2^-24 +
2^-22 (1 + |lse|). The kernel holds the weights in two numbers of the activations' type; ``assert_attention_kept`` bounds that."""
import math

import pytest
import torch

from oracle import full_attention as ofa

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def fa():
    from pla_b200.decode import full_attention
    return full_attention


def half(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what="out"):
    """|got - want| <= bound + one rounding to got's type (fp16: or half its smallest step), everywhere."""
    dtype, got, want = got.dtype, got.double().cpu(), want.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all(), f"{what}: non-finite values"
    if got.numel() == 0:
        return
    over = (got - want).abs() - bound - half(dtype) * (want.abs() + bound) - (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert over.max().item() <= 0, f"{what}: {over.max().item():.3e} over its bound at {torch.nonzero(over == over.max())[0].tolist()}"


def i32(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def word():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ frequencies (host)
def test_frequencies_plain_and_scaled(native_built):
    f, m = fa().rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and m == 1.0
    torch.testing.assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15, atol=0)
    lin, _ = fa().rotary_frequencies(8, 10000.0, scaling="linear", factor=4.0)
    torch.testing.assert_close(lin, f / 4, rtol=1e-15, atol=0)
    ntk, _ = fa().rotary_frequencies(8, 10000.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and abs(ntk[-1].item() - 0.00025) < 1e-15              # the slowest is divided by the factor exactly
    bands, _ = fa().rotary_frequencies(128, 500000.0, scaling="bands", factor=8.0, original_max_position=8192)
    plain, _ = fa().rotary_frequencies(128, 500000.0)
    wave = 2 * math.pi / plain
    assert torch.equal(bands[wave < 8192 / 4], plain[wave < 8192 / 4])
    torch.testing.assert_close(bands[wave > 8192], plain[wave > 8192] / 8, rtol=1e-15, atol=0)
    mid = (wave > 8192 / 4) & (wave < 8192)
    assert mid.any() and (bands[mid] < plain[mid]).all() and (bands[mid] > plain[mid] / 8).all()
    yarn, m = fa().rotary_frequencies(64, 10000.0, scaling="yarn", factor=16.0, original_max_position=4096)
    plain, _ = fa().rotary_frequencies(64, 10000.0)
    turns = 4096 * plain / (2 * math.pi)
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-15
    assert torch.equal(yarn[turns > 45], plain[turns > 45])                     # a channel is 1.33 times the next one's turns
    torch.testing.assert_close(yarn[turns < 0.7], plain[turns < 0.7] / 16, rtol=1e-15, atol=0)
    assert (yarn[1:] < yarn[:-1]).all()


@pytest.mark.parametrize("original,fast,slow", [(4, 32.0, 1.0), (128, 64.0, 32.0), (1, 2.0, 0.5)])
def test_yarn_divides_every_slow_channel(native_built, original, fast, slow):
    """A context so short that even the fastest channel turns fewer than beta_slow times: all of them are divided, the first one too."""
    plain, _ = fa().rotary_frequencies(64, 10000.0)
    assert original / (2 * math.pi) < slow
    yarn, _ = fa().rotary_frequencies(64, 10000.0, scaling="yarn", factor=8.0, original_max_position=original, beta_fast=fast, beta_slow=slow)
    torch.testing.assert_close(yarn, plain / 8, rtol=1e-15, atol=0)


@pytest.mark.parametrize("kw", [dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, scaling="other"),
                                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=2, scaling="ntk", factor=2.0),
                                dict(rotary_dim=8, scaling="yarn", beta_fast=1.0, beta_slow=2.0),
                                dict(rotary_dim=8, scaling="bands", low_freq_factor=4.0, high_freq_factor=4.0)])
def test_frequencies_refusals(native_built, kw):
    with pytest.raises(ValueError):
        fa().rotary_frequencies(**kw)


def test_host_tensors_are_refused(native_built):
    q, i = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    cache = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa().apply_rotary(q, None, i, torch.ones(4, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa().paged_attention_decode(q, cache, cache, i[None], i)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa().build_block_tables(i[None], i, torch.zeros(2, dtype=torch.int32), i, 4, num_tokens=0)


# ------------------------------------------------------------------------------------------------ C ABI (host)
def test_abi_entries_are_exported_and_refuse_bad_arguments(native_built):
    """Every entry of the header refuses NULL and sizes out of range before it launches anything; no GPU needed."""
    import ctypes
    from pla_b200 import capi
    lib = capi.load()
    capi.check_layout(lib)
    assert set(capi.ATTENTION_STRUCTS) == {"pla_b200_page_strides", "pla_b200_block_tables_args", "pla_b200_rotary_args",
                                           "pla_b200_paged_decode_args"}
    for name in ("pla_b200_block_tables", "pla_b200_rotary", "pla_b200_paged_decode"):
        assert getattr(lib, name)(None, None) == -1 and b"NULL" in lib.pla_b200_last_error()
    a = capi.pla_b200_paged_decode_args(B=1, Hq=4, Hk=3, D=64)
    assert lib.pla_b200_paged_decode(ctypes.byref(a), None) == -1
    a = capi.pla_b200_paged_decode_args(B=1, Hq=4, Hk=2, D=80)
    assert lib.pla_b200_paged_decode(ctypes.byref(a), None) == -3 and b"head size" in lib.pla_b200_last_error()
    a = capi.pla_b200_paged_decode_args(B=1, Hq=4, Hk=2, D=64, block_size=4)
    assert lib.pla_b200_paged_decode(ctypes.byref(a), None) == -1 and b"required" in lib.pla_b200_last_error()
    assert lib.pla_b200_paged_decode_workspace_bytes(None) == -1
    a = capi.pla_b200_paged_decode_args(B=64, Hq=4, Hk=3, D=64, block_size=16, columns=9)
    assert lib.pla_b200_paged_decode_workspace_bytes(ctypes.byref(a)) == -1
    a.Hk = 2
    assert lib.pla_b200_paged_decode_workspace_bytes(ctypes.byref(a)) > 0
    a.B = 1                                       # little work: clusters, no workspace
    assert lib.pla_b200_paged_decode_workspace_bytes(ctypes.byref(a)) == 0
    r = capi.pla_b200_rotary_args(T=1, Hq=4, D=60, R=8)
    assert lib.pla_b200_rotary(ctypes.byref(r), None) == -1 and b"multiple of 8" in lib.pla_b200_last_error()
    r = capi.pla_b200_rotary_args(T=1, Hq=4, D=64, R=9)
    assert lib.pla_b200_rotary(ctypes.byref(r), None) == -1 and b"even" in lib.pla_b200_last_error()
    t = capi.pla_b200_block_tables_args(N=1, tokens=1, columns=1, block_size=0)
    assert lib.pla_b200_block_tables(ctypes.byref(t), None) == -1 and b"block_size" in lib.pla_b200_last_error()


# ------------------------------------------------------------------------------------------------ block tables
def tables_case(context, new, block_size, columns=None, tokens=None, free=None, start=None, pad=0, first=0):
    """Runs op and oracle on one batch and compares everything, bit for bit."""
    offsets = [first]
    for m in new:
        offsets.append(offsets[-1] + m)
    held = [max(0, -(-c // block_size)) for c in context]
    need = sum(-(-(c + m) // block_size) - h for c, m, h in zip(context, new, held) if c >= 0)
    if columns is None:
        columns = max([-(-(c + m) // block_size) for c, m in zip(context, new)] + [1]) + 1
    g = torch.Generator().manual_seed(len(context) * 31 + block_size)
    ids = torch.randperm(sum(held) + max(need, free or 0, 0) + 5, generator=g).tolist()
    rows, at = [], 0
    for h in held:
        h = min(h, columns)
        rows.append(ids[at:at + h] + [-7] * (columns - h))
        at += h
    free = ids[at:at + need + 3] if free is None else ids[at:at + free]
    tokens = offsets[-1] if tokens is None else tokens
    want = ofa.block_tables(rows, context, offsets, free, block_size, tokens, 0 if start is None else start)
    wide = torch.full((len(rows), columns + pad), -9, dtype=torch.int32, device="cuda")
    if rows:
        wide[:, :columns] = i32(rows)
    status = word()
    plan = fa().build_block_tables(wide[:, :columns], i32(context), i32(offsets), i32(free), block_size, num_tokens=tokens,
                                   free_start=None if start is None else i32([start]), status=status)
    torch.cuda.synchronize()
    assert plan.block_table.tolist() == want[0]
    assert plan.slot_mapping.tolist() == want[1] and plan.slot_mapping.dtype == torch.int64
    assert plan.positions.tolist() == want[2]
    assert plan.seq_lens.tolist() == want[3]
    assert plan.free_next.tolist() == [want[4]]
    assert status.item() == want[5]
    assert (wide[:, columns:] == -9).all()
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("block_size", [1, 7, 16, 64])
@pytest.mark.parametrize("context,new", [
    ([0], [1]), ([16], [1]), ([15], [1]), ([63], [2]), ([0, 5, 0, 64], [3, 0, 0, 1]), ([100, 0, 33], [1, 130, 31]),
    ([i * 7 % 90 for i in range(300)], [1] * 300), ([0] * 6, [0, 300, 0, 257, 1, 0]),
    ([i % 40 for i in range(1500)], [i % 3 for i in range(1500)]), ([5] * 2100, [1] * 2100),
], ids=lambda x: f"{len(x)}x{sum(x)}")
def test_tables_match_the_oracle(native_built, context, new, block_size):
    tables_case(context, new, block_size, pad=3)


@pytest.mark.gpu
def test_tables_edges(native_built):
    want = tables_case([3, 0], [2, 1], 4, tokens=700, start=2)                    # padding rows, a list begun earlier
    assert want[1][3:] == [-1] * 697
    want = tables_case([0, 0, 0], [9, 9, 9], 4, free=4)                           # the list runs out in the second request
    assert want[5] == 32 and want[4] == 4 and want[1][20:] == [-1] * 7
    want = tables_case([0, 3], [9, 1], 4, columns=2)                              # a row with too few columns
    assert want[5] == 64 and want[1][8] == -1
    want = tables_case([30], [1], 4, columns=3)                                   # a context longer than its row
    assert want[5] == 64 and want[1] == [-1]
    want = tables_case([-1, 4], [2, 3], 4)                                        # bad metadata: no slots, no pages
    assert want[5] == 1 and want[1][:2] == [-1, -1]
    tables_case([0], [0], 4)                                                      # nothing to do
    tables_case([2] * 40, [1] * 40, 4, free=0)                                    # no list at all: only pages that are held
    plan = fa().build_block_tables(torch.empty(0, 4, dtype=torch.int32, device="cuda"), i32([]), i32([0]), i32([3]), 4, num_tokens=3)
    assert plan.slot_mapping.tolist() == [-1] * 3 and plan.positions.tolist() == [0] * 3 and plan.free_next.tolist() == [0]
    # offsets past the token rows: the rest is left out, flagged
    table, status = torch.full((2, 3), -7, dtype=torch.int32, device="cuda"), word()
    plan = fa().build_block_tables(table, i32([0, 0]), i32([0, 2, 9]), i32([5, 6, 7]), 4, num_tokens=3, status=status)
    assert status.item() == 1 and plan.slot_mapping.tolist() == [20, 21, 24] and table.tolist() == [[5, -7, -7], [6, -7, -7]]
    # offsets that decrease: the request takes nothing and nothing is written out of place
    table, status = torch.full((2, 3), -7, dtype=torch.int32, device="cuda"), word()
    plan = fa().build_block_tables(table, i32([0, 0]), i32([0, 4, 2]), i32([5, 6]), 4, num_tokens=4, status=status)
    assert status.item() == 1 and table.tolist() == [[5, -7, -7], [-7, -7, -7]] and plan.slot_mapping.tolist() == [20, 21, -1, -1]


@pytest.mark.gpu
def test_tables_leave_out_tokens_without_a_row(native_built):
    """Offsets past the token rows: pages, table entries, lengths and the list's next entry agree on the tokens that have a row."""
    want = tables_case([0, 0], [2, 7], 4, tokens=3)
    assert want[5] == 1 and want[3] == [2, 1] and want[4] == 2
    want = tables_case([6, 3, 8, 0], [5, 9, 1, 40], 4, tokens=8)                  # ends inside a request that holds pages
    assert want[5] == 1 and want[3] == [11, 6, 8, 0]
    want = tables_case([4] * 3, [4] * 3, 4, tokens=0)
    assert want[5] == 1 and want[3] == [4] * 3 and want[4] == 0
    want = tables_case([i % 9 for i in range(1500)], [3] * 1500, 2, tokens=2000)  # in the middle of the first scan of two
    assert want[5] == 1 and want[3][667:] == [i % 9 for i in range(667, 1500)]
    want = tables_case([5, 2 ** 31 - 3], [1, 3], 1 << 20, columns=4)              # a length past 32 bits
    assert want[5] == 1 and want[3] == [6, 2 ** 31 - 3] and want[1][1:] == [-1] * 3
    want = tables_case([0, 2 ** 31 - 10], [900, 9], 1 << 20, columns=4)           # one that just fits, behind other tokens
    assert want[5] == 64 and want[3] == [900, 2 ** 31 - 1] and want[1][900:] == [-1] * 9


@pytest.mark.gpu
@pytest.mark.parametrize("context,new,first,tokens", [
    ([0, 0, 0], [4, -2, 4], 0, 6), ([1] * 5, [10, -8, 1, 1, 8], 0, 12), ([3, 2], [5, 1], -3, 4), ([0] * 4, [3, -5, 9, 2], 0, 9),
    ([2] * 3, [1, 1, 1], 5, 10), ([0, 0], [-2, 6], 0, 8), ([0, 0], [4, -2], 0, 4), ([0, 0], [4, -6], 0, 4), ([i % 7 for i in range(2500)], [1] * 700 + [-300] + [2] * 1799, 0, 4100),
    ([i % 7 for i in range(2500)], [1] * 1023 + [-900, 2] + [1] * 1475, 0, 1700), ([1] * 1500, [3] * 1500, -2000, 2600)],
    ids=["falls", "long", "negative", "below-0", "late", "at-once", "end-falls", "end-below-0", "in-a-scan", "between-scans", "far-below"])
def test_tables_offsets_that_fall(native_built, context, new, first, tokens):
    """Requests that begin below an earlier offset, or below 0, get nothing; table, slots, lengths and the list agree on the others."""
    for block_size in (1, 3, 16):
        want = tables_case(context, new, block_size, tokens=tokens, first=first, columns=16, free=5200)
        assert want[5] == (0 if first > 0 else 1)
        taken = [x for x in want[1] if x >= 0]
        assert len(set(taken)) == len(taken)


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [0, 2])
def test_tables_free_next_stays_inside_the_list(native_built, requests):
    """Nothing to take: the next entry is the first one, at least 0 and at most the list's length, with and without requests."""
    table, lens, offsets = torch.full((requests, 3), -7, dtype=torch.int32, device="cuda"), i32([4] * requests), i32([0] * (requests + 1))
    for start, want in ((None, 0), (3, 3), (4, 4), (9, 4), (-5, 0)):
        status = word()
        plan = fa().build_block_tables(table, lens, offsets, i32([1, 2, 3, 5]), 4, num_tokens=300, free_start=None if start is None else i32([start]),
                                       status=status)
        assert plan.free_next.tolist() == [want] and status.item() == 0
        assert plan.slot_mapping.tolist() == [-1] * 300 and plan.positions.tolist() == [0] * 300 and plan.seq_lens.tolist() == [4] * requests
    plan = fa().build_block_tables(table, lens, offsets, i32([]), 4, num_tokens=0, free_start=i32([2]))
    assert plan.free_next.tolist() == [0] and plan.slot_mapping.shape == (0,)


@pytest.mark.gpu
def test_tables_with_many_requests_and_streams(native_built):
    """More requests than one scan holds, several tiles of tokens; the same on another stream and replayed from a graph with other
    lengths in the same tensors."""
    context, new = [(i * 37) % 500 for i in range(5000)], [(i * 11) % 4 for i in range(5000)]
    tables_case(context, new, 16)
    table, ctx, off = torch.zeros(3, 8, dtype=torch.int32, device="cuda"), i32([0, 0, 0]), i32([0, 4, 8, 12])
    free = i32(list(range(10, 40)))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        plan = fa().build_block_tables(table, ctx, off, free, 4, num_tokens=12)
    side.synchronize()
    assert plan.slot_mapping.tolist() == [4 * p + i for p in (10, 11, 12) for i in range(4)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = fa().build_block_tables(table, ctx, off, free, 4, num_tokens=12)
    for c, o in (([4, 3, 0], [0, 1, 2, 7]), ([0, 0, 8], [0, 0, 0, 1])):
        rows = [[20 + 2 * r, 21 + 2 * r] + [0] * 6 for r in range(3)]
        table.copy_(i32(rows)), ctx.copy_(i32(c)), off.copy_(i32(o))
        g.replay()
        want = ofa.block_tables(rows, c, o, free.tolist(), 4, 12)
        assert plan.slot_mapping.tolist() == want[1] and table.tolist() == want[0] and plan.free_next.tolist() == [want[4]]


@pytest.mark.gpu
def test_tables_slots_past_32_bits(native_built):
    plan = fa().build_block_tables(i32([[-1]]), i32([0]), i32([0, 3]), i32([2 ** 31 - 1]), 1 << 20, num_tokens=3)
    base = (2 ** 31 - 1) << 20
    assert plan.slot_mapping.tolist() == [base, base + 1, base + 2]


@pytest.mark.gpu
def test_tables_refusals(native_built):
    f = fa().build_block_tables
    table, c, o, free = i32([[0, 0]]), i32([0]), i32([0, 1]), i32([1, 2])
    for bad, match in [((table.long(), c, o, free, 4), "int32"), ((table, c.long(), o, free, 4), "context_lens"),
                       ((table, c, i32([0]), free, 4), "query_start_loc"), ((table, c, o, free, 0), "block_size"),
                       ((table, c, o, free.cpu(), 4), "free_blocks"), ((table[:, ::2].expand(1, 2), c, o, free, 4), "columns"),
                       ((table.expand(2, 2), i32([0, 0]), i32([0, 1, 2]), free, 4), "overlap")]:
        with pytest.raises(RuntimeError, match=match):
            f(*bad, num_tokens=1)
    with pytest.raises(RuntimeError, match="num_tokens"):
        f(table, c, o, free, 4, num_tokens=-1)
    with pytest.raises(RuntimeError, match="free_start"):
        f(table, c, o, free, 4, num_tokens=1, free_start=i32([0, 0]))


# ------------------------------------------------------------------------------------------------ rotary
def rows(g, T, hq, hk, D, dtype, extra=0):
    """q, k, v as slices of one packed row."""
    row = torch.randn(T, (hq + 2 * hk) * D + extra, generator=g).to(dtype)
    q, k, v = row[:, :hq * D], row[:, hq * D:(hq + hk) * D], row[:, (hq + hk) * D:(hq + 2 * hk) * D]
    return row, [x.unflatten(1, (-1, D)) for x in (q, k, v)]


def on_gpu(row, hq, hk, D):
    row = row.cuda()
    q, k, v = row[:, :hq * D], row[:, hq * D:(hq + hk) * D], row[:, (hq + hk) * D:(hq + 2 * hk) * D]
    return [x.unflatten(1, (-1, D)) for x in (q, k, v)]


def expect(x, w, pos, freq, inter, factor=1.0, unit=False, eps=1e-6):
    slack = 2.0 ** -20
    if w is not None:
        x, slack = ofa.rms_norm(x, w, eps, unit), 2.0 ** -19
    y, size = ofa.rotate(x, pos, freq, inter, factor)
    return y, slack * size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,hq,hk,D,R", [(1, 1, 1, 8, 2), (1, 32, 8, 128, 128), (3, 16, 2, 256, 64), (130, 5, 1, 96, 48), (7, 6, 3, 80, 20),
                                         (2, 40, 8, 64, 64), (17, 3, 3, 192, 192), (5, 4, 4, 256, 256), (9, 2, 1, 128, 40), (4, 3, 2, 24, 6),
                                         (1025, 4, 2, 64, 32), (3, 2, 1, 64, 0), (2500, 6, 2, 96, 72), (6, 9, 2, 256, 168),
                                         (4, 3, 2, 200, 200), (3, 5, 5, 72, 40), (5001, 3, 1, 128, 128)])
def test_rotary_matches_the_oracle(native_built, T, hq, hk, D, R, inter, dtype):
    g = torch.Generator().manual_seed(T * 7 + D + R)
    row, (q, k, _) = rows(g, T, hq, hk, D, DT[dtype], extra=8)
    pos = torch.randint(0, 1 << 20, (T,), generator=g)
    pos[0] = 1 << 26 if T > 1 else 0
    freq = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / max(R, 1))
    dq, dk, _ = on_gpu(row, hq, hk, D)
    oq, ok = fa().apply_rotary(dq, dk, pos.cuda(), freq.cuda(), interleaved=inter, factor=1.25)
    for got, x, name in ((oq, q, "q"), (ok, k, "k")):
        y, bound = expect(x, None, pos, freq, inter, 1.25)
        assert_within(got, y, bound, name)
        assert torch.equal(got[..., R:].cpu(), x[..., R:])
    assert oq.is_contiguous() and torch.equal(dq.cpu(), q)
    # in place, 32-bit positions (every second entry of a vector), without k
    both = torch.stack([pos.to(torch.int32), torch.zeros(T, dtype=torch.int32)], 1).cuda()
    a, b = fa().apply_rotary(dq, None, both[:, 0], freq.cuda(), interleaved=inter, factor=1.25, out_q=dq)
    assert b is None and torch.equal(dq, oq) and a.data_ptr() == dq.data_ptr()
    assert torch.equal(dk.cpu(), k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", [("bf16", torch.bfloat16), ("fp16", torch.float32)])
@pytest.mark.parametrize("inter,unit", [(False, True), (True, False)])
@pytest.mark.parametrize("T,hq,hk,D,R", [(1, 1, 1, 8, 8), (1, 16, 2, 256, 64), (67, 5, 1, 96, 48), (6, 7, 7, 128, 128), (33, 4, 2, 64, 20), (3, 2, 1, 200, 64), (2400, 3, 2, 128, 40),
                                         (5, 2, 2, 104, 88)])
def test_norm_rotary_matches_the_oracle(native_built, T, hq, hk, D, R, inter, unit, dtype, wdtype):
    g = torch.Generator().manual_seed(T + D + R)
    row, (q, k, _) = rows(g, T, hq, hk, D, DT[dtype])
    row[0, :D] = 0                                                                # a row of zeros: eps alone
    qw, kw = ((torch.randn(D, generator=g) * 0.2 + (0 if unit else 1)).to(wdtype) for _ in range(2))
    pos = torch.randint(0, 70000, (T,), generator=g)
    freq = 500000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / R)
    dq, dk, _ = on_gpu(row, hq, hk, D)
    kw_args = dict(eps=1e-5, unit_offset=unit, interleaved=inter)
    oq, ok = fa().qk_norm_rotary(dq, dk, qw.cuda(), kw.cuda(), pos.cuda(), freq.cuda(), **kw_args)
    for got, x, w, name in ((oq, q, qw, "q"), (ok, k, kw, "k")):
        y, bound = expect(x, w, pos, freq, inter, unit=unit, eps=1e-5)
        assert_within(got, y, bound, name)
    # one side without a norm
    oq2, ok2 = fa().qk_norm_rotary(dq, dk, None, kw.cuda(), pos.cuda(), freq.cuda(), **kw_args)
    assert torch.equal(ok2, ok) and torch.equal(oq2, fa().apply_rotary(dq, None, pos.cuda(), freq.cuda(), interleaved=inter)[0])
    # in place
    fa().qk_norm_rotary(dq, dk, qw.cuda(), kw.cuda(), pos.cuda(), freq.cuda(), out_q=dq, out_k=dk, **kw_args)
    assert torch.equal(dq, oq) and torch.equal(dk, ok)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("D,R,inter", [(128, 64, False), (128, 128, False), (256, 128, True), (96, 72, False), (64, 20, True)])
def test_norm_of_very_small_and_large_rows(native_built, D, R, inter, eps):
    """bf16 rows whose squares are no 32-bit numbers, next to ordinary rows: the norm of the definition, in the bounds of every other row. The
    mean of the squares is taken of rows that are scaled by a power of two, so nothing is added to the bound."""
    sizes = [1.0, 1e-15, 1e-19, 1e-23, 1e-30, 1e-37, 1e19, 1e23, 1e30, 1e36, 3.0]
    g = torch.Generator().manual_seed(D)
    x = (torch.randn(5, len(sizes), D, generator=g) * torch.tensor(sizes)[:, None]).bfloat16()
    if eps > 0:
        x[:, 0] = 0
    w, pos = torch.rand(D, generator=g) + 0.5, torch.arange(5) * 100
    freq = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / R)
    got, _ = fa().qk_norm_rotary(x.cuda(), None, w.cuda(), None, pos.cuda(), freq.cuda(), eps=eps, interleaved=inter)
    y, bound = expect(x, w, pos, freq, inter, eps=eps)
    assert_within(got, y, bound + 2.0 ** -134)            # and half the smallest step of bf16
    x[1, 3, 5], x[2, 7, 9], x[3, 0, 0] = float("inf"), float("nan"), float("-inf")
    got, _ = fa().qk_norm_rotary(x.cuda(), None, w.cuda(), None, pos.cuda(), freq.cuda(), eps=eps, interleaved=inter)
    spoilt = torch.zeros(x.shape[:2], dtype=torch.bool)
    spoilt[1, 3] = spoilt[2, 7] = spoilt[3, 0] = True
    assert torch.equal((~torch.isfinite(got)).any(-1).cpu(), spoilt)
    assert got[2, 7].isnan().all()
    assert_within(got.cpu()[~spoilt], y[~spoilt], bound[~spoilt] + 2.0 ** -134)


def caches(blocks, bs, hk, D, dtype, layout, fill=float("nan")):
    """k and v caches of one of three layouts, addressed [page, token, head, channel]."""
    if layout == "packed":
        both = torch.full((blocks, 2, bs, hk, D), fill, dtype=dtype, device="cuda")
        return both[:, 0], both[:, 1]
    if layout == "heads":
        return tuple(torch.full((blocks, hk, bs, D), fill, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
    return tuple(torch.full((blocks, bs, hk, D), fill, dtype=dtype, device="cuda") for _ in range(2))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["separate", "packed", "heads"])
@pytest.mark.parametrize("T,hq,hk,D,R,bs,norm", [(1, 16, 2, 256, 64, 16, True), (45, 8, 8, 64, 64, 7, True), (300, 5, 1, 96, 48, 1, False),
                                                 (64, 4, 2, 128, 24, 64, True)])
def test_cache_write_matches_the_oracle(native_built, T, hq, hk, D, R, bs, norm, layout):
    g = torch.Generator().manual_seed(T + D)
    row, (q, k, v) = rows(g, T, hq, hk, D, torch.bfloat16)
    blocks = -(-T // bs) + 2
    slots = torch.randperm(blocks * bs, generator=g)[:T]
    if T > 3:
        slots[1], slots[T - 1] = -1, -5                                          # padding rows store nothing
    pos = torch.randint(0, 5000, (T,), generator=g)
    freq = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / R)
    qw = (torch.randn(D, generator=g) * 0.2 + 1).bfloat16() if norm else None
    kc, vc = caches(blocks, bs, hk, D, torch.bfloat16, layout)
    dq, dk, dv = on_gpu(row, hq, hk, D)
    dw = qw.cuda() if norm else None
    status = word()
    out = fa().qk_norm_rotary_cache(dq, dk, dv, dw, dw, pos.cuda(), freq.cuda(), kc, vc, slots.cuda(), status=status)
    assert status.item() == 0
    y, bound = expect(q, qw, pos, freq, False)
    assert_within(out, y, bound, "q")
    y, bound = expect(k, qw, pos, freq, False)
    live = slots >= 0
    page, inside = (slots[live] // bs).cuda(), (slots[live] % bs).cuda()
    assert_within(kc[page, inside], y[live], bound[live], "k")
    assert torch.equal(vc[page, inside].cpu(), v[live])
    kc[page, inside] = float("nan")                                               # every other slot kept its bytes
    vc[page, inside] = float("nan")
    assert kc.isnan().all() and vc.isnan().all()
    # 32-bit slots give the same; a slot outside the pool is flagged and stores nothing
    again = fa().qk_norm_rotary_cache(dq, dk, dv, dw, dw, pos.cuda(), freq.cuda(), kc, vc, slots.to(torch.int32).cuda())
    assert torch.equal(again, out) and not kc[page, inside].isnan().any()
    kc.fill_(float("nan"))
    far = torch.full((T,), blocks * bs, dtype=torch.int64, device="cuda")
    fa().qk_norm_rotary_cache(dq, dk, dv, dw, dw, pos.cuda(), freq.cuda(), kc, vc, far, status=status)
    assert status.item() == 8 and kc.isnan().all()


@pytest.mark.gpu
def test_rotary_empty_and_non_finite(native_built):
    freq = torch.ones(4, dtype=torch.float64, device="cuda")
    q, k = fa().apply_rotary(torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda"), None, i32([]), freq)
    assert q.shape == (0, 2, 64) and k is None
    q, k = fa().apply_rotary(torch.empty(3, 0, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(3, 1, 64, dtype=torch.bfloat16, device="cuda"),
                             i32([0, 0, 0]), freq)
    assert q.shape == (3, 0, 64) and torch.all(k == 1)
    # a NaN or an infinity stays in its pair (rotation) or in its row (norm)
    x = torch.ones(2, 3, 64, dtype=torch.bfloat16, device="cuda")
    x[0, 1, 2], x[1, 2, 40] = float("nan"), float("inf")
    y, _ = fa().apply_rotary(x, None, i32([1, 2]), freq)
    bad = ~torch.isfinite(y)
    assert bad.sum() == 3 and bad[0, 1, 2] and bad[0, 1, 6] and bad[1, 2, 40]
    w = torch.ones(64, device="cuda")
    y, _ = fa().qk_norm_rotary(x, None, w, None, i32([1, 2]), freq)
    ok = torch.isfinite(y).all(-1)
    assert ok.tolist() == [[True, False, True], [True, True, False]]


@pytest.mark.gpu
def test_rotary_refusals(native_built):
    freq = torch.ones(8, dtype=torch.float64, device="cuda")
    x, pos = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda"), i32([0, 1])
    a = fa().apply_rotary
    for args, match in [((x.float(), None, pos, freq), "bf16 or fp16"), ((x[..., :60], None, pos, freq), "multiple of 8"),
                        ((x, x.half(), pos, freq), "dtype"), ((x, x[:1], pos, freq), "tokens"), ((x, None, pos[:1], freq), "positions"),
                        ((x, None, pos.float(), freq), "positions"), ((x, None, pos, freq.float()), "float64"),
                        ((x, None, pos, torch.ones(33, dtype=torch.float64, device="cuda")), "rotated part"),
                        ((x, None, pos.cpu(), freq), "positions"), ((x.transpose(1, 2), None, pos, freq), "contiguous"),
                        ((torch.zeros(2, 2, 264, dtype=torch.bfloat16, device="cuda"), None, pos, freq), "256"),
                        ((torch.zeros(2, 132, dtype=torch.bfloat16, device="cuda")[:, 4:].unflatten(1, (2, 64)), None, pos, freq), "aligned")]:
        with pytest.raises(RuntimeError, match=match):
            a(*args)
    with pytest.raises(RuntimeError, match="out_q"):
        a(x, None, pos, freq, out_q=x[:1])
    w = torch.ones(64, device="cuda")
    with pytest.raises(RuntimeError, match="q_weight"):
        fa().qk_norm_rotary(x, x, w[:32], w, pos, freq)
    kc = torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16, device="cuda")
    c = fa().qk_norm_rotary_cache
    for over, match in [(dict(v=x[:, :1]), "v must match"), (dict(k_cache=kc[:1]), "same shape"), (dict(k_cache=kc.half()), "dtype"),
                        (dict(k_cache=kc[..., :32], v_cache=kc[..., :32]), "heads of size"), (dict(slot_mapping=pos[:1]), "slot_mapping"),
                        (dict(status=torch.zeros(1, device="cuda")), "status")]:
        kw = dict(q=x, k=x, v=x, q_weight=w, k_weight=w, positions=pos, inv_freq=freq, k_cache=kc, v_cache=kc, slot_mapping=pos) | over
        with pytest.raises(RuntimeError, match=match):
            c(**kw)


# ------------------------------------------------------------------------------------------------ paged decode
def paged_inputs(seed, lens, hq, hk, D, bs, dtype=torch.bfloat16, layout="separate", extra_columns=2, sharp=1.0):
    """q, caches and table; everything that no request owns (other pages, the tail of a last page) is NaN, table entries past a
    request's pages are far outside the pool."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // bs) for n in lens]
    blocks = sum(pages) + 2
    order = torch.randperm(blocks, generator=g).tolist()
    columns = max(pages + [1]) + extra_columns
    table = torch.full((len(lens), columns), 1 << 30, dtype=torch.int32)
    kc, vc = caches(blocks, bs, hk, D, dtype, layout)
    for b, n in enumerate(lens):
        own = [order.pop() for _ in range(pages[b])]
        table[b, :pages[b]] = torch.tensor(own, dtype=torch.int32)
        if n:
            t = torch.arange(n)
            at = (table[b, t // bs].long().cuda(), (t % bs).cuda())
            kc[at] = torch.randn(n, hk, D, generator=g).to(dtype).cuda()
            vc[at] = torch.randn(n, hk, D, generator=g).to(dtype).cuda()
    q = (torch.randn(len(lens), hq, D, generator=g) * sharp).to(dtype)
    return q, kc, vc, table


def assert_attention(got, lse, q, kc, vc, table, lens, scale=None):
    out, want_lse, spread, reach = ofa.paged_attention(q, kc.cpu(), vc.cpu(), table, lens, scale)
    D, n = q.shape[-1], torch.tensor([max(int(x), 0) for x in lens], dtype=torch.float64)[:, None]
    e = D * 2.0 ** -24 * reach
    sums = (n + 64) * 2.0 ** -24
    assert_within(got, out, (half(q.dtype) + 2 * e + 2 * sums + 2.0 ** -20)[..., None] * spread)
    if lse is not None:
        empty = torch.isinf(want_lse)
        assert torch.equal(lse.cpu()[empty], want_lse[empty].float())
        limit = e + sums + 2.0 ** -22 * (1 + want_lse.abs())
        over = ((lse.cpu().double() - want_lse).abs() - limit)[~empty]
        assert over.numel() == 0 or over.max().item() <= 0, f"lse {over.max().item():.3e} over its bound"


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 700]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hk,D,bs,layout", [(16, 2, 256, 16, "separate"), (32, 8, 128, 16, "packed"), (8, 8, 64, 1, "heads"), (5, 1, 96, 7, "separate"),
                                               (12, 2, 192, 48, "heads"), (16, 1, 128, 64, "packed"), (3, 1, 256, 128, "heads"), (40, 2, 64, 32, "separate"),
                                               (33, 1, 128, 16, "separate"), (34, 2, 256, 16, "heads"), (16, 2, 256, 7, "heads"), (8, 8, 128, 1, "packed"),
                                               (6, 2, 192, 20, "separate"), (128, 2, 64, 8, "packed"), (18, 1, 256, 1, "separate")])
def test_attention_matches_the_oracle(native_built, hq, hk, D, bs, layout, dtype):
    q, kc, vc, table = paged_inputs(hq * D + bs, EDGES, hq, hk, D, bs, DT[dtype], layout)
    status = word()
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(EDGES), return_lse=True, status=status)
    assert status.item() == 0 and out.shape == q.shape
    assert_attention(out, lse, q, kc, vc, table, EDGES)
    assert torch.all(out[0] == 0) and torch.all(lse[0] == -math.inf)
    again = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(EDGES), out=torch.full_like(out, float("nan")))
    assert torch.equal(again, out)                                                # the same bits every time, into a given tensor


@pytest.mark.gpu
@pytest.mark.parametrize("lens,hq,hk,D,bs", [([5000], 16, 2, 128, 16), ([9001, 3, 0, 1200], 8, 1, 256, 64), ([4096] * 3, 4, 4, 64, 32), ([0, 0], 4, 2, 128, 16),
                                             ([1], 1, 1, 64, 1), ([40] * 300, 8, 2, 64, 16), ([1] * 700, 4, 4, 96, 16), ([i % 5 for i in range(3000)], 2, 1, 64, 4),
                                             ([20011, 7], 4, 1, 192, 9), ([12000, 300, 0, 5], 2, 2, 128, 1), ([64] * 40, 8, 8, 128, 64)],
                         ids=["one-5000", "ragged-9001", "even-4096", "all-empty", "one-token", "300x40", "700x1", "3000-tiny", "rows-20011",
                              "rows-12000", "one-unit-rows"])
def test_attention_lengths(native_built, lens, hq, hk, D, bs):
    q, kc, vc, table = paged_inputs(len(lens) + D, lens, hq, hk, D, bs)
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens), return_lse=True, scale=0.11)
    assert_attention(out, lse, q, kc, vc, table, lens, 0.11)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,hq,hk,D,bs,layout", [([777], 16, 2, 128, 16, "separate"), ([1], 4, 4, 64, 1, "heads"), ([0, 70, 513], 8, 2, 256, 32, "packed"),
                                                    ([4000], 5, 1, 64, 48, "separate"), ([129, 64, 0, 1], 40, 2, 96, 7, "packed"), ([300, 2000], 16, 1, 192, 64, "heads"),
                                                    ([0], 2, 1, 128, 16, "separate"), ([600, 1023], 33, 1, 128, 8, "separate")],
                         ids=["777", "one", "empty-first", "4000", "wide-groups", "192", "nothing", "page-8"])
def test_attention_little_work(native_built, lens, hq, hk, D, bs, layout, dtype):
    """Few heads and short table rows, which clusters take."""
    from pla_b200 import capi
    import ctypes
    q, kc, vc, table = paged_inputs(len(lens) * D + hq, lens, hq, hk, D, bs, DT[dtype], layout, extra_columns=0)
    a = capi.pla_b200_paged_decode_args(B=len(lens), Hq=hq, Hk=hk, D=D, block_size=bs, columns=table.shape[1])
    assert capi.load().pla_b200_paged_decode_workspace_bytes(ctypes.byref(a)) == 0
    status = word()
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens), return_lse=True, status=status)
    assert status.item() == 0
    assert_attention(out, lse, q, kc, vc, table, lens)
    again = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens), out=torch.full_like(out, float("nan")))
    assert torch.equal(again, out)
    # a wide table takes the other way: the same values within both ways' bounds
    wide = torch.full((len(lens), 20000 // bs + 1), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, wide.cuda(), i32(lens), return_lse=True)
    assert_attention(out, lse, q, kc, vc, table, lens)


@pytest.mark.gpu
def test_attention_peaked_and_extreme_scores(native_built):
    """Scores of hundreds, rising and falling along the context (the running maximum changes at every step or never), all equal, and
    negative scale."""
    lens, bs, D = [600, 600, 600], 16, 128
    q, kc, vc, table = paged_inputs(5, lens, 4, 2, D, bs)
    ramp = torch.linspace(-30, 30, 600)
    for b, r in ((0, ramp), (1, ramp.flip(0)), (2, torch.zeros(600))):
        t = torch.arange(600)
        at = (table[b, t // bs].long().cuda(), (t % bs).cuda())
        kc[at] = (r[:, None, None].expand(600, 2, D) / 8).bfloat16().cuda()
    q = torch.full_like(q, 2.0)
    for scale in (D ** -0.5, 2.0, -1.0, 0.0):
        out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens), scale=scale, return_lse=True)
        assert_attention(out, lse, q, kc, vc, table, lens, scale)


def assert_attention_kept(got, lse, q, kc, vc, table, lens, scale=None):
    """``assert_attention`` with the weights of the softmax held in more bits than one number of the activations' type: as two of them, each
    is within half(t)^2 of itself; an fp16 weight also within 2^-32 of the largest one, 2^-25 (half of fp16's smallest step) with the
    weights 2^7 times as large. The rest of the bound is the same."""
    out, want_lse, spread, reach = ofa.paged_attention(q, kc.cpu(), vc.cpu(), table, lens, scale)
    D, n = q.shape[-1], torch.tensor([max(int(x), 0) for x in lens], dtype=torch.float64)[:, None]
    e, sums = D * 2.0 ** -24 * reach, (n + 64) * 2.0 ** -24
    lost = 0.0
    if q.dtype == torch.float16:
        bs, heads = kc.shape[1], q.shape[1] // kc.shape[2]
        lost = torch.zeros_like(out)
        for b, length in enumerate(lens):
            t = torch.arange(max(int(length), 0))
            v = vc.cpu()[table[b, t // bs].long(), t % bs].double().abs().sum(0)          # [kv heads, channels]
            lost[b] = 2.0 ** -32 * v.repeat_interleave(heads, 0)                           # the largest weight is at most 1
    assert_within(got, out, (half(q.dtype) ** 2 + 2 * e + 2 * sums + 2.0 ** -20)[..., None] * spread + lost)
    if lse is not None:
        assert_attention(got, lse, q, kc, vc, table, lens, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lens,hq,hk,D,bs,layout", [(EDGES, 16, 2, 256, 16, "separate"), (EDGES, 5, 1, 96, 7, "separate"), (EDGES, 33, 1, 128, 16, "packed"),
                                                    (EDGES, 12, 3, 64, 1, "heads"), ([777], 16, 2, 128, 16, "separate"), ([0, 70, 513], 34, 2, 192, 32, "packed")])
def test_attention_keeps_the_weights(native_built, lens, hq, hk, D, bs, layout, dtype):
    """The output is the 32-bit value, rounded once: the weights' own rounding does not show."""
    q, kc, vc, table = paged_inputs(hq + D, lens, hq, hk, D, bs, DT[dtype], layout, extra_columns=0)
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens), return_lse=True)
    assert_attention_kept(out, lse, q, kc, vc, table, lens)


@pytest.mark.gpu
def test_attention_fp16_tail_behind_one_token(native_built):
    """One token 25.1 powers of two above 2^16 - 1 others: fp16 has no number that small beside 1, but the sum counts them. All values are 1, so
    the output is exactly 1. There is one request per CTA (three of 64 channels per SM), so that one warp owns the large weight and 2^14 of the
    small ones, 2^-11.1 in all: without them the output is a step below 1. Bound: the 2^10 sums of 16 tokens on the matrix unit are off
    by at most 2^-23 each, 2^-13; the 2^11 additions of the lane that holds the large weight by at most one small weight each, 2^-14.1;
    the weights in fp16 by 2^-32 each, 2^-18: together below 2^-12, half the step below 1."""
    B, D, bs, n = 3 * torch.cuda.get_device_properties(0).multi_processor_count, 64, 64, 1 << 16
    kc = torch.full((2, bs, 1, D), -1.0, dtype=torch.float16, device="cuda")
    kc[0, 0] = 0
    vc = torch.ones_like(kc)
    table = torch.ones(1, n // bs, dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    out, lse = fa().paged_attention_decode(torch.ones(B, 1, D, dtype=torch.float16, device="cuda"), kc, vc, table.expand(B, -1), i32([n] * B),
                                           scale=25.1 * math.log(2) / D, return_lse=True)
    assert torch.all(out == 1)
    assert (lse.double() - math.log1p((n - 1) * 2.0 ** -25.1)).abs().max().item() <= 2.0 ** -13


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("wide", [False, True], ids=["clusters", "two-kernels"])
@pytest.mark.parametrize("hq,hk,D,bs", [(4, 2, 64, 16), (3, 1, 256, 16), (18, 2, 128, 7), (6, 1, 96, 1)])
@pytest.mark.parametrize("where", ["query", "newest key", "first key", "all keys", "value"])
def test_attention_nan_stays(native_built, where, hq, hk, D, bs, wide, dtype):
    """A NaN reaches every output and sum of the softmax that it is part of, whichever way the call takes and whatever the CTA or warp that
    holds it has besides; rows of length 0 stay zeros. Everything else keeps its bound."""
    lens = [1, 64, 65, 0, 300, 16]
    q, kc, vc, table = paged_inputs(D + hq, lens, hq, hk, D, bs, DT[dtype], extra_columns=20000 // bs if wide else 0)
    if where == "query":
        q[:, 1, D // 2] = float("nan")
    for b, n in enumerate(lens):
        for t in {"newest key": [n - 1], "first key": [0], "all keys": range(n), "value": [n // 2]}.get(where, []):
            if n:
                (vc if where == "value" else kc)[table[b, t // bs].item(), t % bs, hk - 1, 3] = float("nan")
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens), return_lse=True)
    want, want_lse, spread, reach = ofa.paged_attention(q, kc.cpu(), vc.cpu(), table, lens)
    assert torch.equal(out.isnan().cpu(), want.isnan()) and torch.equal(lse.isnan().cpu(), want_lse.isnan())
    assert want.isnan().any() and not want.isnan().all()
    e, sums = D * 2.0 ** -24 * reach.nan_to_num(0.0), 400 * 2.0 ** -24
    assert_within(out.nan_to_num(0.0), want.nan_to_num(0.0), (half(q.dtype) + 2 * e + 2 * sums + 2.0 ** -20)[..., None] * spread.nan_to_num(0.0))
    live = torch.isfinite(want_lse)
    assert torch.equal(lse.cpu()[3], torch.full((hq,), -math.inf))
    assert ((lse.cpu().double() - want_lse).abs() - e - sums - 2.0 ** -22 * (1 + want_lse.abs()))[live].le(0).all()


@pytest.mark.gpu
def test_attention_views_and_streams(native_built):
    """q as a slice of a wider row and with heads outermost, a table that is a slice of a wider one, another stream, two calls at
    once: the same results."""
    lens = [70, 500, 33, 2000]
    q, kc, vc, table = paged_inputs(9, lens, 16, 2, 128, 16)
    dq, dt, dl = q.cuda(), table.cuda(), i32(lens)
    want = fa().paged_attention_decode(dq, kc, vc, dt, dl)
    assert_attention(want, None, q, kc, vc, table, lens)
    wide = torch.zeros(4, 20 * 128 + 8, dtype=q.dtype, device="cuda")
    wide[:, 8:8 + 16 * 128] = dq.flatten(1)
    assert torch.equal(fa().paged_attention_decode(wide[:, 8:8 + 16 * 128].unflatten(1, (16, 128)), kc, vc, dt, dl), want)
    assert torch.equal(fa().paged_attention_decode(dq.transpose(0, 1).contiguous().transpose(0, 1), kc, vc, dt, dl), want)
    big = torch.full((4, table.shape[1] + 5), -3, dtype=torch.int32, device="cuda")
    big[:, 2:2 + table.shape[1]] = dt
    assert torch.equal(fa().paged_attention_decode(dq, kc, vc, big[:, 2:2 + table.shape[1]], dl), want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(fa().paged_attention_decode(dq, kc, vc, dt, dl))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.gpu
def test_attention_bad_metadata_is_flagged(native_built):
    """Pages outside the pool are left out, lengths past the row are cut, negative ones are empty: no access out of range (both the host
    checks and the kernel's own bounds), a bit in the status."""
    lens = [100, 50, 20]
    q, kc, vc, table = paged_inputs(11, lens, 8, 2, 64, 16, extra_columns=0)
    table[0, 2], table[0, 4], table[1, 0] = -1, kc.shape[0], 1 << 30
    status = word()
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens), return_lse=True, status=status)
    assert status.item() == 8
    assert_attention(out, lse, q, kc, vc, table, lens)
    table[2, 2:] = -1
    status.zero_()
    bad = [100, -4, table.shape[1] * 16 + 9]
    kc.nan_to_num_(0.5), vc.nan_to_num_(0.5)
    out, lse = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(bad), return_lse=True, status=status)
    assert status.item() == 9
    assert_attention(out, lse, q, kc, vc, table, bad)
    none = torch.zeros(0, 16, 2, 64, dtype=torch.bfloat16, device="cuda")         # an empty pool: nothing can be read
    out = fa().paged_attention_decode(q.cuda(), none, none, table.cuda(), i32(lens), status=status)
    assert torch.all(out == 0)
    out = fa().paged_attention_decode(q.cuda(), kc, vc, table[:, :0].cuda(), i32([0, 0, 0]))
    assert torch.all(out == 0)
    assert fa().paged_attention_decode(q[:0].cuda(), kc, vc, table[:0].cuda(), i32([])).shape == (0, 8, 64)


@pytest.mark.gpu
def test_attention_cache_past_32_bit_offsets(native_built):
    """Pages whose element offsets pass 2^31 and 2^32: the same results as from a small pool."""
    bs, hk, D, lens = 256, 8, 128, [1000, 300]
    q, kc, vc, table = paged_inputs(3, lens, 16, hk, D, bs, extra_columns=0)
    want = fa().paged_attention_decode(q.cuda(), kc, vc, table.clamp(max=kc.shape[0] - 1).cuda(), i32(lens))
    blocks = (1 << 32) // (bs * hk * D) + 16
    if torch.cuda.mem_get_info()[0] < 3 * blocks * bs * hk * D * 2:
        pytest.skip("needs 26 GB")
    big_k = torch.empty(blocks, bs, hk, D, dtype=torch.bfloat16, device="cuda")
    big_v = torch.empty(blocks, bs, hk, D, dtype=torch.bfloat16, device="cuda")
    move = [blocks - 1 - i if i % 2 else blocks // 2 + i for i in range(kc.shape[0])]
    big_k[move], big_v[move] = kc, vc
    moved = torch.tensor([[move[x] if x < kc.shape[0] else 0 for x in r] for r in table.tolist()], dtype=torch.int32)
    assert torch.equal(fa().paged_attention_decode(q.cuda(), big_k, big_v, moved.cuda(), i32(lens)), want)
    # and the write of a row there
    x = torch.randn(1, hk, D).bfloat16().cuda()
    slot = torch.tensor([(blocks - 3) * bs + 5], device="cuda")
    fa().qk_norm_rotary_cache(x, x, x, None, None, i32([0]), torch.ones(8, dtype=torch.float64, device="cuda"), big_k, big_v, slot)
    assert torch.equal(big_k[blocks - 3, 5], x[0]) and torch.equal(big_v[blocks - 3, 5], x[0])


@pytest.mark.gpu
def test_attention_through_the_abi(native_built):
    """The C entry with a workspace that holds garbage; a missing, a too small and an unaligned one are refused."""
    import ctypes
    from pla_b200 import capi
    lib = capi.load()
    lens = [900, 0, 4100]
    q, kc, vc, table = paged_inputs(21, lens, 16, 8, 128, 16)
    dq, dt, dl, out, lse = q.cuda(), table.cuda(), i32(lens), torch.empty_like(q, device="cuda"), torch.empty(3, 16, device="cuda")
    a = capi.pla_b200_paged_decode_args(q=dq.data_ptr(), q_row_stride=dq.stride(0), q_head_stride=dq.stride(1), k_cache=kc.data_ptr(),
                                        v_cache=vc.data_ptr(), block_table=dt.data_ptr(), table_row_stride=dt.stride(0),
                                        seq_lens=dl.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), num_blocks=kc.shape[0], block_size=16,
                                        columns=dt.shape[1], B=3, Hq=16, Hk=8, D=128, act_dtype=0, scale=128 ** -0.5)
    for name, x in (("k_strides", kc), ("v_strides", vc)):
        st = getattr(a, name)
        st.block, st.token, st.head = x.stride(0), x.stride(1), x.stride(2)
    size = lib.pla_b200_paged_decode_workspace_bytes(ctypes.byref(a))
    assert size > 0
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.pla_b200_paged_decode(ctypes.byref(a), stream) == -1 and b"workspace" in lib.pla_b200_last_error()
    space = torch.full((size + 16,), 0xff, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = space.data_ptr(), size - 1
    assert lib.pla_b200_paged_decode(ctypes.byref(a), stream) == -1
    a.workspace, a.workspace_bytes = space.data_ptr() + 8, size
    assert lib.pla_b200_paged_decode(ctypes.byref(a), stream) == -2
    a.workspace = space.data_ptr()
    assert lib.pla_b200_paged_decode(ctypes.byref(a), stream) == 0, lib.pla_b200_last_error()
    torch.cuda.synchronize()
    assert (space[size:] == 0xff).all()
    assert_attention(out, lse, q, kc, vc, table, lens)


@pytest.mark.gpu
def test_attention_refusals(native_built):
    f = fa().paged_attention_decode
    q, kc = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    table, lens = i32([[0], [1]]), i32([1, 1])
    for args, match in [((q.float(), kc, kc, table, lens), "bf16 or fp16"), ((q.half(), kc, kc, table, lens), "dtype"), ((q[:, :3], kc, kc, table, lens), "multiple"),
                        ((q[0], kc, kc, table, lens), "shape"), ((q, kc[..., :32], kc[..., :32], table, lens), "of size"), ((q, kc, kc[:2], table, lens), "same shape"),
                        ((q, kc, kc, table.long(), lens), "int32"), ((q, kc, kc, table[:1], lens), "one row per request"), ((q, kc, kc, table, lens.long()), "seq_lens"),
                        ((q, kc, kc, table, lens.cpu()), "seq_lens"), ((q, kc[0], kc[0], table, lens), "shape"),
                        ((torch.zeros(2, 4, 80, dtype=torch.bfloat16, device="cuda"), kc, kc, table, lens), "head size")]:
        with pytest.raises(RuntimeError, match=match):
            f(*args)
    with pytest.raises(RuntimeError, match="out must"):
        f(q, kc, kc, table, lens, out=q[:1])
    with pytest.raises(RuntimeError, match="scale"):
        f(q, kc, kc, table, lens, scale=math.inf)
    odd = torch.zeros(3 * 16 * 2 * 68, dtype=torch.bfloat16, device="cuda").as_strided((3, 16, 2, 64), (16 * 2 * 68, 2 * 68, 68, 1))
    with pytest.raises(RuntimeError, match="aligned"):
        f(q, odd, odd, table, lens)


@pytest.mark.gpu
def test_scalars_outside_32_bits_are_refused(native_built):
    q, kc = torch.ones(1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    freq, w = torch.ones(4, dtype=torch.float64, device="cuda"), torch.ones(64, device="cuda")
    for scale in (1e39, -1e300, math.nan):
        with pytest.raises(RuntimeError, match="scale"):
            fa().paged_attention_decode(q, kc, kc, i32([[0]]), i32([3]), scale=scale)
    for kw in (dict(factor=1e39), dict(factor=math.nan), dict(eps=1e39), dict(eps=1e-60), dict(eps=-1e-6), dict(eps=math.nan)):
        with pytest.raises(RuntimeError, match="32-bit"):
            fa().qk_norm_rotary(q, None, w, None, i32([0]), freq, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hq,hk,D,R", [(1, 1, 8, 2), (32, 8, 128, 128), (16, 2, 256, 64), (5, 1, 96, 48), (3, 2, 128, 40), (2, 1, 64, 20)])
def test_one_token_is_rotated(native_built, hq, hk, D, R, inter, dtype):
    """A decode step's rotation, at positions where no angle is a whole turn; with the norm and without."""
    g = torch.Generator().manual_seed(D + R)
    row, (q, k, _) = rows(g, 1, hq, hk, D, DT[dtype])
    w = torch.rand(D, generator=g) + 0.5
    freq = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / R)
    dq, dk, _ = on_gpu(row, hq, hk, D)
    for position in (1, 777777, -5):
        pos = torch.tensor([position])
        for weight in (None, w):
            dw = None if weight is None else weight.cuda()
            got = fa().qk_norm_rotary(dq, dk, dw, dw, pos.cuda(), freq.cuda(), interleaved=inter)
            for x, y, name in zip((q, k), got, "qk"):
                want, bound = expect(x, weight, pos, freq, inter)
                assert_within(y, want, bound, name)
                assert weight is not None or not torch.equal(y.cpu(), x)


@pytest.mark.gpu
def test_overlapping_outputs_are_refused(native_built):
    """What a call writes may be its own input, element for element, and nothing else that the call reads or writes; no row of it twice."""
    T, D, bf = 6, 64, dict(dtype=torch.bfloat16, device="cuda")
    freq, pos, w = torch.ones(8, dtype=torch.float64, device="cuda"), torch.arange(T, device="cuda"), torch.ones(D, device="cuda")
    flat = torch.randn(4 * T * 4 * D, **bf)
    q, k = torch.randn(T, 4, D, **bf), torch.randn(T, 4, D, **bf)
    row = flat[:T * 12 * D].view(T, 12, D)
    for kw in [dict(out_q=q[:1].expand(T, 4, D)), dict(out_q=q[:, :1].expand(T, 4, D)), dict(out_k=k[:1].expand(T, 4, D)), dict(out_q=k), dict(out_k=q),
               dict(out_q=q, out_k=q), dict(out_q=row[:, :4], out_k=row[:, 2:6]), dict(out_q=row[:, 8:], out_k=row[:, 8:]), dict(out_q=k, out_k=row[:, :4]), dict(out_q=row[:, :4], out_k=q),
               dict(out_q=flat.as_strided((T, 4, D), (3 * D, D, 1)))]:
        for call in (lambda: fa().apply_rotary(q, k, pos, freq, **kw), lambda: fa().qk_norm_rotary(q, k, w, w, pos, freq, **kw)):
            with pytest.raises(RuntimeError, match="overlap"):
                call()
    with pytest.raises(RuntimeError, match="overlap"):                           # a row further on in the same tensor
        fa().apply_rotary(flat[:T * 4 * D].view(T, 4, D), None, pos, freq, out_q=flat[4 * D:(T + 1) * 4 * D].view(T, 4, D))
    with pytest.raises(RuntimeError, match="overlap"):
        fa().apply_rotary(q[:1].expand(T, 4, D), None, pos, freq, out_q=q[:1].expand(T, 4, D))
    cache = torch.randn(3, 2, 16, 4, D, **bf)
    kc, vc = cache[:, 0], cache[:, 1]
    slots = torch.arange(T, device="cuda")
    rest = dict(q=q, k=k, v=k, q_weight=w, k_weight=w, positions=pos, inv_freq=freq, k_cache=kc, v_cache=vc, slot_mapping=slots)
    for over in [dict(v_cache=kc), dict(k_cache=kc[:1].expand(3, 16, 4, D)), dict(v_cache=vc[:, :1].expand(3, 16, 4, D)), dict(k=kc[0, :T]), dict(v=kc[0, :T]),
                 dict(q=vc[1, :T]), dict(out_q=vc[1, :T]), dict(out_q=k), dict(v_cache=cache.flatten(0, 1)[1:4])]:
        with pytest.raises(RuntimeError, match="overlap"):
            fa().qk_norm_rotary_cache(**(rest | over))
    table, lens = i32([[0, 1]] * T), i32([5] * T)
    for out in (kc[0, :T], flat[:T * 4 * D].view(T, 4, D)):
        with pytest.raises(RuntimeError, match="overlap"):
            fa().paged_attention_decode(flat[D:D + T * 4 * D].view(T, 4, D) if out.data_ptr() == flat.data_ptr() else q, kc, vc, table, lens, out=out)
    both = torch.arange(12, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="overlap"):
        fa().build_block_tables(both[:4].view(2, 2), i32([0, 0]), i32([0, 1, 2]), both[3:], 4, num_tokens=2)


@pytest.mark.gpu
def test_in_place_and_interleaved_views(native_built):
    """Outputs that are their inputs, or lie between them: parts of one packed row, heads side by side, heads outermost, halves of one
    cache, the attention's output in place of its queries. The same bits as with tensors of their own."""
    T, H, D, bf = 70, 4, 128, dict(dtype=torch.bfloat16, device="cuda")
    freq, pos, w = fa().rotary_frequencies(64)[0].cuda(), torch.arange(T, device="cuda"), torch.rand(D, device="cuda")
    fresh = torch.randn(3, T, H, D, **bf)
    want = fa().qk_norm_rotary(fresh[0], fresh[1], w, w, pos, freq)
    packed = torch.cat([x.flatten(1) for x in fresh], 1).contiguous()
    side = torch.stack(list(fresh), 2)                                            # [T, H, 3, D]
    outer = fresh.transpose(1, 2).contiguous()                                    # [3, H, T, D]
    for q, k, v in ((packed[:, :H * D].unflatten(1, (H, D)), packed[:, H * D:2 * H * D].unflatten(1, (H, D)), packed[:, 2 * H * D:].unflatten(1, (H, D))),
                    (side[:, :, 0], side[:, :, 1], side[:, :, 2]), [x.transpose(0, 1) for x in outer]):
        cache = torch.zeros(6, 2, 16, H, D, **bf)
        out = fa().qk_norm_rotary_cache(q, k, v, w, w, pos, freq, cache[:, 0], cache[:, 1], torch.arange(T, device="cuda"), out_q=q)
        assert out.data_ptr() == q.data_ptr() and torch.equal(q, want[0])
        assert torch.equal(cache[:, 0].flatten(0, 1)[:T], want[1]) and torch.equal(cache[:, 1].flatten(0, 1)[:T], fresh[2])
        fa().qk_norm_rotary(v, k, w, w, pos, freq, out_q=v, out_k=k)
        assert torch.equal(k, want[1]) and torch.equal(v, fa().qk_norm_rotary(fresh[2], None, w, None, pos, freq)[0])
    for lens, hq, hk, columns in ([70, 0, 500, 33], 16, 2, 2), ([70, 0, 2000, 33], 16, 2, 1000), ([900] * 40, 8, 8, 0):
        q, kc, vc, table = paged_inputs(9, lens, hq, hk, 128, 16, extra_columns=columns)
        want = fa().paged_attention_decode(q.cuda(), kc, vc, table.cuda(), i32(lens))
        x = q.cuda()
        got = fa().paged_attention_decode(x, kc, vc, table.cuda(), i32(lens), out=x)
        assert got.data_ptr() == x.data_ptr() and torch.equal(got, want)


@pytest.mark.gpu
def test_sanity_check_names_bad_metadata(native_built, monkeypatch):
    monkeypatch.setenv("PLA_SANITY_CHECK", "1")
    q, kc = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="page 3 of request 0"):
        fa().paged_attention_decode(q, kc, kc, i32([[0, 3]]), i32([17]))
    with pytest.raises(RuntimeError, match="length 40"):
        fa().paged_attention_decode(q, kc, kc, i32([[0, 1]]), i32([40]))
    with pytest.raises(RuntimeError, match="slot index 48"):
        fa().qk_norm_rotary_cache(q, q, q, None, None, i32([0]), torch.ones(2, dtype=torch.float64, device="cuda"), kc, kc.clone(), i32([48]))
    with pytest.raises(RuntimeError, match="decrease"):
        fa().build_block_tables(i32([[0], [0]]), i32([0, 0]), i32([0, 2, 1]), i32([1]), 4, num_tokens=2)


# ------------------------------------------------------------------------------------------------ together
class Layer:
    """One full-attention layer of a serving loop, and the same in 64 bits on dense rows that the test keeps."""

    def __init__(self, hq, hk, D, R, bs, blocks, requests, columns, seed):
        self.g = torch.Generator().manual_seed(seed)
        self.hq, self.hk, self.D, self.bs = hq, hk, D, bs
        self.kc, self.vc = caches(blocks, bs, hk, D, torch.bfloat16, "packed")
        self.table = torch.full((requests, columns), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(blocks, generator=self.g).to(torch.int32).cuda()
        self.freq, self.factor = fa().rotary_frequencies(R, scaling="yarn", factor=4.0, original_max_position=64)
        self.qw, self.kw = ((torch.randn(D, generator=self.g) * 0.1 + 1).bfloat16() for _ in range(2))
        self.dfreq, self.dqw, self.dkw = self.freq.cuda(), self.qw.cuda(), self.kw.cuda()
        self.keys, self.values = [[] for _ in range(requests)], [[] for _ in range(requests)]

    def rows(self, T):
        return torch.randn(T, (self.hq + 2 * self.hk) * self.D, generator=self.g).bfloat16()

    def write(self, row, plan):
        q, k, v = (x.unflatten(1, (-1, self.D)) for x in row.split([self.hq * self.D, self.hk * self.D, self.hk * self.D], 1))
        return fa().qk_norm_rotary_cache(q, k, v, self.dqw, self.dkw, plan.positions, self.dfreq, self.kc, self.vc, plan.slot_mapping,
                                         factor=self.factor)

    def remember(self, row, lens, offsets, out, slots):
        """Checks the queries and the rows that the cache got; the rows as they are stored there go to the dense lists."""
        q, k, v = (x.unflatten(1, (-1, self.D)) for x in row.split([self.hq * self.D, self.hk * self.D, self.hk * self.D], 1))
        pos = torch.cat([torch.arange(n) + c for c, n in zip(lens, (b - a for a, b in zip(offsets, offsets[1:])))])
        y, bound = expect(q, self.qw, pos, self.freq, False, self.factor)
        assert_within(out, y, bound, "q")
        y, bound = expect(k, self.kw, pos, self.freq, False, self.factor)
        stored, values = self.kc[slots // self.bs, slots % self.bs], self.vc[slots // self.bs, slots % self.bs]
        assert_within(stored, y, bound, "k")
        assert torch.equal(values.cpu(), v)
        for n, (a, b) in enumerate(zip(offsets, offsets[1:])):
            self.keys[n] += list(stored[a:b].cpu())
            self.values[n] += list(values[a:b].cpu())

    def check_attention(self, out, q, n):
        k, v = (torch.stack(x[n])[:, None] for x in (self.keys, self.values))
        assert_attention(out[n:n + 1], None, q[n:n + 1].cpu(), k, v, torch.arange(len(k))[None], [len(k)])


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_prefill_then_decode_steps_together(native_built, captured):
    """Three prompts enter the cache, then every request gets one token per step, eagerly or as replays of one captured step (with a
    padding row). Queries and stored rows against the formula, attention against dense attention in 64 bits over everything a
    request has stored so far."""
    hq, hk, D, bs, prompts, steps = 6, 2, 128, 16, [37, 5, 64], 20
    layer = Layer(hq, hk, D, 64, bs, 40, 4, 8, seed=2)
    offsets = [0, 37, 42, 106, 106]
    row = layer.rows(106)
    plan = fa().build_block_tables(layer.table, i32([0] * 4), i32(offsets), layer.free, bs, num_tokens=106)
    q = layer.write(row.cuda(), plan)
    layer.remember(row, [0] * 4, offsets, q, plan.slot_mapping)
    assert plan.seq_lens.tolist() == prompts + [0]

    one = i32([0, 1, 2, 3, 3])                      # the fourth row is padding
    lens, start = plan.seq_lens.clone(), plan.free_next.clone()
    status, token = word(), torch.zeros(4, (hq + 2 * hk) * D, dtype=torch.bfloat16, device="cuda")

    def step():
        p = fa().build_block_tables(layer.table, lens, one, layer.free, bs, num_tokens=4, free_start=start, status=status)
        q = layer.write(token, p)
        out = fa().paged_attention_decode(q, layer.kc, layer.vc, p.block_table, p.seq_lens, status=status)
        lens.copy_(p.seq_lens)
        start.copy_(p.free_next)
        return out, q, p.slot_mapping

    graph = None
    if captured:
        keep = [x.clone() for x in (layer.table, lens, start, layer.kc, layer.vc)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = step()
        for x, y in zip((layer.table, lens, start, layer.kc, layer.vc), keep):
            x.copy_(y)
    for i in range(steps):
        row = layer.rows(4)
        token.copy_(row)
        if captured:
            graph.replay()
            out, q, slots = result
        else:
            out, q, slots = step()
        assert slots[3] == -1 and torch.all(out[3] == 0)
        layer.remember(row[:3], [p + i for p in prompts], [0, 1, 2, 3], q[:3], slots[:3])
        for n in range(3):
            layer.check_attention(out, q, n)
    assert status.item() == 0
    assert lens.tolist() == [p + steps for p in prompts] + [0]
    used = [x for r, n in zip(layer.table.tolist(), lens.tolist()) for x in r[:-(-n // bs)]]
    assert len(set(used)) == len(used) == start.item()


@pytest.mark.gpu
def test_two_captured_steps_run_at_once(native_built):
    """Two graphs captured from the same operators, replayed on two streams at the same time: each has its own scratch."""
    cases = [([3000, 20], 16, 2, 128), ([1500] * 5, 8, 8, 64)]
    graphs = []
    for lens, hq, hk, D in cases:
        q, kc, vc, table = paged_inputs(D, lens, hq, hk, D, 16)
        args = (q.cuda(), kc, vc, table.cuda(), i32(lens))
        want = fa().paged_attention_decode(*args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = fa().paged_attention_decode(*args)
        graphs.append((g, out, want, args, torch.cuda.Stream()))
    for _ in range(5):
        for g, out, _, _, s in graphs:
            with torch.cuda.stream(s):
                out.fill_(float("nan"))
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for _, out, want, _, _ in graphs)
