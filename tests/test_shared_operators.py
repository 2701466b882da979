"""Refusals of the entry points for several continuations of one prompt (checked before anything is launched, so they
need no GPU) and the restatements' own properties."""
import numpy as np
import pytest

from oracle import beams as oracle

SHAPE, CAPACITY, ARGUMENT, UNSUPPORTED = 1, 2, 6, 7
A, B = 1 << 20, 1 << 21  # addresses that pass the checks of alignment; nothing is launched


@pytest.fixture(scope="module")
def lib():
    from sejong_b200 import _lib, build
    build.build()
    return _lib.load()


def refused(name, args, code, **kw):
    from sejong_b200._lib import SejongError, call
    assert set(kw) <= set(args), kw
    with pytest.raises(SejongError) as e:
        call(name, *{**args, **kw}.values())
    assert e.value.code == code, str(e.value)
    assert name in str(e.value)


FORK = dict(parent=A, batch=4, page=16, cached=A, table=A, ld_table=8, shares=A, free=A, count=A, pages=10, cached_out=B,
            table_out=B, shares_out=B, free_out=B, count_out=B, copies=B, summary=B, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), SHAPE), (dict(batch=4097), SHAPE), (dict(page=0), SHAPE), (dict(page=(1 << 20) + 1), SHAPE),
    (dict(ld_table=0), SHAPE), (dict(pages=0), SHAPE), (dict(pages=(1 << 18) + 1), SHAPE), (dict(parent=0), ARGUMENT),
    (dict(shares=0), ARGUMENT), (dict(copies=0), ARGUMENT), (dict(count_out=0), ARGUMENT), (dict(table_out=A), ARGUMENT),
    (dict(cached_out=A), ARGUMENT), (dict(free_out=A), ARGUMENT), (dict(shares_out=A), ARGUMENT)])
def test_fork_refusals(lib, kw, code):
    refused("sj_paged_fork", FORK, code, **kw)


COPY = dict(copies=A, most=3, k=A, v=A, layers=2, layer_stride=1 << 14, pages=8, page=16, page_stride=2048,
            head_stride=1024, token_stride=64, hk=2, dim=64, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(most=-1), SHAPE), (dict(layers=0), SHAPE), (dict(layers=4097), SHAPE), (dict(hk=0), SHAPE),
    (dict(dim=96), UNSUPPORTED), (dict(pages=0), SHAPE), (dict(page=0), SHAPE), (dict(copies=0), ARGUMENT),
    (dict(k=A + 8), ARGUMENT), (dict(v=0), ARGUMENT), (dict(layer_stride=4), ARGUMENT),
    (dict(layer_stride=-8), ARGUMENT), (dict(token_stride=60), ARGUMENT), (dict(page_stride=1 << 34), SHAPE)])
def test_copy_refusals(lib, kw, code):
    refused("sj_paged_copy", COPY, code, **kw)


COMPACT = dict(cached=A, batch=4, page=16, table=A, ld_table=8, shares=A, free=A, count=A, pages=10, table_out=B,
               shares_out=B, free_out=B, moves=B, most=5, summary=B, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(batch=0), SHAPE), (dict(batch=4097), SHAPE), (dict(page=0), SHAPE), (dict(pages=(1 << 18) + 1), SHAPE),
    (dict(most=-1), SHAPE), (dict(moves=0), ARGUMENT), (dict(cached=0), ARGUMENT), (dict(table_out=A), ARGUMENT),
    (dict(shares_out=A), ARGUMENT), (dict(free_out=A), ARGUMENT), (dict(summary=0), ARGUMENT)])
def test_compact_refusals(lib, kw, code):
    refused("sj_paged_compact", COMPACT, code, **kw)


SELECT = dict(logits=A, dtype=0, ld=300, score=A, requests=2, beams=3, vocab=257, keep=6, parent=A, token=A, best=A,
              workspace=0, size=0, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(requests=-1), SHAPE), (dict(requests=4097), SHAPE), (dict(beams=0), SHAPE), (dict(beams=65), SHAPE),
    (dict(vocab=0), SHAPE), (dict(ld=256), SHAPE), (dict(keep=0), SHAPE), (dict(keep=65), SHAPE),
    (dict(beams=1, vocab=5, keep=6), SHAPE), (dict(vocab=2 ** 31 - 1 - 2 ** 15, ld=2 ** 31 - 1), SHAPE),
    (dict(dtype=2), ARGUMENT), (dict(logits=0), ARGUMENT), (dict(logits=A + 2), ARGUMENT), (dict(score=0), ARGUMENT),
    (dict(parent=0), ARGUMENT), (dict(vocab=5000, ld=5000), CAPACITY),
    (dict(vocab=5000, ld=5000, workspace=A, size=64), CAPACITY)])
def test_select_refusals(lib, kw, code):
    refused("sj_beam_select", SELECT, code, **kw)


def test_no_work_launches_nothing(lib):
    from sejong_b200._lib import call
    call("sj_beam_select", *{**SELECT, "requests": 0}.values())
    call("sj_paged_copy", *{**COPY, "most": 0}.values())
    call("sj_attn_paged_shared", *{**SHARED, "rows": 0}.values())


SHARED = dict(q=A, ldq=256, k=A, v=A, pages=8, page=16, page_stride=2048, head_stride=1024, token_stride=64, table=A,
              ld_table=4, requests=3, request=0, position=A, rows=3, group=A, groups=1, hq=4, hk=2, dim=64, window=0, o=A,
              ldo=256, lse=0, workspace=A, size=1 << 30, stream=0)


@pytest.mark.parametrize("kw,code", [
    (dict(dim=80), UNSUPPORTED), (dict(rows=-1), SHAPE), (dict(hq=5), SHAPE), (dict(window=-1), SHAPE),
    (dict(requests=0), SHAPE), (dict(rows=4), SHAPE), (dict(groups=-1), SHAPE), (dict(groups=4), SHAPE),
    (dict(ldq=192), SHAPE), (dict(ldo=250), SHAPE), (dict(ldq=260), ARGUMENT), (dict(group=0), ARGUMENT),
    (dict(position=0), ARGUMENT), (dict(q=A + 8), ARGUMENT), (dict(size=0), CAPACITY), (dict(workspace=0), CAPACITY)])
def test_shared_refusals(lib, kw, code):
    refused("sj_attn_paged_shared", SHARED, code, **kw)


# ---------------------------------------------------------------- the restatements
def test_select_prefers_low_indices():
    x = np.zeros((1, 2, 3))
    parent, token, total = oracle.select(x, np.zeros((1, 2)), 4)
    assert parent.tolist() == [[0, 0, 0, 1]] and token.tolist() == [[0, 1, 2, 0]]
    assert np.allclose(total, -np.log(3))


def test_fork_shares_full_pages_and_copies_the_last():
    # two requests: 0 holds pages 5, 3 and half of 1; 1 holds 4
    cached, table = [10, 4], [[5, 3, 1], [4, -1, -1]]
    lengths, out, shares, free, copies, back, status = oracle.fork([0, 0], 4, cached, table, [0] * 6, [2, 0])
    assert status == 0 and back == 1 and lengths.tolist() == [10, 10]
    assert out.tolist() == [[5, 3, 1], [5, 3, 0]] and copies == [(1, 0, 2)]
    assert shares.tolist() == [0, 0, 0, 1, 0, 1] and free == [2, 4]
    assert oracle.fork([0, 0], 4, cached, table, [0] * 6, [])[-1] == 2


def test_compact_fills_holes_in_order():
    table, shares, free, moves = oracle.compact(4, [8, 4], [[5, 0], [3, -1]], [1, 0, 0, 0, 0, 2], [1, 4, 2], 6)
    assert moves == [(3, 1), (5, 2)] and table.tolist() == [[2, 0], [1, -1]]
    assert shares.tolist() == [1, 0, 2, 0, 0, 0] and free == [5, 4, 3]


# ---------------------------------------------------------------- what the kernels decide by, on the host
def host_program(where, body):
    """The output of a program with the kernels' own functions, which runs without a GPU."""
    import subprocess
    from sejong_b200 import build
    source, program = where / "host.cu", where / "host"
    source.write_text('#include <cstdio>\n#include "attention_paged.cuh"\nusing namespace sj;\nint main() {\n'
                      + body + "\nreturn 0;\n}\n")
    subprocess.run([build.nvcc(), *build.ARCH, *build.NVCC_FLAGS, str(source), "-o", str(program)], check=True)
    return subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split()


def test_blocks_that_were_never_written_are_no_ctas(tmp_path):
    """What a broken-off call leaves in the place of a block's CTAs: nothing that the join could go astray by."""
    ctas = 148
    cases = [(0, 0), (0, 147), (147, 147), (5, 9), (0, -1), (9, 5), (-1, 3), (-5, -2), (0, 148), (148, 148), (-2 ** 31, 2 ** 31 - 1),
             (0, 2 ** 31 - 1), (0x3f800000, 0x40000000), (2 ** 31 - 1, -2 ** 31)]
    body = "".join(f'printf("%d ", shared_span_fine(make_int2(int({a}ll), int({b}ll)), {ctas}));' for a, b in cases)
    assert [x == "1" for x in host_program(tmp_path, body)] == [0 <= a <= b < ctas for a, b in cases]


def test_groups_are_in_order_to_the_end(tmp_path):
    """A first row of `rows` ends the list: a smaller one after it is out of order, whatever comes then."""
    rows, requests, most = 9, 4, 100
    cases = [[0, 3, 5], [0, 9, 9], [9, 9, 9], [0, 9, 5], [0, 9, 5, 9], [9, 0], [0, 5, 5], [5, 3], [-1, 3], [0, 10], [8], [9], [10]]
    body = ""
    for first in cases:
        body += f"{{ const int32_t g[] = {{{', '.join(f'{f}, 1, 7' for f in first)}}}; int fine = 1; " \
                f"for (int t = 0; t < {len(first)}; ++t) fine &= shared_group_fine(g, t, {len(first)}, {rows}, {requests}, {most}); " \
                "printf(\"%d \", fine); }\n"
    for b, n in ((-1, 7), (4, 7), (3, -1), (3, 101), (3, 100)):
        body += f"{{ const int32_t g[] = {{0, {b}, {n}}}; printf(\"%d \", shared_group_fine(g, 0, 1, {rows}, {requests}, {most})); }}\n"

    def in_order(first):
        starts = [f for f in first if f != rows]
        return first == starts + [rows] * (len(first) - len(starts)) and all(0 <= f < rows for f in starts) \
            and all(a < b for a, b in zip(starts, starts[1:]))

    assert [x == "1" for x in host_program(tmp_path, body)] == [in_order(c) for c in cases] + [False] * 4 + [True]


def test_warps_give_up_as_a_whole():
    """The warps of attn_shared_kernel that go on by the answer of a wait, and to instructions of all their lanes, wait as
    warps; only the one that issues products, and goes on in any case, and the last look before the end do not."""
    import os
    import re
    from sejong_b200 import build
    text = open(os.path.join(build.CSRC, "attention_shared.cu")).read()
    softmax, rest = text[text.index("if (warp < kSoftmaxWarps) {"):].split("} else if (warp == kMmaWarp) {")
    loads = rest[rest.index("both warps follow the order of all tiles"):rest.index("tc_fence_before();")]
    for part, waits in ((softmax, 4), (loads, 1)):
        assert len(re.findall(r"\bmbar_wait_warp\(", part)) == waits
        assert not re.findall(r"\bmbar_wait\(", part)


def test_load_warps_learn_of_every_wait_that_gave_up():
    """A wait of another warp may give up after they have asked for their last copies: they look behind the barrier of all
    warps, and then wait for the copies."""
    import os
    from sejong_b200 import build
    text = open(os.path.join(build.CSRC, "attention_shared.cu")).read()
    kernel = text[text.index("attn_shared_kernel(const __grid_constant__"):text.index("shared_join_kernel(const")]
    barrier, look = kernel.rindex("__syncthreads();"), kernel.index("warp >= kLoadWarp && *abort_flag != 0")
    assert barrier < look < kernel.index("mbar_wait(&full[last_slot], last_turn, nullptr")
