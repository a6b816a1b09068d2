"""Batches of a paged cache on the CPU: what is refused, where new tokens go, and that the work of the attention kernels covers every row and
every position that it sees exactly once."""
import random
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
OK, INVALID, SHAPE, OVERFLOW = 0, 1, 2, 3


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    out = tmp_path_factory.mktemp("paged") / "paged_plan_check"
    r = subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-I", str(ROOT / "lumen_b200" / "csrc"),
                        str(ROOT / "tests" / "cpp" / "paged_plan_check.cpp"), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]

    def run(seqs, pages=16, page=8, h_kv=2, n_head=4, causal=1, rows=16, keys=64, slots=296, first=None, stride=None):
        """seqs: (new tokens, positions, pages) of each."""
        stride = max((len(t) for _, _, t in seqs), default=0) if stride is None else stride
        words = [pages, page, h_kv, 64, 1, n_head, causal, rows, keys, slots, stride, len(seqs)]
        for i, (q, kv, t) in enumerate(seqs):
            words += [q, kv, -1 if first is None else first[i]] + list(t) + [-1] * (stride - len(t))
        r = subprocess.run([str(out)], input=" ".join(map(str, words)), capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr[-2000:]
        lines = r.stdout.splitlines()
        if int(lines[0]):
            return int(lines[0]), r.stderr
        named = {"token": [], "item": [], "join": []}
        for line in lines[2:]:
            word, *numbers = line.split()
            named[word].append(tuple(map(int, numbers)))
        return 0, tuple(map(int, lines[1].split())), named["token"], named["item"], named["join"]

    return run


@pytest.mark.parametrize("seqs,code", [
    ([(1, 9, [3])], OVERFLOW),                       # nine positions, one page of eight
    ([(1, 9, [3, 16])], INVALID),                    # page 16 of 16
    ([(1, 9, [3, -1])], INVALID),                    # no page given where one is needed
    ([(1, 9, [3, 3])], INVALID),                     # a page twice
    ([(3, 2, [0])], SHAPE),                          # more new tokens than positions
    ([(-1, 2, [0])], INVALID), ([(0, -2, [0])], INVALID),
    ([(1, 2 ** 31 - 1, [0])], OVERFLOW),
])
def test_refused(plan, seqs, code):
    assert plan(seqs)[0] == code


def test_refused_heads_and_positions(plan):
    assert plan([(1, 1, [0])], n_head=5)[0] == SHAPE and plan([(1, 1, [0])], n_head=0)[0] == SHAPE
    assert plan([(1, 1, [0])], first=[-5])[0] == INVALID


def test_refused_more_rows_than_a_gpu_holds(plan):
    assert plan([(2 ** 30 + 1, 1, [0])], h_kv=1, n_head=1, causal=0)[0] == INVALID
    assert plan([(2 ** 28, 1, [0]), (1, 1, [1])], h_kv=2, n_head=4, causal=0)[0] == INVALID


def test_numbers_behind_the_last_page_are_not_looked_at(plan):
    assert plan([(1, 8, [3, 77, -9])])[0] == OK and plan([(0, 0, [99])])[0] == OK and plan([])[0] == OK


def test_tokens_go_to_their_slots(plan):
    rc, (tokens, max_pos, shared, write_shared, can_append), tok, _, _ = plan([(3, 10, [5, 2]), (0, 4, [7]), (2, 2, [1])], first=[100, 0, 7])
    assert rc == OK and (tokens, max_pos, shared, write_shared, can_append) == (5, 102, 0, 0, 1)
    assert tok == [(5 * 8 + 7, 100), (2 * 8, 101), (2 * 8 + 1, 102), (8, 7), (9, 8)]


def test_shared_pages(plan):
    both = [(1, 9, [4, 5]), (1, 9, [4, 6])]
    assert plan(both)[1][2:4] == (1, 0)                                   # a common prefix that nobody writes
    assert plan([(1, 8, [4]), (1, 9, [4, 6])])[1][2:4] == (1, 1)          # the first sequence's new row is in it
    assert plan([(1, 9, [4, 6]), (1, 8, [4])])[1][2:4] == (1, 1)
    assert plan([(0, 8, [4]), (1, 9, [4, 6]), (0, 3, [6])])[1][2:4] == (1, 1)
    assert plan([(0, 8, [4]), (0, 8, [4])])[1][2:4] == (1, 0)


def test_a_query_without_positions_cannot_be_appended(plan):
    rc, head, tok, items, _ = plan([(3, 1, [4])], causal=0)
    assert rc == OK and head[4] == 0 and tok[0][0] == -1 and all(i[4:6] == (0, 1) for i in items)


def _covers(items, joins, seqs, h_kv, group, causal, rows, keys):
    parts = {}
    for s, h, row0, n, part, splits in joins:
        for i in range(splits):
            parts[part + i * n] = (s, h, row0, n)
    seen = {}
    for s, h, row0, n, key0, key1, part in items:
        assert 0 < n <= rows and key0 % keys == 0
        if part >= 0:
            assert parts.pop(part) == (s, h, row0, n) and key1 > key0
        seen.setdefault((s, h, row0, n), []).append((key0, key1, part))
    assert not parts
    for s, (q, kv, _) in enumerate(seqs):
        for h in range(h_kv):
            mine = sorted(k for k in seen if k[:2] == (s, h))
            at = 0
            for k in mine:
                assert k[2] == at
                at += k[3]
                end = (kv - q + (at - 1) // group + 1) if causal else kv
                spans = sorted(seen[k])
                assert spans[0][0] == 0 and spans[-1][1] == end and all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
                assert len(spans) == 1 or [p for _, _, p in spans] == [spans[0][2] + i * k[3] for i in range(len(spans))]
            assert at == q * group


@pytest.mark.parametrize("seed", range(30))
def test_every_row_meets_every_position_once(plan, seed):
    rng = random.Random(seed)
    page, h_kv, group, causal = rng.choice([8, 32, 256]), rng.choice([1, 2, 8]), rng.choice([1, 4, 7]), rng.randint(0, 1)
    rows, keys, slots = rng.choice([(16, 64, 296), (128, 128, 148), (256, 128, 148), (128, 64, 148)])
    seqs, pages = [], 0
    for _ in range(rng.randint(1, 9)):
        kv = rng.choice([0, 1, rng.randint(1, 300), rng.randint(1, 6000)])
        q = rng.choice([0, min(kv, 1), rng.randint(0, min(kv, 400))])
        need = -(-kv // page)
        seqs.append((q, kv, list(range(pages, pages + need))))
        pages += need
    rc, _, _, items, joins = plan(seqs, pages=max(pages, 1), page=page, h_kv=h_kv, n_head=h_kv * group, causal=causal, rows=rows, keys=keys, slots=slots)
    assert rc == OK
    _covers(items, joins, seqs, h_kv, group, causal, rows, keys)
    lengths = [i[5] - i[4] for i in items]
    assert lengths == sorted(lengths, reverse=True)


def test_few_long_sequences_fill_the_slots(plan):
    rc, _, _, items, joins = plan([(1, 16000, list(range(250)))], pages=250, page=64, h_kv=8, n_head=32, slots=148)
    assert rc == OK and 120 <= len(items) <= 148 and len(joins) == 8


def test_kernels_let_the_next_start_behind_their_allocation():
    """As the other kernels that take tensor memory: every CTA has its own by the time it lets the next kernel start, and waits for the kernel before on
    every way out."""
    seen = 0
    for p in sorted((ROOT / "lumen_b200" / "csrc").glob("paged*.cu")):
        for body in p.read_text().split("__global__")[1:]:
            assert "pdl_wait();" in body, p.name
            if "tcgen05.alloc" in body:
                between = body[body.index("tcgen05.alloc"): body.index("paged_start_next();")]
                assert "tcgen05.relinquish_alloc_permit" in between and "__syncthreads()" in between, p.name
                assert "return;" not in body[: body.index("tcgen05.alloc")], p.name
                seen += 1
    assert seen == 4
