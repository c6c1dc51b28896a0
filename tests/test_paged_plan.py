"""The host plan of a paged batch (bg_paged_plan.h), compiled for the CPU: every new row meets every
position it attends exactly once, through its own pages; refusals; where new rows are written."""
import os
import random
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "paged_plan")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-Wall",
                    "-Werror", os.path.join(HERE, "paged_plan.cpp"), "-o", exe], check=True)

    def run(rows, lens, tables, KV=8, G=4, D=128, dtype=1, page=64, n_pages=4096, cus=256, limits=None, repeat=2):
        stride = max((len(t) for t in tables), default=0)
        flat = [x for t in tables for x in list(t) + [-7] * (stride - len(t))]
        limits = limits or (max(1, len(rows)), max(1, sum(rows)), max(1, sum(map(len, tables))))
        words = [KV, G, D, dtype, page, n_pages, cus, *limits, repeat, len(rows), stride, *rows, *lens, *flat]
        out = subprocess.run([exe], input=" ".join(map(str, words)), capture_output=True, text=True, check=True).stdout
        if out.startswith("error "):
            return out[6:].strip()
        got = {ln.split()[0]: [int(x) for x in ln.split()[1:]] for ln in out.splitlines()}
        names = ("kind", "tok", "rho0", "n_rho", "table", "key0", "key1", "mask0", "chunk", "p0", "p1", "p2", "p3")
        got["units"] = [dict(zip(names, got["units"][i:i + 16])) for i in range(0, len(got["units"]), 16)]
        got["toks"] = [tuple(got["toks"][i:i + 3]) for i in range(0, len(got["toks"]), 4)]
        got["merges"] = [tuple(got["merges"][i:i + 3]) for i in range(0, len(got["merges"]), 4)]
        return got
    return run


def check(p, rows, lens, tables, G, page, dtype):
    """Coverage, bounds and partial slots of a plan."""
    T = sum(rows)
    n_tokens, n_parts, _, _, max_units, max_toks = p["counts"]
    assert n_tokens == T and len(p["units"]) <= max_units and len(p["toks"]) <= max_toks
    seq = [b for b, r in enumerate(rows) for _ in range(r)]
    pos = [n - r + i for r, n in zip(rows, lens) for i in range(r)]
    assert p["dst"] == [tables[seq[t]][pos[t] // page] * page + pos[t] % page for t in range(T)]
    seen = [[[] for _ in range(G)] for _ in range(T)]     # per (token, head): (key0, key1) scanned
    slots = [[set() for _ in range(G)] for _ in range(T)]
    merged = {t: (part, n) for t, part, n in p["merges"]}
    assert len(merged) == len(p["merges"]) and all(n > 1 for _, n in merged.values())
    taken = sorted((part, part + n) for part, n in merged.values())
    assert all(a[1] <= b[0] for a, b in zip(taken, taken[1:])) and (not taken or taken[-1][1] <= n_parts)
    for u in p["units"]:
        width = {0: 128, 1: 32, 2: 16}[u["kind"]]
        assert 1 <= u["n_rho"] <= width
        assert u["key0"] % 32 == 0 and u["key0"] <= u["key1"]
        if u["kind"] == 0 and u["key1"] > u["key0"]:      # a step of 64 holds no half of another chunk
            assert (u["key1"] - u["key0"]) % 64 == 0 or u["mask0"] <= u["key1"]
        for rho in range(u["rho0"], u["rho0"] + u["n_rho"]):
            t, at, part = p["toks"][u["tok"] + rho // G]
            assert at == pos[t]
            lo, hi = u["key0"], min(u["key1"], at + 1)
            if u["mask0"] < u["key1"]:
                assert u["mask0"] <= at + 1
            else:
                assert u["key1"] <= at + 1                # unmasked: the row sees the whole unit
            if hi > lo:
                own = tables[seq[t]]
                for i in range(lo // page, (hi - 1) // page + 1):
                    assert p["pages"][u["table"] + i] == own[i]
                seen[t][rho % G].append((lo, hi))
            for w in range(4):                                # the pages of a unit's first tiles
                if u["key0"] + 32 * w < u["key1"]:
                    assert u[f"p{w}"] == p["pages"][u["table"] + (u["key0"] + 32 * w) // page]
            # what the kernels read past the row's positions is still inside a listed page
            assert u["key1"] == 0 or u["table"] + (u["key1"] - 1) // page < len(p["pages"])
            if t in merged:
                assert merged[t][0] <= part + u["chunk"] < merged[t][0] + merged[t][1]
                assert part + u["chunk"] not in slots[t][rho % G]
                slots[t][rho % G].add(part + u["chunk"])
            else:
                assert part == -1 and not slots[t][rho % G]
                slots[t][rho % G].add(-1)
    for t in range(T):
        for g in range(G):
            spans = sorted(seen[t][g])
            assert spans[0][0] == 0 and spans[-1][1] == pos[t] + 1
            assert all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
            assert len(slots[t][g]) == (merged[t][1] if t in merged else 1)
    stored = [t for t in p["v_single"]] + [t + i for t in p["v_group"] for i in range(16)]
    assert sorted(stored) == list(range(T))
    for t in p["v_group"]:
        assert p["dst"][t] % 16 == 0 and [p["dst"][t + i] - p["dst"][t] for i in range(16)] == list(range(16))


def tree(rng, B, page, max_len):
    """Page lists of B sequences forked from each other at page borders, new rows in pages of their own."""
    ids = iter(range(10 ** 6))
    tables, lens, rows = [], [], []
    for b in range(B):
        parent = rng.randrange(b) if b and rng.random() < 0.8 else None
        keep = 0 if parent is None else rng.randint(0, (lens[parent] - rows[parent]) // page)
        r = rng.choice([0, 1, 1, 1, rng.randint(1, 9), rng.randint(1, 200)])
        n = keep * page + rng.randint(r, max(r, max_len))
        tables.append((tables[parent][:keep] if parent is not None else []) + [next(ids) for _ in range(-(-n // page) - keep)])
        rows.append(r)
        lens.append(n)
    return rows, lens, tables, next(ids)


@pytest.mark.parametrize("seed", range(40))
def test_plan_covers_every_row_once(plan, seed):
    rng = random.Random(seed)
    page = rng.choice([32, 64, 128, 256])
    G = rng.choice([1, 2, 4, 6, 8, 40])
    dtype, D = rng.choice([0, 1, 2]), rng.choice([128, 256])
    rows, lens, tables, n_pages = tree(rng, rng.choice([1, 2, 7, 20]), page, rng.choice([3, 70, 1000, 5000]))
    p = plan(rows, lens, tables, KV=rng.choice([1, 4, 8]), G=G, D=D, dtype=dtype, page=page, n_pages=n_pages,
             cus=rng.choice([1, 80, 256]))
    assert isinstance(p, dict), p
    assert p["counts"][3] == -1
    check(p, rows, lens, tables, G, page, dtype)


def test_a_common_prefix_is_scanned_once(plan):
    pre = list(range(100))
    tables = [pre + [200 + b] for b in range(32)]
    lens = [6400 + 1 + b for b in range(32)]
    p = plan([1] * 32, lens, tables)
    check(p, [1] * 32, lens, tables, 4, 64, 1)
    assert p["counts"][2] == 1
    # the segments' first row tiles scan every stored position once
    assert sum(u["key1"] - u["key0"] for u in p["units"] if u["rho0"] == 0) == 6400 + sum(n - 6400 for n in lens)


def test_forks_of_forks_share_at_each_level(plan):
    a, b, c = list(range(50)), list(range(50, 90)), list(range(90, 130))
    tables = [a + b + [200], a + b + [201], a + c + [202], a + c + [203], [204]]
    lens = [90 * 64 + 5] * 4 + [17]
    p = plan([1] * 5, lens, tables)
    check(p, [1] * 5, lens, tables, 4, 64, 1)
    assert p["counts"][2] == 3  # a; b; c


def test_a_chain_of_forks_stays_within_its_arrays(plan):
    # sequence i shares i + 1 stretches of 4 pages with the next ones: deeper than the levels kept
    B, stretch = 24, 4
    path = list(range(B * stretch))
    tables = [path[:(i + 1) * stretch] + [1000 + i] for i in range(B)]
    lens = [len(t) * 64 - 10 for t in tables]
    p = plan([1] * B, lens, tables)
    check(p, [1] * B, lens, tables, 4, 64, 1)


def test_prompts_stay_private_and_short_runs_are_not_worth_it(plan):
    pre = list(range(10))
    tables = [pre + list(range(100, 110)), pre + list(range(110, 120))]
    p = plan([600, 600], [1240, 1240], tables)
    check(p, [600, 600], [1240, 1240], tables, 4, 64, 1)
    assert p["counts"][2] == 0
    # one shared page of 32 positions, 30 rows each: the partials would cost more than the reads saved
    tables = [[0, 1, 2], [0, 3, 4]]
    p = plan([30, 30], [90, 90], tables, page=32)
    check(p, [30, 30], [90, 90], tables, 4, 32, 1)
    assert p["counts"][2] == 0


def test_units_fit_the_batch_arrays(plan):
    # far more positions than rows: the split stops at the arrays' units
    tables = [list(range(b * 500, (b + 1) * 500)) for b in range(3)]
    p = plan([1] * 3, [32000] * 3, tables, KV=1, cus=4)
    check(p, [1] * 3, [32000] * 3, tables, 4, 64, 1)


def test_empty_batches(plan):
    for rows, lens, tables in (([], [], []), ([0], [0], [[]]), ([0, 0], [100, 0], [[1, 2], []])):
        p = plan(rows, lens, tables)
        assert p["units"] == [] and p["toks"] == [] and p["counts"][0] == 0


@pytest.mark.parametrize("rows,lens,tables,kw,msg", [
    ([2], [1], [[0]], {}, "2 new rows of 1 positions"),
    ([-1], [5], [[0]], {}, "-1 new rows"),
    ([0], [-5], [[0]], {}, "of -5 positions"),
    ([1], [2 ** 30 + 1], [[0]], {}, "positions"),
    ([1], [2 ** 31 - 1], [[0]], {}, "positions"),
    ([1], [65], [[0]], {}, "need 2 pages of 64, its list holds 1"),
    ([1], [10], [[4096]], {}, "page 0 of its list is 4096, of 4096"),
    ([1], [10], [[-1]], {}, "page 0 of its list is -1"),
    ([1, 1], [10, 130], [[0], [1, 2, -3]], {}, "sequence 1: page 2 of its list is -3"),
    ([1, 1], [10, 10], [[0], [1]], {"limits": (1, 9, 9)}, "2 sequences in a batch of at most 1"),
    ([5, 5], [10, 10], [[0], [1]], {"limits": (2, 9, 9)}, "10 new rows"),
    ([1, 1], [100, 100], [[0, 1], [2, 3]], {"limits": (2, 9, 3)}, "4 pages"),
])
def test_refusals(plan, rows, lens, tables, kw, msg):
    p = plan(rows, lens, tables, **kw)
    assert isinstance(p, str) and msg in p


def test_entries_past_the_positions_are_not_read(plan):
    p = plan([1], [64], [[3, -9, 10 ** 9]])
    assert isinstance(p, dict) and p["pages"] == [3]


@pytest.mark.parametrize("rows,lens,tables,page", [
    ([1, 1], [10, 20], [[5], [5]], 5),                # two sequences write one page
    ([1], [70], [[5, 5]], 5),                         # a page twice in a list, written the second time
    ([1, 0], [10, 40], [[5], [5]], 5),                # written at 9, read by another up to 39
    ([70], [70], [[6, 6]], 6),                        # the same page written twice
])
def test_pages_written_and_listed_elsewhere_are_found(plan, rows, lens, tables, page):
    assert plan(rows, lens, tables)["counts"][3] == page


@pytest.mark.parametrize("rows,lens,tables", [
    ([1, 0], [41, 40], [[5], [5]]),                   # the other reads only what was there before
    ([1, 1], [130, 130], [[5, 6, 7], [5, 6, 8]]),     # a shared prefix
])
def test_pages_read_elsewhere_below_the_new_rows_are_fine(plan, rows, lens, tables):
    assert plan(rows, lens, tables)["counts"][3] == -1
