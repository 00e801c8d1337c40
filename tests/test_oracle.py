"""The CPU oracle (oracle/c2_oracle.c) against the reference's golden vectors (CPU only).

Pins the oracle: every known answer of the reference's own unit tests, plus vectors generated by
running the reference's Cython code (tests/golden/make_golden.py).  When oracle/_ref is present
(dev container, or shipped prebuilt to the GPU box) the oracle is additionally fuzzed live against it.
"""
import numpy as np
import pytest

import oracle
from helpers import load_golden, matrices, payload_diff


@pytest.fixture(scope="module")
def mats():
    return matrices()


def test_oracle_matches_reference_unit_test_answers(mats):
    kats = load_golden("ref_unit_kats.json")
    assert len(kats) >= 50
    n_align = n_cls = 0
    for k in kats:
        if k["fn"] == "global_align":
            got = oracle.global_align(k["seqj"], k["seqi"], mats[k["matrix"]], np.array(k["gap_incentive"], dtype=np.int64),
                                      k["gap_open"], k["gap_extend"])
            assert list(got) == k["out"], k["ref_test"]
            n_align += 1
        elif k["fn"] == "find_indels_substitutions":
            got = oracle.find_indels_substitutions(k["read_al"], k["ref_al"], k["include"])
            assert payload_diff(got, k["out"]) == [], k["ref_test"]
            n_cls += 1
    assert n_align >= 30 and n_cls >= 10


def test_oracle_align_fuzz_vectors(mats):
    for v in load_golden("fuzz_align.json"):
        got = oracle.global_align(v["seqj"], v["seqi"], mats[v["matrix"]], np.array(v["gap_incentive"], dtype=np.int64),
                                  v["gap_open"], v["gap_extend"])
        assert list(got) == v["out"], v


def test_oracle_classify_fuzz_vectors():
    n = 0
    for v in load_golden("fuzz_classify.json"):
        if v["fn"] != "find_indels_substitutions":
            continue
        got = oracle.find_indels_substitutions(v["read_al"], v["ref_al"], v["include"])
        assert payload_diff(got, v["out"]) == [], v
        n += 1
    assert n >= 400


def test_oracle_realistic_vectors(mats):
    for v in load_golden("realistic.json"):
        got = oracle.global_align(v["seqj"], v["seqi"], mats[v["matrix"]], np.array(v["gap_incentive"], dtype=np.int64),
                                  v["gap_open"], v["gap_extend"])
        assert list(got) == v["out"]
        p = oracle.find_indels_substitutions(got[0], got[1], v["include"])
        assert payload_diff(p, v["payload"]) == []


def test_oracle_error_behaviour(mats):
    m = mats["EDNAFULL"]
    # CRISPResso2Align.pyx:124-126: wrong gap_incentive length -> returns the int 0
    assert oracle.global_align("ACGT", "ACGT", m, np.zeros(3, dtype=np.int64)) == 0
    # zero-length input is undefined in the reference; the oracle refuses
    st = oracle.global_align_raw("", "ACGT", m, np.zeros(5, dtype=np.int64))[0]
    assert st & oracle.ERR_EMPTY
    # out-of-matrix characters: a reference character >= 90, a read character that the largest reference character pushes
    # past the end of the flat buffer ('Y' = 89: 89 * 90 + 97 >= 8100), bytes >= 128 (signed char in the reference)
    assert oracle.global_align_raw("ACGT", "ACGa", m, np.zeros(5, dtype=np.int64))[0] & oracle.ERR_OOB_CHAR
    assert oracle.global_align_raw("ACGa", "ACGY", m, np.zeros(5, dtype=np.int64))[0] & oracle.ERR_OOB_CHAR
    assert oracle.global_align_raw("ACG\x85", "ACGT", m, np.zeros(5, dtype=np.int64))[0] & oracle.ERR_OOB_CHAR
    # ... while 'a' against 'T' (84 * 90 + 97 < 8100) is an element of the buffer: what the reference itself reads
    assert oracle.global_align_raw("ACGa", "ACGT", m, np.zeros(5, dtype=np.int64))[0] == 0


def test_read_characters_beyond_the_matrix_follow_the_reference(mats):
    """CRISPResso2Align.pyx:212 indexes matrix[ci, cj] with bounds checking off: lower-case reads, and the string "None" that
    every default run of the reference aligns as a flexiguide (CRISPRessoCORE.py:3095-3105), read later rows of the flat
    buffer.  The restatement against the reference's own compiled module, on such reads."""
    ref = oracle.ref()
    if ref is None:
        pytest.skip("oracle/_ref not built")
    A, _ = ref
    rng = np.random.default_rng(77)
    for name, gaps in (("EDNAFULL", [(-20, -2), (-5, -3), (-50, 0)]), ("BLOSUM62", [(-5, -3)])):
        m = mats[name]
        for t in range(60):
            L = int(rng.integers(20, 120))
            amp = "".join(rng.choice(list("ACGT"), L))
            rd = list(amp[int(rng.integers(0, 5)):L - int(rng.integers(0, 5))])
            for _ in range(int(rng.integers(1, 8))):
                rd[int(rng.integers(0, len(rd)))] = str(rng.choice(list("acgtnxyzo e_~")))
            rd = "".join(rd) if t else "None"
            g = np.zeros(L + 1, dtype=np.int64)
            g[int(rng.integers(0, L + 1))] = 1
            for go, ge in gaps:
                want = A.global_align(rd, amp, matrix=m, gap_incentive=g, gap_open=go, gap_extend=ge)
                assert tuple(oracle.global_align(rd, amp, m, g, go, ge)) == want, (rd, amp)


def test_matrix_files_match_reference(mats):
    ref = oracle.ref()
    if ref is None:
        pytest.skip("oracle/_ref not built")
    import os
    d = os.path.join(os.path.dirname(oracle.__file__), "_ref")
    for name in ("EDNAFULL", "BLOSUM62"):
        assert np.array_equal(ref[0].read_matrix(os.path.join(d, name)), mats[name])
    from crispresso2_amd import CRISPResso2Align as A
    assert np.array_equal(ref[0].make_matrix(), A.make_matrix())
    assert np.array_equal(ref[0].make_matrix(3, -2, -1, 0), A.make_matrix(3, -2, -1, 0))


def test_oracle_live_fuzz_against_reference(mats):
    ref = oracle.ref()
    if ref is None:
        pytest.skip("oracle/_ref not built")
    A, R = ref
    rng = np.random.default_rng(31337)
    m = mats["EDNAFULL"]
    for _ in range(300):
        L = int(rng.integers(1, 90))
        refseq = "".join(rng.choice(list("ACGTN"), L))
        read = "".join(rng.choice(list("ACGTN"), int(rng.integers(1, 90)))) if rng.random() < 0.3 else refseq[int(rng.integers(0, 5)):] + "ACG"[: int(rng.integers(0, 4))]
        g = np.zeros(L + 1, dtype=np.int64)
        g[int(rng.integers(0, L + 1))] = 1
        go, ge = [(-20, -2), (-50, 0), (-5, -3)][int(rng.integers(0, 3))]
        exp = A.global_align(read, refseq, matrix=m, gap_incentive=g, gap_open=go, gap_extend=ge)
        got = oracle.global_align(read, refseq, m, g, go, ge)
        assert tuple(got) == tuple(exp)
        inc = list(range(int(rng.integers(0, L)), L))[: int(rng.integers(1, 20))]
        assert payload_diff(oracle.find_indels_substitutions(got[0], got[1], inc),
                            R.find_indels_substitutions(exp[0], exp[1], inc).__dict__) == []


@pytest.mark.parametrize("codes", [list, np.array])
def test_aggregate_takes_substituted_bases_as_letters_or_byte_codes(codes):
    """The reference's payload spells a substituted base as a letter, the classifier kernels' flat lists hold its byte code: the same
    vectors from both, against counts written out by hand (an N in the read is no substitution, COREResources.pyx:113)."""
    from oracle import aggregate
    amp = "ACGTACGTAC"
    reads = [("TCGTACGTAC", 3), ("ACGNACGTAA", 5), ("ACCTACGTAG", 7)]
    letters, flat = [], []
    for s1, c in reads:
        p = oracle.find_indels_substitutions(s1, amp, [2, 3])
        p["aln_seq"], p["aln_ref"] = s1, amp
        assert all(isinstance(b, str) for b in p["all_substitution_values"])
        letters.append((p, c))
        q = dict(p)
        for k in ("all_substitution_values", "substitution_values"):
            q[k] = codes([ord(b) for b in p[k]])
        flat.append((q, c))
    want = {"T": {0: 3}, "N": {}, "A": {9: 5}, "C": {2: 7}, "G": {9: 7}}
    for items in (letters, flat):
        got = aggregate.aggregate(items, len(amp))
        for n in "ACGTN":
            assert {int(k): int(got["all_substitution_base_vectors_" + n][k]) for k in np.flatnonzero(got["all_substitution_base_vectors_" + n])} == want[n]
    a, b = aggregate.aggregate(letters, len(amp)), aggregate.aggregate(flat, len(amp))
    assert a.keys() == b.keys() and all(np.array_equal(a[k], b[k]) for k in a)
