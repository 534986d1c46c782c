"""That the play of the 8-bit attention kernels' waits (``test_fp8_pipeline_cpu``) is of the kernels as they stand, and sees what
is wrong.

The sizes of the rings, the arrivals that a barrier's phase takes and each role's waits are read from the kernels' source and
compared with the play's; and the play is run with a wait taken out or a ring too small, which some schedule has to find.
"""

import inspect
import os
import random
import re

import pytest

import test_fp8_pipeline_cpu as play

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dropkv_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//(?! =)[^\n]*", "", f.read())  # (without comments, but for the lines that head a role)


def constant(text, name):
    return re.search(rf"\b{name} = ([^;,]+)[;,]", text).group(1).strip()


WAIT = re.compile(r"\bwait\((&(?:bars|full|empty)\[.*?\]), ([^()]*?(?:\([^()]*\))?[^()]*?), [^,()]+\)")


def waits(section):
    return [(re.sub(r"L::B_", "", bar), count) for bar, count in WAIT.findall(section)]


def test_many_rows_is_the_kernel():
    text = source("fp8_attn.cu")
    assert constant(text, "NS") == "PARTS == 2 ? 3 : 2"             # the play's 2 and 3
    assert constant(text, "SCALES") == "NS + 2"
    body = inspect.getsource(play.many_rows)
    assert "scales = NS + 2" in body
    # arrivals of a phase; where bytes are counted too, the play has their landing as one more
    inits = dict(re.findall(r"mbar_init\(&bars\[L::B_(\w+)(?: \+ i)?\], (\d+)\)", text))
    assert inits == dict(KF="1", KE="1", VF="1", VE="2", S="2", P="4", W="2", O="1", Q="1", END="1")
    for name, need in (("KF", 2), ("KE", 1), ("VF", 2), ("VE", 2), ("S", 2), ("P", 4), ("W", 2), ("O", 1)):
        assert f'("{name}", {need})' in body
    # each role's waits, in order
    roles = re.split(r"// =+ ([\w ]+?) =+\n", text)
    roles = dict(zip(roles[1::2], roles[2::2]))
    assert list(roles) == ["TMA producer", "MMA issuer", "V to fp16", "softmax"]
    assert waits(roles["TMA producer"]) == [
        ("&bars[KE + (n - 1) % NS]", "(n - 1) / NS"),                               # the last piece's queries are read
        ("&bars[(kv ? VE : KE) + slot]", "turn - 1")]
    assert waits(roles["MMA issuer"]) == [
        ("&bars[W + buf]", "i >> 1"), ("&bars[P + buf]", "i >> 1"),                  # the second product
        ("&bars[Q]", "pieces++"), ("&bars[KF + slot]", "turn"), ("&bars[O + buf]", "(j - 2) >> 1")]
    assert waits(roles["V to fp16"]) == [("&bars[VF + slot]", "turn"), ("&bars[O + buf]", "(j - 2) >> 1")]
    assert waits(roles["softmax"]) == [
        ("&bars[O + 1 - buf]", "(j - 1) >> 1"),                                     # a reference moves
        ("&bars[S + buf]", "j >> 1"), ("&bars[W + buf]", "j >> 1"),                  # (of a masked tile)
        ("&bars[O + (last & 1)]", "last >> 1")]


def test_few_rows_is_the_kernel():
    text = source("fp8_decode.cu")
    assert constant(text, "SLOTS") == "(R16 ? 4 : 5) * (128 / D)"    # 4, 5, 8 and 10
    assert constant(text, "SCALES") == "SLOTS / 2 + 1"
    assert "scales = NS // 2 + 1" in inspect.getsource(play.few_rows)
    assert constant(text, "FD_WARPS") == "4"
    assert re.findall(r"mbar_init\(&(\w+)\[i\], (\w+)\)", text) == [("full", "1"), ("empty", "WARPS")]
    assert waits(text) == [("&empty[slot]", "n / NS - 1"), ("&full[slot]", "turn"), ("&full[slot]", "turn")]


def changed(function, old, new, place=0):
    """The play with a piece of its text (the place-th of its kind) put differently."""
    text = inspect.getsource(function)
    parts = text.split(old)
    assert len(parts) > place + 1, old
    text = old.join(parts[:place + 1]) + new + old.join(parts[place + 1:])
    space = dict(vars(play))
    exec(text, space)
    return space[function.__name__]


def found(run):
    """Some schedule ends in a failed check, a wait without end, or what was never written."""
    for seed in range(300):
        try:
            run(seed)
        except (AssertionError, KeyError):
            return True
    return False


def many(function, NS):
    def run(seed):
        r = random.Random(seed)
        pieces = [[9, 7], [1, 1, 1, 2], [13], [2, 5, 1, 4]][seed % 4]
        share = r.choice([0.0, 0.5, 1.0]), r.choice([0.0, 0.5, 1.0])
        picks = [(r.random() < share[0], r.random() < share[1]) for _ in range(sum(pieces))]
        function(pieces, NS, seed, lambda j: picks[j])
    return run


@pytest.mark.parametrize("NS", [2, 3])
@pytest.mark.parametrize("what,old,new,place", [
    ("nothing", "scales = NS + 2", "scales = NS + 2", 0),
    ("scales of a tile less", "scales = NS + 2", "scales = NS + 1", 0),
    ("queries over those that products read", "            if n:\n                yield (\"KE\", (n - 1) % NS), (n - 1) // NS\n", "", 0),
    ("loads into slots that are read", "                    if n >= NS:\n                        yield (kv + \"E\", slot), n // NS - 1\n", "", 0),
    ("the second product without V", "            yield (\"W\", i & 1), i >> 1\n", "", 0),
    ("the second product without weights", "            yield (\"P\", i & 1), i >> 1\n", "", 0),
    ("products without queries", "            yield \"Q\", p\n", "", 0),
    ("products without K", "                yield (\"KF\", j % NS), j // NS\n", "", 0),
    # (S over weights that are read needs no wait: products run in the order of their issue)
    ("V16 over what is read", "            if j >= 2:\n                yield (\"O\", j & 1), (j - 2) >> 1\n            assert", "            assert", 0),
    ("V before it is there", "            yield (\"VF\", j % NS), j // NS\n", "", 0),
    ("logits before they are there", "                yield (\"S\", j & 1), j >> 1\n", "", 0),
    ("O while a product adds to it", "                if moves and j > first[p]:\n                    yield (\"O\", 1 - (j & 1)), (j - 1) >> 1\n",
     "                if moves and j > first[p]:\n", 0),
    ("O before its last product", "            yield (\"O\", last & 1), last >> 1\n", "", 0),
    ("V's slots given back by one warp", "(\"VE\", 2)", "(\"VE\", 1)", 0),
    ("weights of some warps", "(\"P\", 4)", "(\"P\", 3)", 0),
])
def test_many_rows_finds_what_is_taken_out(what, old, new, place, NS):
    assert found(many(changed(play.many_rows, old, new, place), NS)) == (what != "nothing")


@pytest.mark.parametrize("NS", [4, 5, 8, 10])
@pytest.mark.parametrize("what,old,new", [
    ("nothing", "scales = NS // 2 + 1", "scales = NS // 2 + 1"),
    ("scales of a tile less", "scales = NS // 2 + 1", "scales = (NS + 1) // 2 - 1"),  # (an even NS has one to spare)
    ("loads into slots that are read", "            if n >= NS:\n                yield (\"empty\", slot), n // NS - 1\n", ""),
    ("tiles before they are there", "            yield (\"full\", n % NS), n // NS\n", ""),
    ("slots given back by some warps", "(\"empty\", i), 4", "(\"empty\", i), 3"),
])
def test_few_rows_finds_what_is_taken_out(what, old, new, NS):
    run = changed(play.few_rows, old, new)
    assert found(lambda seed: run([5, 23][seed % 2], NS, seed)) == (what != "nothing")
