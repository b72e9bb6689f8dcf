"""Layout of the draft attention's shared memory, from the kernel's own constants: what a row reads lies within its arrays."""
import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hs-guard_b200", "csrc", "draft_attn.cuh")


@pytest.fixture(scope="module")
def index():
    """The kernel's place of a row's mask words, (item, row, G, block, KT) -> word."""
    text = open(SOURCE).read()
    where = re.search(r"const uint32_t\* first_words = row_words \+ (.*);", text).group(1)
    token = re.search(r"constexpr int da_row_token\(int row, int group, int block\) \{\s*return (.*) \? (.*) : (.*);", text)
    row_tok = re.search(r"const int row_tok = (.*);", text).group(1)

    def function(names, expression, **known):
        return eval("lambda %s: %s" % (names, expression.replace("/", "//").replace("plan.block", "block")), known)

    own = function("row, G", row_tok)
    clamped = token and function("row, group, block", "%s if %s else %s" % (token.group(2), token.group(1), token.group(3)))
    place = function("item, row, G, block, KT, row_tok", where, da_row_token=clamped)
    return lambda item, row, G, block, KT: place(item, row, G, block, KT, own(row, G))


@pytest.mark.parametrize("KT", [64, 128])
def test_rows_read_mask_words_of_their_items_tokens(index, KT):
    words = KT // 32
    for G in range(1, 129):
        for max_tree in (1, 2, 128 // G, 1024):
            block = min(max_tree, 128 // G)
            for item in range(2):
                for row in range(128):
                    first = index(item, row, G, block, KT)
                    assert item * block * words <= first and first + words <= (item + 1) * block * words, (G, block, item, row)
                    if row < block * G:
                        assert first == (item * block + row // G) * words


def test_rotations_are_read_from_where_two_fit():
    """draft_norm_kernel reads its (cos, sin) pairs two at a time, 16 bytes: more than float2 is aligned to by itself."""
    text = open(os.path.join(os.path.dirname(SOURCE), "draft_rows.cuh")).read()
    assert "reinterpret_cast<const float4*>(s_turn + " in text
    assert re.search(r"extern __shared__ __align__\(16\) float2 s_turn\[\];", text)
