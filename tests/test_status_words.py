"""A status word that more than one fault is reported in: no report takes another's bit away."""
import glob
import os
import re
from collections import defaultdict

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moonshine_b200", "csrc")


def test_words_of_several_bits_are_only_added_to():
    raised = defaultdict(set)                    # word -> (bit, how)
    for path in glob.glob(os.path.join(CSRC, "*.cu")):
        text = open(path).read()
        for how, word, bit in re.findall(r"(atomicExch|atomicOr)\(&(g_\w+_status), (\d+)u\)", text):
            raised[word].add((bit, how))
        for word, bit in re.findall(r"(?<!uint32_t )\b(g_\w+_status) = (\d+)u", text):
            raised[word].add((bit, "="))
    assert len(raised) >= 8
    several = {word: reports for word, reports in raised.items() if len({bit for bit, _ in reports}) > 1}
    assert several                               # the pattern above still finds the one there is
    for word, reports in several.items():
        assert {how for _, how in reports} == {"atomicOr"}, (word, reports)
