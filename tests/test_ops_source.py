"""The policy operators' inline assembly names every register that it writes."""
import os
import re

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "urgym_amd", "ops", "csrc")


def test_inline_assembly_names_the_registers_it_writes():
    found = 0
    for name in sorted(os.listdir(SRC)):
        for body in re.findall(r"\basm\s*(?:volatile)?\s*\((.*?)\)\s*;", open(os.path.join(SRC, name)).read(), re.S):
            template = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', re.split(r"::|(?<!:):(?!:)", body)[0]))
            for line in re.split(r"\\n\\t|\\n", template):
                words = re.findall(r"[^\s,]+", line)
                if len(words) > 1 and re.fullmatch(r"m0|vcc|exec|scc|[sv]\d+|[sv]\[\d+:\d+\]", words[1]) and not words[0].startswith("s_waitcnt"):
                    found += 1
                    assert f'"{words[1]}"' in body.split(":")[-1], (name, line)
    assert found
