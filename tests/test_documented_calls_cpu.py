"""The documents' Python examples: their calls of the serving operators take the arguments that these have, and an
append to the 8-bit cache after a reservation says how many tokens were served."""
from __future__ import annotations

import ast
import inspect
import re

from conftest import REPO
from kernels import logit_rules, paged_cache, paged_cache8, paged_tables, spec_verify

OPERATORS = {f.__name__: f for f in (
    paged_cache.paged_append, paged_cache.paged_attention, paged_cache.rope_table, paged_cache8.cache8, paged_cache8.paged_append8,
    paged_cache8.paged_attention8, paged_tables.page_pool, paged_tables.paged_reserve, paged_tables.paged_release,
    logit_rules.adjust_logits, logit_rules.count_tokens, logit_rules.token_bits, spec_verify.speculative_verify)}


def blocks():
    """(document, [(operator, call)]) of every Python block that calls some."""
    for doc in sorted(REPO.glob("*.md")):
        for text in re.findall(r"^```python\n(.*?)^```", doc.read_text(), re.M | re.S):
            try:
                tree = ast.parse(text)
            except SyntaxError:              # an outline, not a program
                continue
            calls = [(n.func.id, n) for n in ast.walk(tree)
                     if isinstance(n, ast.Call) and isinstance(n.func, ast.Name) and n.func.id in OPERATORS]
            if calls:
                yield doc.name, calls


def test_calls_have_the_operators_arguments():
    used = set()
    for doc, calls in blocks():
        for name, call in calls:
            used.add(name)
            if any(isinstance(a, ast.Starred) for a in call.args) and name in ("paged_append8", "paged_attention8"):
                args = [x for a in call.args for x in ([None] * 4 if isinstance(a, ast.Starred) else [a])]   # *cache
            else:
                args = call.args
            inspect.signature(OPERATORS[name]).bind(*args, **{k.arg: k.value for k in call.keywords})
    assert used >= {"paged_append", "paged_attention", "paged_append8", "paged_attention8", "paged_reserve", "adjust_logits"}


def test_an_append_after_a_reservation_takes_what_was_served():
    """Without `count` all rows are new tokens, and those of a sequence that got less would overwrite its older ones."""
    seen = 0
    for doc, calls in blocks():
        if "paged_reserve" not in dict(calls):
            continue
        for name, call in calls:
            if name == "paged_append8":
                seen += 1
                assert any(k.arg == "count" for k in call.keywords), f"{doc}: {ast.unparse(call)}"
    assert seen
