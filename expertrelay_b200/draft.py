"""Drafts: guesses at the next tokens of a text for QwenMoeModel.generate_drafted.

The reference decodes one token a call (runtime/generate.py). A draft needs no
model: texts repeat themselves.
"""

from __future__ import annotations


def from_text(text: list[int], *, nodes: int = 32, length: int = 8, match: int = 3) -> tuple[list[int], list[int]]:
    """What followed the text's last `match` tokens (or as many as recur) where they
    occurred before, the latest occurrences first, `length` tokens of each: a tree
    of up to `nodes` guesses, (tokens, parents); empty where nothing recurs."""
    tokens: list[int] = []
    parents: list[int] = []
    children: dict[tuple[int, int], int] = {}
    n = len(text)
    for m in range(min(match, n - 1), 0, -1):
        for at in range(n - m - 1, -1, -1):
            if text[at:at + m] != text[n - m:]:
                continue
            parent = -1
            for t in text[at + m:at + m + length]:
                if (parent, t) not in children:
                    if len(tokens) == nodes:
                        return tokens, parents
                    children[parent, t] = len(tokens)
                    tokens.append(t)
                    parents.append(parent)
                parent = children[parent, t]
        if tokens:
            break
    return tokens, parents
