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

    def add(at: int) -> bool:
        """The guesses text[at:at + length]; False once there are `nodes`."""
        parent = -1
        for t in text[at:at + length]:
            if (parent, t) not in children:
                if len(tokens) == nodes:
                    return False
                children[parent, t] = len(tokens)
                tokens.append(t)
                parents.append(parent)
            parent = children[parent, t]
        return True

    # the places where the last token occurred before, the latest first, by list.index (100000 tokens in a millisecond),
    # and how many tokens up to there recur
    n, back, at = len(text), text[::-1], 0
    most, found = 1, []
    while match > 0 and n:
        try:
            at = back.index(back[0], at + 1)
        except ValueError:
            break
        m = 1
        while m < match and at + m < n and back[at + m] == back[m]:
            m += 1
        if m == match:
            if not add(n - at):
                return tokens, parents
        elif m > most:
            most, found = m, [at]
        elif m == most:
            found.append(at)
    if not tokens:
        for at in found:
            if not add(n - at):
                break
    return tokens, parents
