"""The API page's lines on the device operations and optimizers are what their docstrings say."""
import importlib
import inspect
import re
from pathlib import Path

import pytest

PAGE = (Path(__file__).resolve().parent.parent / "docs" / "api.md").read_text()


def entries(module):
    section = re.search(rf"## `{re.escape(module)}`.*?\n(.*?)(?=\n## |\Z)", PAGE, re.S).group(1)
    # (a signature can hold the column's separator: the kind follows the last of the name's backquotes)
    return re.findall(r"^\| `([\w.]+)\(.*?\)[^`]*` \| (?:function|class) \| (.*) \|$", section, re.M)


def first_paragraph(thing):
    return " ".join(inspect.getdoc(thing).split("\n\n")[0].split())


@pytest.mark.parametrize("module,least", [("nangila.ops", 12), ("nangila.optim", 1)])
def test_the_page_says_what_the_docstrings_say(module, least):
    found = entries(module)
    assert len(found) >= least, found
    for name, text in found:
        thing = importlib.import_module(module)
        for part in name.split("."):
            thing = getattr(thing, part)
        assert text == first_paragraph(thing), name
