"""The command line's beam search, with an engine that is none."""
import types

import pytest

from gpullama3.java_b200.engine import api, cli


class _Engine:
    max_length, last_metrics = 100, types.SimpleNamespace(prompt_tokens=4, generated_tokens=5, decode_steps=2, seconds=1.0, prefill_seconds=0.5,
                                                          decode_seconds=0.5, total_tokens=9, tokens_per_second=9.0)

    @classmethod
    def from_folder(cls, *args, **kwargs):
        return cls()

    def beam_search(self, prompts, beams, max_new_tokens, *, length_penalty, stop_ids):
        return [[100 + p[0], 7] for p in prompts]

    def generate(self, prompts, *, on_token, **kwargs):
        outs = [[100 + p[0], 7] for p in prompts]
        for i, out in enumerate(outs):
            for t in out:
                on_token(i, t)
        return outs


@pytest.mark.parametrize("beams", [1, 3])
def test_echo_copies_every_token(monkeypatch, capsys, beams):
    monkeypatch.setattr(api, "Engine", _Engine)
    rc = cli.main(["-m", "folder", "-p", "5 6", "-p", "8 9", "--echo", "true", "--stream", "false", "--beams", str(beams)])
    out, err = capsys.readouterr()
    assert rc in (0, None) and out.split() == ["105", "7", "108", "7"]
    assert " ".join(err.split()).startswith("5 6 8 9 105 7 108 7")


def test_no_echo_copies_none(monkeypatch, capsys):
    monkeypatch.setattr(api, "Engine", _Engine)
    cli.main(["-m", "folder", "-p", "5 6", "--beams", "2"])
    out, err = capsys.readouterr()
    assert out.split() == ["105", "7"] and "105" not in err
