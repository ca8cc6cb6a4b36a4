"""Calls of the samplers, verifiers and grammars on a named stream, without a GPU (stand-ins as in test_kv_binding): what
they make belongs to that stream, what they are given is held until it is through."""

from __future__ import annotations

import inspect

import pytest
import torch

import sixi_smp as S
from sixi_smp import json_grammar, json_schema
from test_kv_binding import F32, I32, I64, MAIN, SIDE, Tensor, lib  # noqa: F401

U8 = torch.uint8


def handle(kind):
    x = object.__new__(kind)
    x.h, x.device, x.vocab, x.mask_words = None, 0, 64, 2
    return x


def rows(n=6):
    return Tensor((n, 64), F32)


def calls():
    smp, gram, schema = handle(S.Sampler), handle(json_grammar.JsonGrammar), handle(json_schema.SchemaGrammar)
    params, drafts, states, tokens = Tensor((2, 64), U8), Tensor((2, 2), I32), Tensor((2, 32), U8), Tensor((2,), I32)
    return {
        "sample": (smp.sample, [rows(), params]),
        "sample_indexed": (smp.sample_indexed, [rows(), tokens, params, Tensor((6,), I32), Tensor((6,), I32)]),
        "gather_rows": (smp.gather_rows, [rows(), tokens, 64]),
        "greedy_argmax": (smp.greedy_argmax, [rows()]),
        "candidates": (smp.candidates, [rows(), params]),
        "verify": (smp.verify, [rows(), drafts, params]),
        "verify_draft_logits": (smp.verify_draft_logits, [rows(), rows(4), Tensor((2,), F32), drafts, params]),
        "full_distribution": (smp.full_distribution, [rows(), Tensor((6,), F32)]),
        "numeric_policy": (smp.numeric_policy, [rows()]),
        "suffix_draft": (smp.suffix_draft, [Tensor((9,), I32), Tensor((3,), I64)]),
        "shard_candidates": (smp.shard_candidates, [rows(), 0, 64, params]),
        "merge_shards": (smp.merge_shards, [Tensor((2, 6, 64, 2), I32), Tensor((2, 6, 24), U8), params]),
        "verify_static": (S.verify_static, [64, rows(), drafts, params]),
        "json reset": (gram.reset, [states]),
        "json fill_masks": (gram.fill_masks, [states]),
        "json advance": (gram.advance, [states, tokens]),
        "json expand_drafts": (gram.expand_drafts, [states, drafts]),
        "schema reset": (schema.reset, [states]),
        "schema fill_masks": (schema.fill_masks, [states]),
        "schema advance": (schema.advance, [states, tokens]),
    }


@pytest.mark.parametrize("name", list(calls()))
def test_a_named_stream_owns_what_the_call_makes(lib, name):  # noqa: F811
    call, args = calls()[name]
    call(*args, stream=SIDE)
    assert all(s is SIDE for s, _ in lib.made)
    assert all(t.used_on[:1] == [SIDE] for t in args if isinstance(t, Tensor))
    assert len(lib.calls) == 1 and lib.current == [MAIN]
    lib.made.clear()
    call, args = calls()[name]
    call(*args)
    assert all(s is MAIN for s, _ in lib.made) and not any(t.used_on for t in args if isinstance(t, Tensor))


def test_every_call_with_a_stream_is_among_them():
    with_stream = set()
    for kind, prefix in ((S.Sampler, ""), (json_grammar.JsonGrammar, "json "), (json_schema.SchemaGrammar, "schema ")):
        with_stream |= {prefix + n for n, f in vars(kind).items()
                        if inspect.isfunction(f) and not n.startswith("_") and "stream" in inspect.signature(f).parameters}
    # (sample_host takes host arrays and allocates nothing on the device)
    assert with_stream - {"sample_host"} == set(calls()) - {"verify_static"}
