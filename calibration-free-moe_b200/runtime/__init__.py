"""Callers of the reader inside a serving engine: decode/prefill row split, chunking, reports; and the exact side of
a decode step around it: router, whole routed experts, scores of logits."""
