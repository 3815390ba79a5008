"""Refusals of the serving operators at the ends of their ranges: arguments are checked before anything touches a device."""
from test_serving_cpu import refused, rules


def test_rules_refuse_vocabularies_that_steps_over_them_would_leave():
    # a step of 16384 tokens from the last multiple below 2^31 ends beyond 32 bits
    refused(rules(vocab=2 ** 31 - 1, ld_logits=2 ** 31, ld_out=2 ** 31), "dimensions")
    refused(rules(vocab=2 ** 30 + 1, ld_logits=2 ** 31, ld_out=2 ** 31), "dimensions")
