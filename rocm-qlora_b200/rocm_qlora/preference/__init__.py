"""Token log-probabilities and the paired preference loss."""
from rocm_qlora.preference.loss import PreferenceOutput, preference_loss, token_logprobs

__all__ = ["PreferenceOutput", "preference_loss", "token_logprobs"]
